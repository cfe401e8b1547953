"""The scratch buffer that the libtorch layer's tree attention keeps per (device, stream): the attention kernel leaves
partial results in it that the merge reads, so no other host thread may enqueue a call on the stream between the two."""
import os
import subprocess

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "xllm_wxh_amd", "csrc")


def test_one_call_at_a_time_on_a_stream(tmp_path):
    exe = str(tmp_path / "stream_scratch_harness")
    subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-pthread", "-I", CSRC,
                    os.path.join(REPO, "tests", "stream_scratch_harness.cpp"), "-o", exe], check=True)
    run = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert run.returncode == 0 and "stream scratch ok 4000" in run.stdout, run.stdout[-4000:]


@pytest.mark.gpu
def test_threads_of_one_stream(gpu):
    """Calls of different sizes from several threads on the default stream, the scratch outgrown on the way."""
    import threading

    from test_gpu_tree_attention import TreeCase
    from xllm_wxh_amd import ops

    cases = [TreeCase([n] * b, [1500 + 37 * n] * b, 8, 2, 128, 16, seed=50 + n) for n, b in ((3, 1), (9, 2), (17, 3), (40, 1))]
    want = [c.run()[0] for c in cases]
    outs = [[torch.zeros_like(c.q) for _ in range(8)] for c in cases]

    def work(i):
        c = cases[i]
        for o in outs[i]:
            ops.batch_tree_decode(c.q, c.k, c.v, o, c.d_table, c.d_lens, c.d_mask, scale=c.scale, q_indptr=c.d_indptr,
                                  q_per_seq=max(c.counts))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for w, got in zip(want, outs):
        for o in got:
            assert torch.equal(o, w)
