// Two host threads that use the scratch buffer of one stream, without a GPU: the stream is a list of what was enqueued.
#include <atomic>
#include <chrono>
#include <cstdio>
#include <future>
#include <thread>
#include <vector>

#include "torch_shim/stream_scratch.h"

using xllm::kernel::hip::StreamScratch;

int main() {
  StreamScratch<int> scratch;
  int stream_a = 0, stream_b = 0;

  // While a call holds a stream's buffer another call on that stream waits, one on another stream or device does not.
  std::atomic<bool> entered{false};
  std::future<void> other;
  {
    const auto held = scratch.hold(0, &stream_a);
    *held = 7;
    other = std::async(std::launch::async, [&] {
      const auto mine = scratch.hold(0, &stream_a);
      entered = true;
      if (*mine != 8) std::printf("the buffer was not handed over\n");
    });
    *scratch.hold(0, &stream_b) = 1;
    *scratch.hold(1, &stream_a) = 2;
    if (other.wait_for(std::chrono::milliseconds(300)) == std::future_status::ready || entered) {
      std::printf("two calls hold one stream's buffer\n");
      return 1;
    }
    *held = 8;
  }
  other.get();
  if (!entered || *scratch.hold(0, &stream_b) != 1 || *scratch.hold(1, &stream_a) != 2) {
    std::printf("a buffer is not its stream's\n");
    return 1;
  }

  // Calls of two launches from four threads: the second of a call follows its first on the stream.
  std::vector<int> stream;  // (two entries to a call; written under the buffer only)
  std::vector<std::thread> threads;
  for (int t = 0; t < 4; ++t) {
    threads.emplace_back([&, t] {
      for (int i = 0; i < 500; ++i) {
        const auto held = scratch.hold(0, &stream_a);
        stream.push_back(t);
        std::this_thread::yield();
        stream.push_back(t);
      }
    });
  }
  for (auto& t : threads) t.join();
  for (size_t i = 0; i + 1 < stream.size(); i += 2) {
    if (stream[i] != stream[i + 1]) {
      std::printf("the launches of two calls are mixed\n");
      return 1;
    }
  }
  std::printf("stream scratch ok %zu\n", stream.size());
  return 0;
}
