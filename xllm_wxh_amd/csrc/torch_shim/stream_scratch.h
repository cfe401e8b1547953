// Scratch memory that calls of several kernel launches share, one buffer per (device, stream).  Whoever holds a stream's
// buffer enqueues all of a call's launches before the next holder enqueues its first: launches run in the order of the
// stream, so what one call leaves in the buffer between its launches is its own, from however many host threads the stream
// is used.
#pragma once

#include <map>
#include <mutex>
#include <utility>

namespace xllm::kernel::hip {

template <class Buffer>
class StreamScratch {
  struct Entry {
    std::mutex busy;
    Buffer buffer;
  };

 public:
  // The buffer of a stream, this holder's until it goes out of scope.
  class Held {
   public:
    Buffer& operator*() const { return entry_->buffer; }

   private:
    friend class StreamScratch;
    explicit Held(Entry& entry) : entry_(&entry), lock_(entry.busy) {}
    Entry* entry_;
    std::unique_lock<std::mutex> lock_;
  };

  // Waits for the stream's holder, if there is one; other streams' holders are not waited for.
  Held hold(int device, void* stream) {
    Entry* entry;
    {
      std::lock_guard<std::mutex> lock(mutex_);
      entry = &entries_[{device, stream}];
    }
    return Held(*entry);
  }

 private:
  std::mutex mutex_;
  std::map<std::pair<int, void*>, Entry> entries_;  // (entries stay where they are)
};

}  // namespace xllm::kernel::hip
