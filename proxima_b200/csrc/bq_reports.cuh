// bq_reports.cuh — failures of block products that only the device sees, kept apart by caller.
//
// A caller has a record: two words of pinned host memory that its calls' kernels write, and a number that they
// write into them. Callers are the sessions, the streams of calls made with the context itself, and
// each host call. Numbers are never used twice, so a kernel or graph that outlives its caller tells nobody
// else, and the words stay allocated until the context goes. They are given out again late: behind at
// least QUARANTINE others.
#pragma once

#include <deque>
#include <memory>
#include <mutex>
#include <unordered_map>
#include <vector>

#include "common.cuh"

namespace pxc {
namespace bq {

// A word of a record each.
enum Fault : uint32_t { FAULT_OFFSETS = 0, FAULT_TIMEOUT = 1, FAULT_WORDS = 2 };

struct Record {
  uint32_t* words = nullptr;
  uint32_t id = 0;

  // Reports a failure, once. Of two kinds, the other stays for the next call.
  void take() const {
    for (const Fault f : {FAULT_TIMEOUT, FAULT_OFFSETS}) {
      uint32_t seen = __atomic_load_n(words + f, __ATOMIC_RELAXED);
      if (seen != id || !__atomic_compare_exchange_n(words + f, &seen, 0u, false, __ATOMIC_RELAXED, __ATOMIC_RELAXED))
        continue;
      if (f == FAULT_TIMEOUT)
        throw make_failure(PXC_TIMEOUT, 0, 0, nullptr, "a device-side wait of a block product ran out");
      throw make_failure(PXC_CONFIGURATION, 0, 0, "offsets",
                         "a grouped product's offsets fell, left the rows, or did not fit the output");
    }
  }
};

class Reports {
 public:
  explicit Reports(pxc_ctx* ctx) : ctx_(ctx) { add_slab(); }
  ~Reports() { close(); }
  Reports(const Reports&) = delete;
  Reports& operator=(const Reports&) = delete;

  // NULL once the context has gone; sessions may outlive it.
  pxc_ctx* context() const { return __atomic_load_n(&ctx_, __ATOMIC_ACQUIRE); }

  void close() {
    std::lock_guard<std::mutex> lock(mu_);
    __atomic_store_n(&ctx_, static_cast<pxc_ctx*>(nullptr), __ATOMIC_RELEASE);
    for (uint32_t* s : slabs_) cudaFreeHost(s);
    slabs_.clear();
    free_.clear();
  }

  Record lease() {
    std::lock_guard<std::mutex> lock(mu_);
    return take_slot();
  }

  void give_back(const Record& r) noexcept {
    try {
      std::lock_guard<std::mutex> lock(mu_);
      if (!slabs_.empty()) free_.push_back(r.words);
    } catch (...) {  // no memory for the list: this one stays out of it
    }
  }

  // The record of calls made with the context on `s`, and the one that all its captured calls share: on which
  // stream a graph runs is not known when it is captured.
  Record of_stream(cudaStream_t s) {
    static thread_local char thread;  // the per-thread default stream is another one in each thread
    std::lock_guard<std::mutex> lock(mu_);
    Record& r = streams_[s == cudaStreamPerThread ? static_cast<const void*>(&thread) : s];
    if (!r.words) r = take_slot();
    return r;
  }
  const Record& captured() const { return captured_; }

 private:
  static constexpr size_t SLAB = 1024, QUARANTINE = 512;

  Record take_slot() {
    if (free_.size() <= QUARANTINE) add_slab();
    Record r;
    r.words = free_.front();
    free_.pop_front();
    if (++last_id_ == 0) ++last_id_;
    r.id = last_id_;
    return r;
  }

  void add_slab() {
    DeviceGuard g(ctx_->device);
    // allocating must not disturb a capture that is under way in this thread
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    PXC_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
    uint32_t* s = nullptr;
    const cudaError_t e = cudaHostAlloc(&s, SLAB * FAULT_WORDS * sizeof(uint32_t), cudaHostAllocPortable);
    PXC_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
    PXC_CUDA(e);
    slabs_.push_back(s);
    std::memset(s, 0, SLAB * FAULT_WORDS * sizeof(uint32_t));
    for (size_t i = 0; i < SLAB; ++i) free_.push_back(s + i * FAULT_WORDS);
    if (!captured_.words) captured_ = take_slot();
  }

  pxc_ctx* ctx_;
  std::mutex mu_;
  std::vector<uint32_t*> slabs_;
  std::deque<uint32_t*> free_;
  std::unordered_map<const void*, Record> streams_;
  Record captured_;
  uint32_t last_id_ = 0;
};

// A record for one host call.
struct Leased {
  Reports& reports;
  const Record record;
  explicit Leased(Reports& r) : reports(r), record(r.lease()) {}
  ~Leased() { reports.give_back(record); }
};

}  // namespace bq
}  // namespace pxc

struct pxc_bq_session {
  std::shared_ptr<pxc::bq::Reports> reports;
  pxc::bq::Record record;
};
