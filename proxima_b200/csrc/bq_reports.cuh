// bq_reports.cuh — failures of block products that only the device sees, kept apart by caller.
//
// A caller has a record: two words of pinned host memory that its calls' kernels write, and an id that they
// write into them. Callers are those that name themselves by a number, the streams of calls made without one, and
// each host call. Ids are never used twice, so a kernel or graph that outlives its caller is not taken for
// another's, and the words stay allocated until the context goes. A record whose caller has gone is given out again
// late, behind at least QUARANTINE others, or never if a graph may hold its calls; what its work leaves is for
// whoever checks.
#pragma once

#include <deque>
#include <mutex>
#include <unordered_map>
#include <unordered_set>
#include <vector>

#include "common.cuh"

namespace pxc {
namespace bq {

// A word of a record each.
enum Fault : uint32_t { FAULT_OFFSETS = 0, FAULT_TIMEOUT = 1, FAULT_WORDS = 2 };

struct Record {
  uint32_t* words = nullptr;
  uint32_t id = 0;

  // Whether a failure of this kind is there; it is so once.
  bool taken(Fault f) const {
    uint32_t seen = __atomic_load_n(words + f, __ATOMIC_RELAXED);
    return seen == id && id != 0 &&
           __atomic_compare_exchange_n(words + f, &seen, 0u, false, __ATOMIC_RELAXED, __ATOMIC_RELAXED);
  }
  // Reports a failure, once. Of two kinds, the other stays for the next call.
  void take() const {
    for (const Fault f : {FAULT_TIMEOUT, FAULT_OFFSETS})
      if (taken(f)) raise(f);
  }
  [[noreturn]] static void raise(Fault f) {
    if (f == FAULT_TIMEOUT)
      throw make_failure(PXC_TIMEOUT, 0, 0, nullptr, "a device-side wait of a block product ran out");
    throw make_failure(PXC_CONFIGURATION, 0, 0, "offsets",
                       "a grouped product's offsets fell, left the rows, or did not fit the output");
  }
};

class Reports {
 public:
  explicit Reports(int device) : device_(device) { add_slab(); }
  ~Reports() {
    for (uint32_t* s : slabs_) cudaFreeHost(s);
  }
  Reports(const Reports&) = delete;
  Reports& operator=(const Reports&) = delete;

  Record lease() {
    std::lock_guard<std::mutex> lock(mu_);
    return take_slot();
  }

  void give_back(const Record& r) noexcept {
    try {
      std::lock_guard<std::mutex> lock(mu_);
      free_.push_back(Record{r.words, 0});
    } catch (...) {  // no memory for the list: this one stays out of it
    }
  }

  // The record of a caller's number. Without `make`, an empty one where no call has needed it yet.
  Record of_caller(uint64_t caller, bool make) {
    std::lock_guard<std::mutex> lock(mu_);
    const auto found = callers_.find(caller);
    if (found != callers_.end()) return found->second;
    if (!make) return Record{};
    Record& r = callers_[caller];
    return r = take_slot();
  }
  // The caller's graphs may run whenever, also once it has gone.
  void keep(uint64_t caller) {
    std::lock_guard<std::mutex> lock(mu_);
    kept_.insert(caller);
  }
  void forget(const uint64_t* callers, uint64_t count) {
    std::lock_guard<std::mutex> lock(mu_);
    for (uint64_t i = 0; i < count; ++i) {
      const auto found = callers_.find(callers[i]);
      if (found == callers_.end()) continue;
      if (kept_.erase(callers[i]))
        of_graphs_.push_back(found->second);
      else
        free_.push_back(found->second);
      callers_.erase(found);
    }
  }
  // Reports a failure that the work of a caller left who has gone.
  void take_left() {
    std::lock_guard<std::mutex> lock(mu_);
    for (const Record& r : free_) r.take();
    for (const Record& r : of_graphs_) r.take();
    for (const Fault f : {FAULT_TIMEOUT, FAULT_OFFSETS})
      if (left_[f]) {
        left_[f] = false;
        Record::raise(f);
      }
  }

  // The record of calls without a number on `s`, and the one that all such captured calls share: on which
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
    Record r = free_.front();
    free_.pop_front();
    for (const Fault f : {FAULT_TIMEOUT, FAULT_OFFSETS}) left_[f] = r.taken(f) || left_[f];
    if (++last_id_ == 0) ++last_id_;
    r.id = last_id_;
    return r;
  }

  void add_slab() {
    DeviceGuard g(device_);
    // allocating must not disturb a capture that is under way in this thread
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    PXC_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
    uint32_t* s = nullptr;
    const cudaError_t e = cudaHostAlloc(&s, SLAB * FAULT_WORDS * sizeof(uint32_t), cudaHostAllocPortable);
    PXC_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
    PXC_CUDA(e);
    slabs_.push_back(s);
    std::memset(s, 0, SLAB * FAULT_WORDS * sizeof(uint32_t));
    for (size_t i = 0; i < SLAB; ++i) free_.push_back(Record{s + i * FAULT_WORDS, 0});
    if (!captured_.words) captured_ = take_slot();
  }

  const int device_;
  std::mutex mu_;
  std::vector<uint32_t*> slabs_;
  std::deque<Record> free_;  // with the ids of callers who have gone
  bool left_[FAULT_WORDS] = {};  // failures found in a record that was given out again
  std::unordered_map<uint64_t, Record> callers_;
  std::unordered_set<uint64_t> kept_;  // those of them that a graph may hold calls of
  std::vector<Record> of_graphs_;      // and the records of such callers who have gone
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
