// What the decode kernel of queries that share rows leaves for its merge kernel: one record for every item that was cut. Plain C++,
// so that the host can try which records the merge takes.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define B200KV_HOST_DEVICE __host__ __device__
#else
#define B200KV_HOST_DEVICE
#endif

namespace b200kv {

constexpr int32_t kMergeParts = 128;  // of an item, at most: no fewer than there are runs

struct alignas(16) MergeRecord {
  int32_t q0, q1;       // the item's queries, q1 < 0: a query alone; q0 < 0: nothing to merge
  int32_t first, last;  // the runs that began and that finished it
};

// Whether the record at `entry` asks for a merge that stays inside the call's arrays. A run that gave up on a wait does not write
// its items' records, and the workspace may hold anything there; what has been written always holds. Records are listed by the
// item's first query (by_query) or by the run that finished it.
B200KV_HOST_DEVICE inline bool MergeHolds(const MergeRecord& r, int32_t entry, bool by_query, int32_t batch, int32_t runs) {
  return r.q0 >= 0 && r.q0 < batch && (r.q1 < 0 || (r.q1 == r.q0 + 1 && r.q1 < batch)) && r.first >= 0 && r.first < r.last && r.last < runs &&
         (by_query ? r.q0 : r.last) == entry;
}

}  // namespace b200kv
