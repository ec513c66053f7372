// Decode attention of queries that share rows of the cache, on tcgen05 tensor cores (sm_100a), 64 heads x (512 + 64).
//
// Sequences forked from one prompt, the draft tokens of a step and the tokens of a prompt's chunk attend over the same rows.
// With 64 heads a row of 1,152 bytes is worth 139,264 operations a query: from two queries on the tensor cores are the bound and
// not HBM, so the work is arranged around them. Two queries (128 rows of S) and a pair of CTAs belong together:
//
//   S   [128 rows x 64 tokens]    each CTA for ITS 64 of a step's 128 tokens:  Q (A) x K^T (B), M = 128 N = 64, 36 k-steps;
//   P   = exp2(S * scale * log2e - m), bf16, written to shared memory and copied into the other CTA's;
//   O   [128 rows x 256 columns]  each CTA for ITS half of the 512 value columns, over all 128 tokens: P (A) x V (B), M = 128
//                                 N = 256, 8 k-steps.
//
// So each of the 128 x 512 sums lives in one CTA's tensor memory (a whole O would fill it and leave no room for S), nothing is
// computed twice, every MMA has M = 128, and the tokens' rows that a CTA takes in are its own 64 x 576 and the other's
// 64 x 256. Q does not fit beside them in shared memory: two thirds of it lie in tensor memory as the A operand, which also
// halves what those MMAs read of shared memory. Tensor memory: O 256 columns, S 64, Q 192: all 512.
//
// The two CTAs keep one running maximum: each sends its 128 rows' maxima over its tokens to the other before it exponentiates
// (one asynchronous 4-byte store a thread), and both come to the same reference. As in the other kernels O is rescaled only when
// the maximum grows by more than 2^8. The tensor cores take P in bf16, each weight off by at most 2^-8 of itself: the only rounding
// below fp32 before the result's own (sums and the log-sum-exp take the fp32 weights).
//
// The list of work. A pair of queries is an item of n steps: first the tokens that both share (or a prefix of them: the tokens
// of one sequence each attend up to themselves), then the first query's own tokens, then the second's, all into the same
// accumulators; in the latter, only that query's 64 lanes of O are touched. All items' steps form one flat list, cut into one run
// per CTA pair by cost; a run's first and last item may be cut, and then leave fp32 partials (m, l, O) in the workspace which
// the second kernel merges. A tile of tokens that is complete for one of the two queries only is two steps, one per query,
// so that a NaN or an infinity in a row behind a query's end never meets that query's weights (0 x NaN).
//
// Warps 0-3: softmax and epilogue (thread = row), 4: T and V, 5: QK, 6: PV, 7: Q and W. Every wait is bounded; the CTAs of a pair
// leave together through the cluster barrier.
//
// What bounds it. The matrix instructions of a step take 2,365 cycles (measured alone: 1,354 and 1,032 for S and O; neither tiles
// arriving at 54 bytes a cycle nor shared-memory stores slow them down). A step takes 3,100 to 3,500: S needs T, whose one buffer is
// filled anew every step, and the softmax of a step (2,400 cycles with the exchange of maxima) stands between its S and its O. Another
// item costs 2.5 steps more, a call 4.5 us until S comes for the first time, 2.3 us for partials at the rate at which an SM can
// write, and 7 us for the merge. 128 sequences behind 8,192 common tokens: 134 us (1,120 TFLOP/s), 157 to 160 us when they follow one another
// for long: the GPU is at its power limit then, with the clock at 1.65 GHz.
#include <cuda.h>

#include <climits>

#include "common.cuh"
#include "mla_tc_common.cuh"
#include "shared_merge_record.h"
#include "sm100_ptx.cuh"

namespace b200kv {

int32_t ValidatePoolView(const b200kv_pool_view* pool);
int32_t SimtSplitCount(int32_t batch, int32_t sms);
size_t SimtWorkspaceBytes(int32_t batch, int32_t heads, int32_t sms);
size_t TcWorkspaceBytes(int32_t n_ctas);
int32_t GetRowMap(const void* base, int64_t stride, int64_t rows, int32_t width, int32_t box_rows, CUtensorMap* out);
int32_t GetSlabMap(const void* base, int64_t stride, int64_t rows, int32_t slabs, CUtensorMap* out);
int32_t GetQSlabMap(const void* base, int64_t head_stride, int64_t seq_stride, int32_t batch, int32_t heads, int32_t slabs,
                    CUtensorMap* out);

namespace {

using namespace mla;

constexpr int kThreads = 256;
constexpr int kRows = 2 * kHeads;   // two queries
constexpr int kStep = 2 * kTile;    // tokens of a step: a tile for each CTA of the pair
constexpr int kHalf = kLatent / 2;  // value columns of a CTA
// K slabs of 64 columns: those of the CTA's own half of the value columns ("V", four), the other four and the rope ("T", five).
// Q's slabs in the same order: T0, T1 and V0-V3 in tensor memory, T2, T3 and the rope in shared memory.
constexpr int kTSlabs = 5, kVSlabs = 4, kQSmemSlabs = 3, kQTmemSlabs = 6;
constexpr int kQSlab = kRows * 128;  // 16,384
constexpr uint32_t kColO = 0, kColS = 256, kColQ = 320;
static_assert(kColQ + kQTmemSlabs * 32 == kTmemCols, "tensor memory is full");

// Shared memory (offsets from a 1024-byte aligned base).
constexpr int kOffQ = 0;
constexpr int kOffT = kOffQ + kQSmemSlabs * kQSlab;
constexpr int kOffV = kOffT + kTSlabs * kSlabBytes;           // two sets: PV of a step reads one while the next step's QK reads the other
constexpr int kOffW = kOffV + 2 * kVSlabs * kSlabBytes;       // the other CTA's tokens, this CTA's columns
constexpr int kOffP = kOffW + kVSlabs * kSlabBytes;           // weights of this CTA's tokens
constexpr int kPBytes = kRows * 128;
constexpr int kOffPeerP = kOffP + kPBytes;                    // weights of the other CTA's tokens
constexpr int kOffMisc = kOffPeerP + kPBytes;
constexpr int kMiscBytes = 4096;
// An item's slabs of Q for tensor memory come two at a time, through buffers that hold nothing then: V's set of the item's first
// step, T, and V's set again; for a run's first item, whose tiles come at the same time, V's second set, W and both buffers of weights.
constexpr int kRounds = 3;
static_assert(2 * kRounds == kQTmemSlabs && 2 * kQSlab <= kVSlabs * kSlabBytes && 2 * kQSlab <= 2 * kPBytes && kOffPeerP == kOffP + kPBytes);
__device__ __forceinline__ int StageOffset(int round, int seg, int set) {
  if (seg == 0) return round == 0 ? kOffV + kVSlabs * kSlabBytes : round == 1 ? kOffW : kOffP;
  return round == 1 ? kOffT : kOffV + set * kVSlabs * kSlabBytes;
}
constexpr int kSmemBytes = kOffMisc + kMiscBytes + 1024;
static_assert(kSmemBytes <= 232448, "shared memory budget exceeded");

struct Item {
  int q0, q1;        // q1 < 0: a query alone
  int row0, row1;    // their table rows
  int len0, len1;
  int lim0, lim1;    // tokens of the common part that each query attends over
  int own;           // where the own tokens begin
  int split;         // common tile that is two steps, or -1
  int common, own0, own1;  // steps
  __device__ __forceinline__ int steps() const { return common + own0 + own1; }
};

constexpr int kListed = 32;  // a run of up to so many items finds them in shared memory

struct Misc {
  uint64_t t_full[2], t_empty[2];  // T2, T3 and the rope; T0 and T1
  uint64_t v_full[2], v_empty[2];
  uint64_t w_full, w_empty;    // w_empty: PV of the step is complete
  uint64_t q_full, q_empty;    // the slabs in shared memory
  uint64_t qt_full;            // the slabs in tensor memory
  uint64_t stage_full[kRounds], stage_empty[kRounds];  // and on their way there
  uint64_t s_full, s_empty;
  uint64_t p_full;             // own weights written, rows behind the end zeroed
  uint64_t peer_p_full;        // the other CTA's weights have landed
  uint64_t p_empty;            // PV has read this CTA's weights
  uint64_t p_sent;             // and their copy has landed in the other CTA
  uint64_t peer_p_empty;       // the other CTA's PV has read the copy it holds of them
  uint64_t o_empty;
  uint64_t max_full[2][kSoftmaxWarps];
  uint64_t drain[2];
  uint32_t tmem_base;
  int32_t abort_flag;
  int32_t start_step;  // in the run's first item
  int32_t began_in;    // the run that item began in
  long long start_ordinal, end_ordinal;  // the run's items
  long long flat_lo, flat_hi;
  longlong2 scan[kThreads / 32];
  float peer_max[2][kRows];
  Item items[kListed];  // by ordinal % kListed; a run of more than kListed items reads SharedParams::items
};
static_assert(sizeof(Misc) <= kMiscBytes, "Misc does not fit its reservation");

struct SharedParams {
  const int32_t* block_table;
  int64_t max_blocks;
  int64_t table_rows;
  const int32_t* table_index;
  const int32_t* kv_len;
  const int32_t* leader;
  const int32_t* shared_len;
  int64_t pool_rows;
  int32_t batch;
  int32_t block_size;
  int32_t longest;  // a token more than a table row holds: a longer kv_len is cut there, at its first missing block
  int32_t stable_tables;
  float scale_log2;
  double natural;  // scale / scale_log2: from the kernels' log2 domain back to natural logarithms
  __nv_bfloat16* out;
  float* lse;
  // Partials: slot 2c of run c is an item it continues, slot 2c + 1 one it begins and does not finish. O as [slot][128 column
  // quads][128 rows][4 columns]: an epilogue thread owns a row, and a warp's stores are 512 contiguous bytes.
  float4* ws_o;
  float* ws_m;  // [slot][128], log2 domain
  float* ws_l;
  Item* items;   // [batch]: the items, in order (those of a run are written by the run's CTAs)
  // What there is to merge. By the item's first query where the batch has no more queries than there are runs, else by the run that
  // finished it.
  MergeRecord* merges;
  int32_t merges_by_query;
  int32_t runs;
  int32_t* status;
};

__device__ __forceinline__ MergeRecord NothingToMerge() { return {-1, -1, 0, 0}; }

// ---- the list of work -------------------------------------------------------------------------------------------------
// Query b is the second of a pair if the one before it has the same leader and stands at an even distance from it. Whatever the
// arrays hold, every query belongs to exactly one item.
__device__ __forceinline__ int StepsOf(int tokens) { return tokens > 0 ? (tokens - 1) / kStep + 1 : 0; }

__device__ __forceinline__ Item MakeItem(int q0, int q1, int row0, int row1, int len0, int len1, int shared0, int shared1) {
  Item it;
  it.q0 = q0;
  it.q1 = q1;
  it.row0 = row0;
  it.row1 = row1;
  it.len0 = max(len0, 0);
  it.len1 = q1 >= 0 ? max(len1, 0) : 0;
  it.split = -1;
  it.own0 = it.own1 = 0;
  it.own = 0;
  if (q1 < 0) {
    it.lim0 = it.len0;
    it.lim1 = 0;
    it.common = StepsOf(it.len0);
    return it;
  }
  const int shared = max(min(shared0, shared1), 0);
  it.own = shared & ~(kTile - 1);  // (a tile is 64 consecutive rows of a block)
  it.lim0 = it.len0 <= shared ? it.len0 : it.own;
  it.lim1 = it.len1 <= shared ? it.len1 : it.own;
  const int less = min(it.lim0, it.lim1);
  it.common = StepsOf(max(it.lim0, it.lim1));
  if (it.lim0 != it.lim1 && (less & (kStep - 1)) != 0) {
    it.split = less / kStep;
    ++it.common;
  }
  if (it.len0 > shared) it.own0 = StepsOf(it.len0 - it.own);
  if (it.len1 > shared) it.own1 = StepsOf(it.len1 - it.own);
  return it;
}

// The item that begins with query b, without steps if b is the second of a pair. The loads go out together.
__device__ __forceinline__ Item ItemAt(const SharedParams& p, int b, bool* second) {
  const int prev = max(b - 1, 0), next = min(b + 1, p.batch - 1);
  const int lead_prev = p.leader[prev], lead = p.leader[b], lead_next = p.leader[next];
  const int len0 = min(p.kv_len[b], p.longest), len1 = min(p.kv_len[next], p.longest), shared0 = p.shared_len[b], shared1 = p.shared_len[next];
  int row0 = b, row1 = next;
  if (p.table_index != nullptr) {
    row0 = p.table_index[b];
    row1 = p.table_index[next];
  }
  *second = b > 0 && lead == lead_prev && ((static_cast<unsigned>(prev) - static_cast<unsigned>(lead)) & 1u) == 0;
  const bool pair = next > b && lead == lead_next && ((static_cast<unsigned>(b) - static_cast<unsigned>(lead)) & 1u) == 0;
  return MakeItem(b, pair ? next : -1, row0, row1, *second ? 0 : len0, pair && !*second ? len1 : 0, shared0, shared1);
}

struct Step {
  int query;   // whose table row
  int row;     // and which
  int token;   // first token
  int valid;   // 1 .. 128 tokens
  int active;  // bit 0: the first query's rows, bit 1: the second's
};

__device__ __forceinline__ Step StepAt(const Item& it, int s) {
  Step st;
  if (s < it.common) {
    int tile = s;
    st.query = it.q0;
    st.row = it.row0;
    if (it.split >= 0 && s > it.split) --tile;
    st.token = tile * kStep;
    const int in0 = it.lim0 - st.token, in1 = it.lim1 - st.token;
    if (it.split >= 0 && tile == it.split) {  // first the query that ends in this tile, then the other
      const bool first_ends = it.lim0 < it.lim1;
      st.active = (s == it.split) == first_ends ? 1 : 2;
    } else {
      st.active = (in0 > 0 ? 1 : 0) | (in1 > 0 ? 2 : 0);
    }
    st.valid = min(kStep, st.active == 1 ? in0 : st.active == 2 ? in1 : min(in0, in1));
    return st;
  }
  s -= it.common;
  const bool second = s >= it.own0;
  if (second) s -= it.own0;
  st.query = second ? it.q1 : it.q0;
  st.row = second ? it.row1 : it.row0;
  st.token = it.own + s * kStep;
  st.active = second ? 2 : 1;
  st.valid = min(kStep, (second ? it.len1 : it.len0) - st.token);
  return st;
}

// The cut: a step costs 2, entering another item in mid-run 8 more (Q is loaded anew and the accumulators are drained). Step x
// of the flat list, of the item with ordinal s, stands at cost position 2x + 8s; run c takes the positions
// [ceil(c C / G), ceil((c + 1) C / G)).
struct Cut {
  long long total_cost;
  long long runs;
  static constexpr long long kStepCost = 2, kEnterCost = 8;
  __device__ static long long Pos(long long x, long long s) { return kStepCost * x + kEnterCost * s; }
  // Non-negative quotient; the 32-bit division is several times shorter and covers every realistic size.
  __device__ static long long Div(long long a, long long b) {
    if (((a | b) >> 32) == 0) return static_cast<long long>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b));
    return a / b;
  }
  __device__ long long First(long long c) const { return Div(c * total_cost + runs - 1, runs); }
  __device__ long long RunOf(long long pos) const { return Div(pos * runs, total_cost); }
};

// The items of this run, one after the other. Every role runs the same walk.
struct Walk {
  const Item* items;
  uint32_t at, mask;
  int step;
  long long remaining;
  __device__ Walk(const SharedParams& p, const Misc* misc) : step(misc->start_step), remaining(misc->flat_hi - misc->flat_lo) {
    const bool listed = misc->end_ordinal - misc->start_ordinal <= kListed;
    items = listed ? misc->items : p.items;
    mask = listed ? kListed - 1 : 0xffffffffu;
    at = static_cast<uint32_t>(misc->start_ordinal);
  }
  __device__ __forceinline__ bool Next(Item* item, int* lo, int* hi) {
    if (remaining <= 0) return false;
    *item = items[at++ & mask];
    *lo = step;
    *hi = static_cast<int>(min(remaining, static_cast<long long>(item->steps() - step))) + step;
    remaining -= *hi - step;
    step = 0;
    return true;
  }
};

// A bounded wait by all lanes of a warp together, behind an inline probe. It spins: a parked warp resumes some 500 cycles after
// its phase, a fifth of a step.
__device__ __forceinline__ bool WarpWait(uint32_t bar, uint32_t parity, Misc* misc, int32_t* status, int site) {
  if (__all_sync(0xffffffffu, ptx::MbarTestWait(bar, parity))) return true;
  return __all_sync(0xffffffffu, BoundedSpin(bar, parity, misc, status, site));
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    MlaDecodeSharedKernel(const __grid_constant__ CUtensorMap latent_map, const __grid_constant__ CUtensorMap t_map,
                          const __grid_constant__ CUtensorMap rope_map, const __grid_constant__ CUtensorMap q_map,
                          const __grid_constant__ CUtensorMap q_rope_map, const __grid_constant__ SharedParams p) {
  extern __shared__ unsigned char smem_dyn[];
  const uint32_t raw = ptx::SmemAddr(smem_dyn);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char* smem = smem_dyn + (base - raw);
  Misc* misc = reinterpret_cast<Misc*>(smem + kOffMisc);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1;
  const int run = blockIdx.x >> 1;
  const int runs = gridDim.x >> 1;
  auto bar = [&](const uint64_t* b) { return ptx::SmemAddr(b); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      ptx::MbarInit(bar(&misc->t_full[s]), 1);
      ptx::MbarInit(bar(&misc->t_empty[s]), 1);
      ptx::MbarInit(bar(&misc->v_full[s]), 1);
      ptx::MbarInit(bar(&misc->v_empty[s]), 1);
      ptx::MbarInit(bar(&misc->drain[s]), 1);
      for (int w = 0; w < kSoftmaxWarps; ++w) ptx::MbarInit(bar(&misc->max_full[s][w]), 1);
    }
    ptx::MbarInit(bar(&misc->w_full), 1);
    ptx::MbarInit(bar(&misc->w_empty), 1);
    ptx::MbarInit(bar(&misc->q_full), 1);
    ptx::MbarInit(bar(&misc->q_empty), 1);
    ptx::MbarInit(bar(&misc->qt_full), kSoftmaxWarps);
    for (int r = 0; r < kRounds; ++r) {
      ptx::MbarInit(bar(&misc->stage_full[r]), 1);
      ptx::MbarInit(bar(&misc->stage_empty[r]), kSoftmaxWarps);
    }
    ptx::MbarInit(bar(&misc->s_full), 1);
    ptx::MbarInit(bar(&misc->s_empty), kSoftmaxWarps);
    ptx::MbarInit(bar(&misc->p_full), kSoftmaxWarps);
    ptx::MbarInit(bar(&misc->peer_p_full), 1);
    ptx::MbarInit(bar(&misc->p_empty), 1);
    ptx::MbarInit(bar(&misc->p_sent), 1);
    ptx::MbarInit(bar(&misc->peer_p_empty), 1);
    ptx::MbarInit(bar(&misc->o_empty), kSoftmaxWarps);
    misc->abort_flag = 0;
    misc->start_step = 0;
    misc->began_in = 0;
    misc->start_ordinal = misc->end_ordinal = 0;
    misc->flat_lo = LLONG_MAX;  // (a run between two items has none)
    misc->flat_hi = 0;
    ptx::FenceBarrierInit();
    ptx::PrefetchTensorMap(&latent_map);
    ptx::PrefetchTensorMap(&t_map);
    ptx::PrefetchTensorMap(&rope_map);
    ptx::PrefetchTensorMap(&q_map);
    ptx::PrefetchTensorMap(&q_rope_map);
  }
  if (warp == 5) {
    ptx::TmemAlloc(ptx::SmemAddr(&misc->tmem_base), kTmemCols);
    ptx::TmemRelinquish();
  }
  __syncwarp();
  ptx::ClusterArrive();  // (the barriers are ready: waited for before the peer's are touched)
  if (p.stable_tables == 0) GridDependencyWait();

  // ---- this run of the list: totals, then the first step at or after the run's first cost position and the next run's ------
  // Each thread has a stretch of the queries: sums over it, one scan over the threads, and those threads that have items of this
  // run go over their stretch again.
  const int each = (p.batch - 1) / kThreads + 1;
  const int stretch = min(static_cast<int>(threadIdx.x) * each, p.batch), stretch_end = min(stretch + each, p.batch);
  bool any_empty = false;
  {
    Item mine;
    long long n = 0;
    int n_items = 0;
#pragma unroll 2
    for (int b = stretch; b < stretch_end; ++b) {
      bool second;
      mine = ItemAt(p, b, &second);
      const int steps = mine.steps();
      n += steps;
      n_items += steps > 0 ? 1 : 0;
      any_empty |= steps == 0 && !second;
    }
    long long incl = n;
    int incl_items = n_items;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, incl, off);
      const int up_items = __shfl_up_sync(0xffffffffu, incl_items, off);
      if (lane >= off) {
        incl += up;
        incl_items += up_items;
      }
    }
    if (lane == 31) misc->scan[warp] = make_longlong2(incl, incl_items);
    __syncthreads();
    long long total = 0, total_items = 0, before = incl - n, before_items = incl_items - n_items;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      const longlong2 of = misc->scan[w];
      before += w < warp ? of.x : 0;
      before_items += w < warp ? of.y : 0;
      total += of.x;
      total_items += of.y;
    }
    const long long cost = Cut::Pos(total, total_items > 0 ? total_items - 1 : 0);
    // No more runs than steps' cost: a run's share is at least a step's, so that none between two of an item's is empty. And no
    // more than pays: r runs take a step's 1.7 us times steps / r, and their parts cost the merge some 0.13 us times r / items
    // (two queries of 16,384 tokens: 41 runs 23.7 us, all 74 of them 27.5; from 8 queries of 8,192 on it is all of them).
    const long long paying = static_cast<long long>(sqrtf(13.0f * static_cast<float>(total) * static_cast<float>(total_items)));
    const Cut cut{cost, max(1ll, min(static_cast<long long>(runs), min(cost / Cut::kStepCost, paying)))};
    const long long k_lo = run < cut.runs ? cut.First(run) : cost, k_hi = run < cut.runs ? cut.First(run + 1) : cost;
    // The stretch's items, in order: f(item, its first step, its ordinal).
    auto each_item = [&](auto f) {
      long long first = before, s = before_items;
#pragma unroll 1
      for (int b = stretch; b < stretch_end; ++b) {
        if (each > 1) {  // (a stretch of one is still at hand)
          bool second;
          mine = ItemAt(p, b, &second);
        }
        const int steps = mine.steps();
        if (steps == 0) continue;
        f(mine, first, s);
        first += steps;
        ++s;
      }
    };
    const bool here = n_items > 0 && Cut::Pos(before + n - 1, before_items + n_items - 1) >= k_lo &&
                      (before_items == 0 || Cut::Pos(before - 1, before_items - 1) < k_hi);
    if (here) {
      each_item([&](const Item& item, long long first, long long s) {
        const long long first_pos = Cut::Pos(first, s), last_pos = Cut::Pos(first + item.steps() - 1, s);
        const long long last_before = Cut::Pos(first - 1, s - 1);  // the item before this one ends here
        auto at_or_after = [&](long long k) {                      // first step at or after cost position k, if it is in this item
          const long long x = (k - Cut::kEnterCost * s + 1) >> 1;
          return x > first ? x : first;
        };
        if (last_pos >= k_lo && first_pos < k_hi) {
          misc->items[s % kListed] = item;  // (of more than kListed none is read)
          if (s == 0 || last_before < k_lo) {
            const long long x = at_or_after(k_lo);
            misc->flat_lo = x;
            misc->start_step = static_cast<int>(x - first);
            misc->start_ordinal = s;
            misc->began_in = static_cast<int>(cut.RunOf(first_pos));
          }
          atomicMax(reinterpret_cast<unsigned long long*>(&misc->end_ordinal), static_cast<unsigned long long>(s + 1));
        }
        if (last_pos >= k_hi && (s == 0 || last_before < k_hi)) misc->flat_hi = at_or_after(k_hi);
      });
    }
    // Up to the last cost position and behind it: the end of the list.
    if (threadIdx.x == 0 && k_lo >= cost) misc->flat_lo = total;
    if (threadIdx.x == 0 && k_hi >= cost) misc->flat_hi = total;
    if (p.stable_tables != 0) GridDependencyWait();
    // A run of more than kListed items lists them in the workspace, only here, behind the wait: the kernel before may still read a
    // workspace that it shares with this call.
    if (p.batch > kListed) {
      __syncthreads();
      if (here && misc->end_ordinal - misc->start_ordinal > kListed) {
        each_item([&](const Item& item, long long, long long s) {
          if (s >= misc->start_ordinal && s < misc->end_ordinal) p.items[s] = item;
        });
      }
    }
  }
  // (the merge kernel's CTAs may come from here on; they read only what this kernel leaves, and wait for its end)
  GridDependencyTrigger();
  ptx::TcFenceBeforeSync();
  any_empty = __syncthreads_or(any_empty) != 0;
  ptx::TcFenceAfterSync();
  if (threadIdx.x == 0 && rank == 0 && p.merges_by_query == 0) p.merges[run] = NothingToMerge();
  if (any_empty) {  // queries that attend over nothing, alone or with one like them
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
      Item it;
      bool second;
      int at = b;
#pragma unroll 1
      do {  // (the second of a pair: the pair's)
        it = ItemAt(p, at--, &second);
      } while (second);
      if (it.steps() > 0) continue;
      if (threadIdx.x == 0 && p.merges_by_query != 0) p.merges[b] = NothingToMerge();
      int4* out = reinterpret_cast<int4*>(p.out + static_cast<int64_t>(b) * kHeads * kLatent);
      for (int i = threadIdx.x; i < kHeads * kLatent / 8; i += kThreads) out[i] = make_int4(0, 0, 0, 0);
      if (p.lse != nullptr && threadIdx.x < kHeads) p.lse[static_cast<int64_t>(b) * kHeads + threadIdx.x] = -INFINITY;
    }
  }

  const uint32_t tmem = misc->tmem_base;
  bool ok = true;

  if (warp == 4 || warp == 7) {
    // ======================= loads ============================================================================
    // Warp 4 brings a step's T and V, warp 7 an item's Q and a step's W, which waits for the PV before: in one warp that wait would
    // hold the next step's T back.
    // Pool row of a tile, through the block table; the row behind the pool (which loads as zeros) for a tile without tokens and
    // for a bad entry, which is recorded.
    auto tile_row = [&](const Step& st, int tile) -> int32_t {
      const int in_step = tile * kTile;
      if (in_step >= st.valid) return static_cast<int32_t>(p.pool_rows);
      const int token = st.token + in_step;
      const int64_t column = token / p.block_size;
      const bool inside = st.row >= 0 && st.row < p.table_rows && column < p.max_blocks;
      const int64_t block = inside ? p.block_table[st.row * p.max_blocks + column] : -1;
      const int64_t row = block * p.block_size + token % p.block_size;
      if (block < 0 || row + kTile > p.pool_rows) {
        RecordError(p.status, B200KV_DEV_BAD_BLOCK, st.query, static_cast<int32_t>(column), static_cast<int32_t>(block));
        return static_cast<int32_t>(p.pool_rows);
      }
      return static_cast<int32_t>(row);
    };
    // Warp 4: lane 0 T2 and T3, lane 1 the rope slab, lane 2 T0 and T1, lane 3 V. Warp 7: lane 0 the other tile's slabs of V's
    // columns. Several slabs are one box: a warp issues a load only every 170 cycles or so.
    const bool is_w = warp == 7, is_t = !is_w && lane < 3;
    const bool loader = lane < (is_w ? 1 : 4);
    const bool is_rope = is_t && lane == 1;
    const int group = lane == 2 ? 1 : 0;  // of T
    const int first_slab = is_t ? kVSlabs * (1 - rank) + (group == 0 ? 2 : 0) : kVSlabs * rank;
    const bool announces = loader && !is_rope;
    const uint32_t announced = (!is_t ? kVSlabs : group == 0 ? 3 : 2) * kSlabBytes;
    const uint32_t dst0 = base + (is_t ? kOffT : is_w ? kOffW : kOffV) + (is_rope ? 4 : is_t && group == 0 ? 2 : 0) * kSlabBytes;
    const CUtensorMap* const map = is_t ? &t_map : &latent_map;
    Walk walk(p, misc);
    Item item;
    int lo, hi;
    int g = 0, seg = 0;
    while (ok && walk.Next(&item, &lo, &hi)) {
      // Once the item before has had its last S, Q's old slabs, T and what was staged have been read (the waits for stage_empty
      // below take an earlier phase for the item's otherwise); V's set was the PV's before the last.
      if (seg > 0) ok = WarpWait(bar(&misc->q_empty), (seg - 1) & 1, misc, p.status, 11);
      if (!ok) break;
      if (is_w) {
        if (g > 1) ok = WarpWait(bar(&misc->v_empty[g & 1]), ((g >> 1) & 1) ^ 1, misc, p.status, 12);
        if (!ok) break;
        // A box is 64 heads of both queries (alone, the first brings its neighbour, or zeros, whose rows no one reads).
        auto staged = [&](int round) {
          const uint32_t full = bar(&misc->stage_full[round]);
          ptx::MbarArriveExpectTx(full, 2 * kQSlab);
          ptx::TmaLoad4D(base + StageOffset(round, seg, g & 1), &q_map, 0, 0, item.q0, round == 0 ? kVSlabs * (1 - rank) : kVSlabs * rank + 2 * round - 2, full);
        };
        if (lane == 0) {
          staged(0);
          staged(1);
          if (seg == 0) staged(2);
          const uint32_t full = bar(&misc->q_full);  // the slabs in shared memory: T2, T3, rope
          ptx::MbarArriveExpectTx(full, kQSmemSlabs * kQSlab);
          ptx::TmaLoad4D(base + kOffQ, &q_map, 0, 0, item.q0, kVSlabs * (1 - rank) + 2, full);
          ptx::TmaLoad4D(base + kOffQ + 2 * kQSlab, &q_rope_map, 0, 0, item.q0, kLatent / 64, full);
        }
        __syncwarp();
        if (seg > 0) {
          ok = WarpWait(bar(&misc->stage_empty[0]), seg & 1, misc, p.status, 13);
          if (!ok) break;
          if (lane == 0) staged(2);
          __syncwarp();
        }
      }
      for (int s = lo; s < hi; ++s, ++g) {
        const int32_t row = tile_row(StepAt(item, s), is_w ? 1 - rank : rank);
        const int set = g & 1;
        const uint32_t full = is_t ? bar(&misc->t_full[group]) : is_w ? bar(&misc->w_full) : bar(&misc->v_full[set]);
        uint32_t empty = is_t ? bar(&misc->t_empty[group]) : is_w ? bar(&misc->w_empty) : bar(&misc->v_empty[set]);
        const uint32_t dst = dst0 + (!is_t && !is_w ? set * kVSlabs * kSlabBytes : 0);
        // Phase of the buffer's last use: T and W are used every step, a V set every other. An item's first tiles come behind the
        // slabs of Q that have passed through their buffers; in a run's first item these are W's first and V's second.
        const bool every = is_t || is_w;
        const bool first_use = g == 0 && !is_w;
        uint32_t parity = every ? (g & 1) ^ 1 : ((g >> 1) & 1) ^ 1;
        if (seg == 0 ? (is_w ? g == 0 : !is_t && g == 1) : s == lo && !is_w) {
          empty = bar(&misc->stage_empty[every ? 1 : seg == 0 ? 0 : 2]);
          parity = seg & 1;
        }
        // The warp polls together; a lane issues its slab the moment its buffer has been given back.
        bool done = !loader;
        uint64_t start = 0;
        for (uint32_t it = 0;; ++it) {
          if (!done && (first_use || ptx::MbarTestWait(empty, parity))) {
            if (announces) ptx::MbarArriveExpectTx(full, announced);
            if (is_rope) {
              ptx::TmaLoad2D(dst, &rope_map, 0, row, full);
            } else {
              ptx::TmaLoad3D(dst, map, 0, row, first_slab, full);
            }
            done = true;
          }
          if (__all_sync(0xffffffffu, done)) break;
          if ((it & 1023u) == 1023u) {
            const uint64_t now = ptx::GlobalTimerNs();
            if (start == 0) start = now;
            if (Aborting(misc) || now - start > 1000000000ull) {
              if (!Aborting(misc) && lane == 0) RaiseTimeout(misc, p.status, 10, parity);
              ok = false;
              break;
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      ++seg;
    }
  } else if (warp == 5) {
    // ======================= QK ================================================================================
    constexpr uint32_t kIdesc = ptx::InstrDescBf16(kRows, kTile, 0, 0);
    const uint64_t q_desc = ptx::SmemDescSw128(base + kOffQ, 16, 1024);
    const uint64_t t_desc = ptx::SmemDescSw128(base + kOffT, 16, 1024);
    const uint64_t v_desc0 = ptx::SmemDescSw128(base + kOffV, 16, 1024);
    const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t d = tmem_u + kColS;
    Walk walk(p, misc);
    Item item;
    int lo, hi;
    int g = 0, seg = 0;
    while (ok) {
      const int have = walk.Next(&item, &lo, &hi) ? 1 : 0;
      if (__shfl_sync(0xffffffffu, have, 0) == 0) break;
      const int n = __shfl_sync(0xffffffffu, hi - lo, 0);
      for (int i = 0; i < n && ok; ++i, ++g) {
        if (i == 0) {
          ok = WarpWait(bar(&misc->q_full), seg & 1, misc, p.status, 22);
        }
        if (ok && g > 0) ok = WarpWait(bar(&misc->s_empty), (g & 1) ^ 1, misc, p.status, 25);
        if (ok) ok = WarpWait(bar(&misc->t_full[0]), g & 1, misc, p.status, 24);
        if (!ok) break;
        ptx::TcFenceAfterSync();
        if (ptx::ElectOne()) {
#pragma unroll
          for (int k = 8; k < 4 * kTSlabs; ++k) {  // T2 and on, whose Q lies in shared memory
            const int slab = k >> 2, kk = k & 3;
            ptx::MmaF16SS(d, DescAt(q_desc, (slab - 2) * kQSlab + kk * 32), DescAt(t_desc, slab * kSlabBytes + kk * 32), kIdesc, k > 8 ? 1u : 0u);
          }
          ptx::TcCommit(bar(&misc->t_empty[0]));
        }
        __syncwarp();
        ok = WarpWait(bar(&misc->t_full[1]), g & 1, misc, p.status, 24);
        if (ok && i == 0) ok = WarpWait(bar(&misc->qt_full), seg & 1, misc, p.status, 23);
        if (!ok) break;
        ptx::TcFenceAfterSync();
        if (ptx::ElectOne()) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int slab = k >> 2, kk = k & 3;
            ptx::MmaF16TS(d, tmem_u + kColQ + slab * 32 + kk * 8, DescAt(t_desc, slab * kSlabBytes + kk * 32), kIdesc, 1u);
          }
          ptx::TcCommit(bar(&misc->t_empty[1]));
        }
        __syncwarp();
        const int set = __shfl_sync(0xffffffffu, g & 1, 0);
        const uint64_t v_desc = DescAt(v_desc0, set * kVSlabs * kSlabBytes);
        ok = WarpWait(bar(&misc->v_full[set]), (g >> 1) & 1, misc, p.status, 26);
        if (!ok) break;
        ptx::TcFenceAfterSync();
        if (ptx::ElectOne()) {
#pragma unroll
          for (int k = 0; k < 4 * kVSlabs; ++k) {
            const int slab = k >> 2, kk = k & 3;
            ptx::MmaF16TS(d, tmem_u + kColQ + (2 + slab) * 32 + kk * 8, DescAt(v_desc, slab * kSlabBytes + kk * 32), kIdesc, 1u);
          }
          ptx::TcCommit(bar(&misc->s_full));
          if (i == n - 1) ptx::TcCommit(bar(&misc->q_empty));
        }
      }
      ++seg;
    }
    if (ptx::ElectOne()) {  // nothing of this warp's may be in flight when tensor memory is freed
      ptx::TcCommit(bar(&misc->drain[0]));
      const uint64_t t0 = ptx::GlobalTimerNs();
      while (!ptx::MbarTryWait(bar(&misc->drain[0]), 0)) {
        if (ptx::GlobalTimerNs() - t0 > 200000000ull) break;
      }
    }
    __syncwarp();
  } else if (warp == 6) {
    // ======================= PV ================================================================================
    constexpr uint32_t kIdesc = ptx::InstrDescBf16(kRows, kHalf, 0, 1);
    const uint64_t p_desc = ptx::SmemDescSw128(base + kOffP, 16, 1024);  // K-major: row = row of P, 32 bytes a k-step
    const uint64_t peer_p_desc = DescAt(p_desc, kOffPeerP - kOffP);
    const uint64_t v_desc0 = ptx::SmemDescSw128(base + kOffV, kSlabBytes, 1024);  // MN-major B: next 64 columns a slab further
    const uint64_t w_desc = DescAt(v_desc0, kOffW - kOffV);
    const uint32_t peer_p_sent = ptx::MapToRank(bar(&misc->p_sent), rank ^ 1);
    ptx::ClusterWait();  // (the peer's barriers are touched from here on)
    const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
    Walk walk(p, misc);
    Item item;
    int lo, hi;
    int g = 0, seg = 0;
    while (ok) {
      const int have = walk.Next(&item, &lo, &hi) ? 1 : 0;
      if (__shfl_sync(0xffffffffu, have, 0) == 0) break;
      if (seg > 0) ok = WarpWait(bar(&misc->o_empty), (seg - 1) & 1, misc, p.status, 27);
      int started = 0;  // queries whose accumulators hold something
      for (int s = lo; s < hi && ok; ++s, ++g) {
        const int active = __shfl_sync(0xffffffffu, StepAt(item, s).active, 0);
        if (ptx::ElectOne()) ptx::MbarArriveExpectTx(bar(&misc->peer_p_full), kPBytes);
        ok = WarpWait(bar(&misc->p_full), g & 1, misc, p.status, 21);
        if (!ok) break;
        ptx::TcFenceAfterSync();
        const int set = __shfl_sync(0xffffffffu, g & 1, 0);
        const uint64_t v_desc = DescAt(v_desc0, set * kVSlabs * kSlabBytes);
        // Both queries' rows in one pass, or (one of them takes no part, or has begun and the other has not) a pass for each that
        // leaves the other's lanes alone. This CTA's tokens first: the other's weights are on their way meanwhile.
        const bool one_pass = active == 3 && (started == 0 || started == 3);
#pragma unroll
        for (int theirs = 0; theirs < 2; ++theirs) {
          if (theirs != 0) {
            ok = WarpWait(bar(&misc->peer_p_full), g & 1, misc, p.status, 29);
            if (!ok) break;
            if (ptx::ElectOne()) ptx::MbarArriveRemoteRelaxed(peer_p_sent);
            ok = WarpWait(bar(&misc->w_full), g & 1, misc, p.status, 28);
            if (!ok) break;
            ptx::TcFenceAfterSync();
          }
          const uint64_t weights = theirs != 0 ? peer_p_desc : p_desc, values = theirs != 0 ? w_desc : v_desc;
          if (one_pass) {
            const uint32_t keep = theirs != 0 || started != 0 ? 1u : 0u;
            if (ptx::ElectOne()) {
#pragma unroll
              for (int k = 0; k < kTile / 16; ++k) {
                ptx::MmaF16SS(tmem_u + kColO, DescAt(weights, k * 32), DescAt(values, k * 2048), kIdesc, k > 0 ? 1u : keep);
              }
            }
          } else {
#pragma unroll 1
            for (int q = 0; q < 2; ++q) {
              if ((active >> q & 1) == 0) continue;
              const uint32_t keep = theirs != 0 ? 1u : (started >> q) & 1;
              const uint32_t off_lo = q == 0 ? 0u : 0xffffffffu;
              if (ptx::ElectOne()) {
#pragma unroll
                for (int k = 0; k < kTile / 16; ++k) {
                  ptx::MmaF16SSLanes(tmem_u + kColO, DescAt(weights, k * 32), DescAt(values, k * 2048), kIdesc, off_lo, ~off_lo, k > 0 ? 1u : keep);
                }
              }
              __syncwarp();
            }
          }
          __syncwarp();
          if (ptx::ElectOne()) {
            if (theirs == 0) {
              ptx::TcCommit(bar(&misc->v_empty[set]));
              ptx::TcCommit(bar(&misc->p_empty));
            } else {
              ptx::TcCommit(bar(&misc->w_empty));
              ptx::TcCommitTo(bar(&misc->peer_p_empty), static_cast<uint16_t>(1u << (rank ^ 1)));
            }
          }
        }
        if (!ok) break;
        started |= active;
      }
      ++seg;
    }
    if (ptx::ElectOne()) {
      ptx::TcCommit(bar(&misc->drain[1]));
      const uint64_t t0 = ptx::GlobalTimerNs();
      while (!ptx::MbarTryWait(bar(&misc->drain[1]), 0)) {
        if (ptx::GlobalTimerNs() - t0 > 200000000ull) break;
      }
    }
    __syncwarp();
  } else if (warp < kSoftmaxWarps) {
    // ======================= softmax + epilogue: thread = row ====================================================
    const int row = threadIdx.x;
    const int which = row >> 6, head = row & (kHeads - 1);
    const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t peer = rank ^ 1;
    const uint32_t peer_max_at = ptx::MapToRank(ptx::SmemAddr(&misc->peer_max[0][row]), peer);
    const uint32_t peer_max_bar = ptx::MapToRank(bar(&misc->max_full[0][warp]), peer);
    const uint32_t p_row = base + kOffP + row * 128;
    const uint32_t p_warp = base + kOffP + warp * 32 * 128;
    const uint32_t peer_p_warp = ptx::MapToRank(base + kOffPeerP + warp * 32 * 128, peer);
    const uint32_t peer_p_bar = ptx::MapToRank(bar(&misc->peer_p_full), peer);
    Walk walk(p, misc);
    Item item;
    int lo, hi;
    int g = 0;
    int x = 0;  // exchanges with the peer
    // Sends a value to the peer's thread of the same row and returns that thread's. Slots and barriers alternate: the peer
    // sends its value of exchange x + 2 only after this thread's of x + 1, which this thread sends after it has read x.
    auto send = [&](float v) {
      const int slot = x & 1;
      if (lane == 0) ptx::MbarArriveExpectTx(bar(&misc->max_full[slot][warp]), 32 * 4);
      __syncwarp();
      ptx::StAsyncF32(peer_max_at + slot * kRows * 4, v, peer_max_bar + slot * kSoftmaxWarps * 8);
    };
    auto receive = [&]() -> float {
      const int slot = x & 1;
      ok = WarpWait(bar(&misc->max_full[slot][warp]), (x >> 1) & 1, misc, p.status, 33) && ok;
      ++x;
      return *reinterpret_cast<volatile float*>(&misc->peer_max[slot][row]);
    };
    // The warp's weights of step g - 1 may be overwritten: PV has read them, and so has the copy.
    auto weights_free = [&]() {
      if (g > 0) {
        ok = WarpWait(bar(&misc->p_empty), (g & 1) ^ 1, misc, p.status, 31) && WarpWait(bar(&misc->p_sent), (g & 1) ^ 1, misc, p.status, 38) && ok;
      }
    };
    // An item's rows of Q from where they have been brought into tensor memory, where a row is a lane: T0, T1, V0-V3. The item
    // before has had its last S, so no MMA reads the old ones. (Reads of Q by the threads themselves take two to three times as
    // long as this way through shared memory, 24 or 48 of them a thread.)
    int seg = 0;
    auto load_q = [&](int set) {
#pragma unroll 1
      for (int round = 0; round < kRounds; ++round) {
        ok = WarpWait(bar(&misc->stage_full[round]), seg & 1, misc, p.status, 44) && ok;
        const uint32_t at = base + StageOffset(round, seg, set) + row * 128;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t r[32];
#pragma unroll
          for (int c = 0; c < 8; ++c) ptx::LdShared128(at + k * kQSlab + ((c ^ (row & 7)) << 4), r[4 * c], r[4 * c + 1], r[4 * c + 2], r[4 * c + 3]);
          ptx::TmemSt32(tmem + lane_base + kColQ + (2 * round + k) * 32, r);
        }
        ptx::FenceProxyAsyncShared();
        __syncwarp();
        if (lane == 0) ptx::MbarArrive(bar(&misc->stage_empty[round]));
      }
      ptx::TmemWaitSt();
      ptx::TcFenceBeforeSync();
      __syncwarp();
      if (lane == 0) ptx::MbarArrive(bar(&misc->qt_full));
      ++seg;
    };
    bool have = false, continued = misc->start_step > 0;
    float m_run = kLowest, l_run = 0.0f;
    for (;;) {
      // The next item's Q first: its first S is then computed under this item's epilogue.
      Item next_item;
      int next_lo, next_hi;
      const bool more = walk.Next(&next_item, &next_lo, &next_hi);
      if (have) send(l_run);  // (the sum of this item's weights, received in its epilogue)
      if (more) load_q(g & 1);
      if (!have) ptx::ClusterWait();  // (the peer's barriers are touched from here on)
      if (have) {
        // ---- epilogue of the item ----
        const float l_all = l_run + receive();
        ok = WarpWait(bar(&misc->w_empty), (g & 1) ^ 1, misc, p.status, 32) && ok;
        weights_free();
        if (!ok) break;
        ptx::TcFenceAfterSync();
        const bool ends = hi == item.steps();
        const bool whole = lo == 0 && ends;
        const int slot = 2 * run + (lo == 0 ? 1 : 0);
        const int query = which == 0 ? item.q0 : item.q1;
        const bool nothing = l_all == 0.0f;  // no weights, and O may hold anything
        const float inv_l = nothing ? 0.0f : 1.0f / l_all;
        if (rank == 0) {
          if (row == 0 && ends) {
            if (p.merges_by_query != 0) {
              p.merges[item.q0] = continued ? MergeRecord{item.q0, item.q1, misc->began_in, run} : NothingToMerge();
              if (item.q1 >= 0) p.merges[item.q1] = NothingToMerge();
            } else if (continued) {
              p.merges[run] = MergeRecord{item.q0, item.q1, misc->began_in, run};
            }
          }
          if (!whole) {
            p.ws_m[slot * kRows + row] = m_run;
            p.ws_l[slot * kRows + row] = l_all;
          } else if (p.lse != nullptr && query >= 0) {
            p.lse[static_cast<int64_t>(query) * kHeads + head] =
                nothing ? -INFINITY : static_cast<float>(static_cast<double>(m_run) * p.natural + static_cast<double>(logf(l_all)));
          }
        }
        continued = false;
        if (query >= 0) {
#pragma unroll 1
          for (int c = 0; c < kHalf / 64; ++c) {
            uint32_t o[2][32];
            ptx::TmemLd32(tmem + lane_base + kColO + 64 * c, o[0]);
            ptx::TmemLd32(tmem + lane_base + kColO + 64 * c + 32, o[1]);
            ptx::TmemWaitLd();
            if (!whole) {
              uint4* dst = reinterpret_cast<uint4*>(p.ws_o) + (static_cast<int64_t>(slot) * (kLatent / 4) + (kHalf * rank + 64 * c) / 4) * kRows + row;
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const int j = 4 * (k & 7);
                dst[k * kRows] = make_uint4(o[k >> 3][j], o[k >> 3][j + 1], o[k >> 3][j + 2], o[k >> 3][j + 3]);
              }
            } else {
              if (__any_sync(0xffffffffu, nothing)) {
#pragma unroll
                for (int j = 0; j < 64; ++j) o[j >> 5][j & 31] = nothing ? 0u : o[j >> 5][j & 31];
              }
              // A lane has a row; the rows' 128 bytes change places in the warp's part of the weights' buffer, so that a store
              // instruction writes four rows' and not a piece of each of 32.
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                uint32_t two[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int j = 8 * (k & 3) + 2 * e;
                  const __nv_bfloat162 t = __floats2bfloat162_rn(__uint_as_float(o[k >> 2][j]) * inv_l, __uint_as_float(o[k >> 2][j + 1]) * inv_l);
                  two[e] = *reinterpret_cast<const uint32_t*>(&t);
                }
                ptx::StShared128(p_row + ((k ^ (row & 7)) << 4), two[0], two[1], two[2], two[3]);
              }
              __syncwarp();
              const int sub = lane >> 3, chunk = lane & 7;
              __nv_bfloat16* dst = p.out + (static_cast<int64_t>(query) * kHeads + (warp & 1) * 32 + sub) * kLatent + kHalf * rank + 64 * c + 8 * chunk;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                uint4 v;
                ptx::LdShared128(p_warp + (4 * i + sub) * 128 + ((chunk ^ (4 * (i & 1) + sub)) << 4), v.x, v.y, v.z, v.w);
                *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(4 * i) * kLatent) = v;
              }
              __syncwarp();
            }
          }
        }
        ptx::TcFenceBeforeSync();
        __syncwarp();
        if (lane == 0) ptx::MbarArrive(bar(&misc->o_empty));
      }
      if (!more) break;
      item = next_item;
      lo = next_lo;
      hi = next_hi;
      have = true;
      m_run = kLowest;
      l_run = 0.0f;
      for (int s = lo; s < hi && ok; ++s, ++g) {  // (ok is the warp's; warps that give up leave the others' waits to run out)
        const Step st = StepAt(item, s);
        const int mine = max(0, min(kTile, st.valid - kTile * rank)), others = max(0, min(kTile, st.valid - kTile * static_cast<int>(peer)));
        const int valid = (st.active >> which & 1) != 0 ? mine : 0;
        ok = WarpWait(bar(&misc->s_full), g & 1, misc, p.status, 30) && ok;
        ptx::TcFenceAfterSync();
        uint32_t sr[2][32];
        ptx::TmemLd32(tmem + lane_base + kColS, sr[0]);
        ptx::TmemLd32(tmem + lane_base + kColS + 32, sr[1]);
        ptx::TmemWaitLd();
        ptx::TcFenceBeforeSync();
        __syncwarp();
        if (lane == 0) ptx::MbarArrive(bar(&misc->s_empty));
        float (&f)[2][32] = reinterpret_cast<float (&)[2][32]>(sr);
        if (valid < kTile) {
#pragma unroll
          for (int c = 0; c < kTile; ++c) {
            if (c >= valid) f[c >> 5][c & 31] = -INFINITY;
          }
        }
        float top[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) top[c] = f[0][c];
#pragma unroll
        for (int c = 8; c < kTile; ++c) top[c & 7] = fmaxf(top[c & 7], f[c >> 5][c & 31]);
        float tile_max = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), fmaxf(fmaxf(top[4], top[5]), fmaxf(top[6], top[7])));
        send(tile_max);
        // The weights with the reference there is, while the peer's maximum is on its way; again if that makes it move. (With a
        // reference that this tile alone moves, the first one above all, that round would be in vain. A row of which nothing has
        // been seen has scores of -infinity here, whose weights are zero whatever the reference.)
        uint32_t packed[32];
        float sum = 0.0f;
        auto weigh = [&](float neg_m) {
          float part[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const float p0 = ptx::Ex2Approx(fmaf(f[c >> 4][2 * (c & 15)], p.scale_log2, neg_m));
            const float p1 = ptx::Ex2Approx(fmaf(f[c >> 4][2 * (c & 15) + 1], p.scale_log2, neg_m));
            const __nv_bfloat162 pb = __floats2bfloat162_rn(p0, p1);
            packed[c] = *reinterpret_cast<const uint32_t*>(&pb);
            part[c & 7] += p0 + p1;
          }
          sum = ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
        };
        bool again = __any_sync(0xffffffffu, tile_max * p.scale_log2 > m_run + kRescaleThreshold);
        if (!again) weigh(-m_run);
        tile_max = fmaxf(tile_max, receive()) * p.scale_log2;
        const bool moves = tile_max > m_run + kRescaleThreshold;
        const bool rescale = moves && m_run != kLowest;
        const float m_new = moves ? tile_max : m_run;
        const float factor = rescale ? ptx::Ex2Approx(m_run - m_new) : 1.0f;
        m_run = m_new;
        again |= __any_sync(0xffffffffu, moves) != 0;
        if (again) weigh(-m_run);
        l_run = l_run * factor + sum;

        weights_free();
        if (__any_sync(0xffffffffu, rescale)) {
          // The warp's lanes of O are scaled between this step's PV and the one before.
          if (g > 0) ok = WarpWait(bar(&misc->w_empty), (g & 1) ^ 1, misc, p.status, 35) && ok;
          ptx::TcFenceAfterSync();
#pragma unroll 1
          for (int c = 0; c < kHalf / 32; ++c) {
            uint32_t o[32];
            ptx::TmemLd32(tmem + lane_base + kColO + 32 * c, o);
            ptx::TmemWaitLd();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * factor);
            ptx::TmemSt32(tmem + lane_base + kColO + 32 * c, o);
          }
          ptx::TmemWaitSt();
          ptx::TcFenceBeforeSync();
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {  // 128-byte swizzle: chunk c of row r at c ^ (r % 8)
          ptx::StShared128(p_row + ((c ^ (row & 7)) << 4), packed[4 * c], packed[4 * c + 1], packed[4 * c + 2], packed[4 * c + 3]);
        }
        // Rows behind the end hold whatever the pool held there: zeroed, so that 0 x NaN cannot reach O. (A tile without any
        // token was loaded as zeros.)
        if (mine > 0 && mine < kTile) {
          unsigned char* slabs = smem + kOffV + (g & 1) * kVSlabs * kSlabBytes;
          for (int i = row; i < (kTile - mine) * kVSlabs * 8; i += kSoftmaxThreads) {
            *reinterpret_cast<int4*>(slabs + ((i >> 3) & 3) * kSlabBytes + (mine + (i >> 5)) * 128 + (i & 7) * 16) = make_int4(0, 0, 0, 0);
          }
        }
        if (others > 0 && others < kTile) {
          ok = WarpWait(bar(&misc->w_full), g & 1, misc, p.status, 34) && ok;
          for (int i = row; i < (kTile - others) * kVSlabs * 8; i += kSoftmaxThreads) {
            *reinterpret_cast<int4*>(smem + kOffW + ((i >> 3) & 3) * kSlabBytes + (others + (i >> 5)) * 128 + (i & 7) * 16) = make_int4(0, 0, 0, 0);
          }
        }
        ptx::FenceProxyAsyncShared();
        __syncwarp();
        if (lane == 0) ptx::MbarArrive(bar(&misc->p_full));
        if (g > 0) ok = WarpWait(bar(&misc->peer_p_empty), (g & 1) ^ 1, misc, p.status, 36) && ok;
        if (lane == 0) ptx::BulkCopyToCta(peer_p_warp, p_warp, 32 * 128, peer_p_bar);
      }
      if (!ok) break;
    }
    // The peer's last signals have arrived before this CTA may leave.
    if (ok && g > 0) {
      WarpWait(bar(&misc->peer_p_empty), (g & 1) ^ 1, misc, p.status, 37);
      WarpWait(bar(&misc->p_sent), (g & 1) ^ 1, misc, p.status, 37);
    }
  }

  if (warp == 4 || warp == 5 || warp == 7) ptx::ClusterWait();
  // ---- teardown: the peer may still write into this CTA's shared memory until it has come here too ------------------
  __syncthreads();
  if (Aborting(misc)) {
    // Copies may still be in flight towards this CTA or the peer (its weights, the tiles of an unfinished step): none takes
    // longer than this.
    const uint64_t t0 = ptx::GlobalTimerNs();
    while (ptx::GlobalTimerNs() - t0 < 2000000ull) {
    }
  }
  ptx::TcFenceBeforeSync();
  ptx::ClusterArrive();
  ptx::ClusterWait();
  ptx::TcFenceAfterSync();
  if (warp == 5) ptx::TmemDealloc(tmem, kTmemCols);
}

// Merges what the runs left of every item that was cut. A CTA takes 32 rows x kColumns columns of one. A warp has eight rows x four
// quads of columns: it reads 128 bytes of a quad's rows and writes 32 bytes of a row, and goes over the strips of 16 columns of its
// half of the CTA's columns; with 16 columns a CTA the two halves of the warps share the parts out instead (an item of few queries
// and many parts: two queries of 16,384 tokens 27.9 us a call with 32 columns a CTA, 23.8 with 16). The rows' weights are worked out once, by the whole CTA.
constexpr int kMergeRows = 32;

// kStrips strips of kParts parts are in flight at a time: eight loads a thread, whatever the number of parts. The first eight are
// the caller's, on their way while it works out the weights.
struct MergeData {
  const float4* at;   // this thread's row and first quad in slot 0
  int first, begin, parts;  // the parts begin .. parts - 1 are this thread's
  // Part r is run (first + r)'s, in the slot of the item that it begins (the first) or continues.
  __device__ __forceinline__ float4 Load(int strip, int r) const {
    return at[static_cast<int64_t>(2 * (first + r) + (r == 0 ? 1 : 0)) * (kLatent / 4 * kRows) + strip * (4 * kRows)];
  }
};
template <int kAllStrips, int kStrips, int kParts, bool kSplit>
__device__ __forceinline__ void MergeStrips(const MergeData& data, float4 (&d)[8], const float* weight, float inv, __nv_bfloat16* out, float4* other) {
  static_assert(kStrips * kParts == 8);
#pragma unroll 1
  for (int s0 = 0; s0 < kAllStrips; s0 += kStrips) {
    float4 acc[kStrips];
#pragma unroll
    for (int s = 0; s < kStrips; ++s) acc[s] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int r0 = data.begin; r0 < data.parts; r0 += kParts) {
      if (s0 > 0 || r0 > data.begin) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (r0 + e % kParts < data.parts) d[e] = data.Load(s0 + e / kParts, r0 + e % kParts);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float w = r0 + e % kParts < data.parts ? weight[(r0 + e % kParts) * kMergeRows] : 0.0f;
        if (w == 0.0f) continue;  // no weight, and the accumulator may hold anything
        float4& a = acc[e / kParts];
        a.x = fmaf(d[e].x, w, a.x);
        a.y = fmaf(d[e].y, w, a.y);
        a.z = fmaf(d[e].z, w, a.z);
        a.w = fmaf(d[e].w, w, a.w);
      }
    }
    if constexpr (kSplit) {  // the second half of the warps hands its sums over
      const int at = threadIdx.x & 127;
      if (threadIdx.x >= 128) other[at] = acc[0];
      __syncthreads();
      if (threadIdx.x >= 128) return;
      acc[0].x += other[at].x;
      acc[0].y += other[at].y;
      acc[0].z += other[at].z;
      acc[0].w += other[at].w;
    }
#pragma unroll
    for (int s = 0; s < kStrips; ++s) {
      const bool nothing = inv == 0.0f;  // a row without weights
      const __nv_bfloat162 lo = __floats2bfloat162_rn(nothing ? 0.0f : acc[s].x * inv, nothing ? 0.0f : acc[s].y * inv);
      const __nv_bfloat162 hi = __floats2bfloat162_rn(nothing ? 0.0f : acc[s].z * inv, nothing ? 0.0f : acc[s].w * inv);
      *reinterpret_cast<uint2*>(out + 16 * (s0 + s)) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  }
}

template <int kColumns>
__global__ void __launch_bounds__(256) MlaSharedMergeKernel(const __grid_constant__ SharedParams p) {
  const int rows = blockIdx.x / (kLatent / kColumns) * kMergeRows, columns = blockIdx.x % (kLatent / kColumns) * kColumns;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __shared__ float s_w[kMergeParts][kMergeRows];
  __shared__ float s_m[8][kMergeRows], s_l[8][kMergeRows];
  __shared__ float4 s_other[kColumns == 16 ? 128 : 1];
  GridDependencyWait();
  GridDependencyTrigger();
  const MergeRecord merge = p.merges[blockIdx.y];
  if (!MergeHolds(merge, static_cast<int>(blockIdx.y), p.merges_by_query != 0, p.batch, p.runs)) return;
  const int query = rows < kHeads ? merge.q0 : merge.q1;
  if (query < 0) return;
  const int first = merge.first, parts = merge.last - first + 1;
  constexpr bool kSplit = kColumns == 16;
  constexpr int kStrips = kSplit ? 1 : kColumns / 32;
  const int mine = 8 * (warp & 3) + (lane & 7);                                                 // this thread's row of the 32
  const int quad = columns / 4 + (kSplit ? 0 : (warp >> 2) * (kColumns / 8)) + (lane >> 3);     // and its first quad of columns
  const int middle = kSplit ? (parts + 1) / 2 : parts;
  const MergeData data{p.ws_o + static_cast<int64_t>(quad) * kRows + rows + mine, first, kSplit && warp >= 4 ? middle : 0, kSplit && warp >= 4 ? parts : middle};
  const int width = kStrips >= 4 && parts <= 2 ? 2 : kStrips >= 2 && parts <= 4 ? 4 : 8;  // parts in flight
  float4 d[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int r = data.begin + (e & (width - 1));
    if (r < data.parts) d[e] = data.Load(width == 2 ? e >> 1 : width == 4 ? e >> 2 : 0, r);
  }
  float l;
  {
    // Warp w takes parts w, w + 8, ..; a lane has a row.
    const int row = rows + lane;
    float m = kLowest, pl[kMergeParts / 8];
#pragma unroll
    for (int i = 0; i < kMergeParts / 8; ++i) {
      const int r = 8 * i + warp;
      pl[i] = 0.0f;
      if (r >= parts) break;
      const int at = (2 * (first + r) + (r == 0 ? 1 : 0)) * kRows + row;
      pl[i] = p.ws_l[at];
      const float pm = p.ws_m[at];
      s_w[r][lane] = pm;
      if (pl[i] != 0.0f) m = fmaxf(m, pm);  // (a part without weights does not count; one whose sum is NaN does)
    }
    s_m[warp][lane] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = fmaxf(m, s_m[w][lane]);
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < kMergeParts / 8; ++i) {
      const int r = 8 * i + warp;
      if (r >= parts) break;
      const float w = pl[i] != 0.0f ? exp2f(s_w[r][lane] - m) : 0.0f;
      s_w[r][lane] = w;
      l += pl[i] * w;
    }
    s_l[warp][lane] = l;
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) l += s_l[w][lane];
    if (columns == 0 && warp == 0 && p.lse != nullptr) {
      p.lse[static_cast<int64_t>(query) * kHeads + (row & (kHeads - 1))] =
          l == 0.0f ? -INFINITY : static_cast<float>(static_cast<double>(m) * p.natural + static_cast<double>(logf(l)));
    }
  }
  l = __shfl_sync(0xffffffffu, l, mine);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  __nv_bfloat16* out = p.out + (static_cast<int64_t>(query) * kHeads + ((rows + mine) & (kHeads - 1))) * kLatent + 4 * quad;
  const float* weight = &s_w[0][mine];
  if constexpr (kStrips >= 4) {
    if (width == 2) return MergeStrips<kStrips, 4, 2, false>(data, d, weight, inv, out, nullptr);
  }
  if constexpr (kStrips >= 2) {
    if (width == 4) return MergeStrips<kStrips, 2, 4, false>(data, d, weight, inv, out, nullptr);
  }
  MergeStrips<kStrips, 1, 8, kSplit>(data, d, weight, inv, out, s_other);
}

int32_t RunsOfDevice() { return CurrentDeviceSmCount() / 2 < kMergeParts ? CurrentDeviceSmCount() / 2 : kMergeParts; }

size_t SharedWorkspaceBytes(int32_t batch) {
  const size_t slots = static_cast<size_t>(RunsOfDevice()) * 2;
  return slots * kRows * (kLatent + 2) * sizeof(float) + static_cast<size_t>(RunsOfDevice()) * sizeof(MergeRecord) + static_cast<size_t>(batch) * sizeof(Item);
}

bool SharedSupports(const b200kv_shared_args& a) {
  return a.heads == kHeads && a.block_size % kTile == 0 && a.q_head_stride % 8 == 0 && a.q_seq_stride % 8 == 0 &&
         (reinterpret_cast<uintptr_t>(a.q) & 15u) == 0 && a.pool.pool_rows < INT32_MAX && a.pool.latent_row_stride * 2 < (1ll << 40);
}

int32_t LaunchShared(const b200kv_shared_args& a, cudaStream_t stream, int32_t* status) {
  static thread_local int configured_device = -1;
  int device = 0;
  if (int32_t rc = CheckCuda(cudaGetDevice(&device), "cudaGetDevice")) return rc;
  if (device != configured_device) {
    if (int32_t rc = CheckCuda(cudaFuncSetAttribute(MlaDecodeSharedKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes),
                               "decode_shared smem opt-in")) {
      return rc;
    }
    configured_device = device;
  }
  CUtensorMap latent_map, t_map, rope_map, q_map, q_rope_map;
  if (int32_t rc = GetSlabMap(a.pool.latent, a.pool.latent_row_stride, a.pool.pool_rows, kVSlabs, &latent_map)) return rc;
  if (int32_t rc = GetSlabMap(a.pool.latent, a.pool.latent_row_stride, a.pool.pool_rows, 2, &t_map)) return rc;
  if (int32_t rc = GetRowMap(a.pool.rope, a.pool.rope_row_stride, a.pool.pool_rows, kRope, kTile, &rope_map)) return rc;
  if (int32_t rc = GetQSlabMap(a.q, a.q_head_stride, a.q_seq_stride, a.batch, kHeads, 2, &q_map)) return rc;
  if (int32_t rc = GetQSlabMap(a.q, a.q_head_stride, a.q_seq_stride, a.batch, kHeads, 1, &q_rope_map)) return rc;
  const int32_t runs = RunsOfDevice();
  SharedParams p{};
  p.block_table = a.block_table;
  p.max_blocks = a.max_blocks;
  p.table_rows = a.table_rows;
  p.table_index = a.table_index;
  p.kv_len = a.kv_len;
  p.leader = a.leader;
  p.shared_len = a.shared_len;
  p.pool_rows = a.pool.pool_rows;
  p.batch = a.batch;
  p.block_size = a.block_size;
  p.longest = static_cast<int32_t>(a.max_blocks < (INT32_MAX - kStep) / a.block_size ? a.max_blocks * a.block_size + 1 : INT32_MAX - kStep);
  p.stable_tables = (a.flags & B200KV_DECODE_STABLE_TABLES) != 0 ? 1 : 0;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.natural = static_cast<double>(a.scale) / static_cast<double>(p.scale_log2);
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.lse = a.lse;
  const size_t slots = static_cast<size_t>(runs) * 2;
  p.ws_o = static_cast<float4*>(a.workspace);
  p.ws_m = reinterpret_cast<float*>(p.ws_o + slots * kRows * (kLatent / 4));
  p.ws_l = p.ws_m + slots * kRows;
  p.merges = reinterpret_cast<MergeRecord*>(p.ws_l + slots * kRows);
  p.items = reinterpret_cast<Item*>(p.merges + runs);
  p.merges_by_query = a.batch <= runs ? 1 : 0;
  p.runs = runs;
  p.status = status;
  if (int32_t rc = CheckCuda(LaunchOverlapped(MlaDecodeSharedKernel, dim3(2 * static_cast<unsigned>(runs)), dim3(kThreads), kSmemBytes, stream,
                                              latent_map, t_map, rope_map, q_map, q_rope_map, p),
                             "decode_shared launch")) {
    return rc;
  }
  // The fewer queries, the fewer items there can be to merge, and the more parts they have: fewer columns a CTA, so that there are
  // enough CTAs. Sequences behind a common prefix, us a call with 16, 32, 64 and 128 columns: 4 x 8,192 21.4, 23.8, 27.2, 35.3;
  // 8 x 8,192 23.9, 24.8, 27.3, 33.4; 16 x 4,096 24.8, 23.3, 24.6, 28.1; 32 x 4,096 36.5, 33.0, 32.8, 33.1; 48 x 4,096 47.5, 41.6, 40.5,
  // 39.7; 256 x 1,024 73.0, 62.0, 59.3, 57.3.
  const unsigned merges = static_cast<unsigned>(a.batch < runs ? a.batch : runs);
  auto merge = [&](auto kernel, int columns) {
    return LaunchOverlapped(kernel, dim3(static_cast<unsigned>(kRows / kMergeRows * (kLatent / columns)), merges), dim3(256), 0, stream, p);
  };
  return CheckCuda(a.batch < 12   ? merge(MlaSharedMergeKernel<16>, 16)
                   : a.batch < 36 ? merge(MlaSharedMergeKernel<32>, 32)
                                  : merge(MlaSharedMergeKernel<128>, 128),
                   "decode_shared merge launch");
}

}  // namespace
}  // namespace b200kv

using namespace b200kv;

extern "C" size_t b200kv_mla_decode_shared_workspace_bytes(int32_t batch, int32_t heads) {
  if (batch <= 0 || heads <= 0) return 0;
  // Beside the kernel's own need that of b200kv_mla_decode, where another geometry goes: its CUDA-core form keeps partials only
  // where it splits sequences, which many queries are not.
  const int32_t sms = CurrentDeviceSmCount();
  size_t need = SharedWorkspaceBytes(batch);
  for (size_t other : {TcWorkspaceBytes(sms), SimtSplitCount(batch, sms) > 1 ? SimtWorkspaceBytes(batch, heads, sms) : 0}) need = other > need ? other : need;
  return need;
}

extern "C" int32_t b200kv_mla_decode_shared(const b200kv_shared_args* args, void* stream, b200kv_status_word* status) {
  if (args == nullptr) {
    SetLastError("decode_shared: args is null");
    return B200KV_ERR_NULLPTR;
  }
  const b200kv_shared_args& a = *args;
  if (int32_t rc = FaultCheck("b200kv_mla_decode_shared")) return rc;
  if (int32_t rc = ValidatePoolView(&a.pool)) return rc;
  if (a.batch == 0) return B200KV_OK;
  if (a.q == nullptr || a.block_table == nullptr || a.kv_len == nullptr || a.leader == nullptr || a.shared_len == nullptr || a.out == nullptr) {
    SetLastError("decode_shared: q, block_table, kv_len, leader, shared_len and out must be non-null");
    return B200KV_ERR_NULLPTR;
  }
  if ((reinterpret_cast<uintptr_t>(a.out) & 15u) != 0) {
    SetLastError("decode_shared refused: out must be 16-byte aligned");
    return B200KV_ERR_INVALID;
  }
  if (a.batch < 0 || a.heads <= 0 || a.block_size <= 0 || a.max_blocks <= 0 || a.pool.pool_rows % a.block_size != 0 || !(a.scale > 0.0f) ||
      a.q_head_stride < kLatent + kRope || (a.batch > 1 && a.q_seq_stride < 0) || (a.out_fp8 == nullptr) != (a.out_scale == nullptr) ||
      a.table_rows < (a.table_index != nullptr ? 1 : a.batch)) {
    SetLastError("decode_shared refused: batch %d heads %d block_size %d table %lld x %lld scale %g q strides %lld/%lld (a table row per query "
                 "without table_index; out_fp8 and out_scale come together)",
                 a.batch, a.heads, a.block_size, static_cast<long long>(a.table_rows), static_cast<long long>(a.max_blocks),
                 static_cast<double>(a.scale), static_cast<long long>(a.q_seq_stride), static_cast<long long>(a.q_head_stride));
    return B200KV_ERR_INVALID;
  }
  if (!SharedSupports(a)) {
    // Any other geometry has each query read its own rows; the result is the same.
    if (a.table_index != nullptr) {
      SetLastError("decode_shared: table_index needs the tensor-core kernel's geometry (64 heads, block_size %% 64 == 0, 16-byte aligned q with "
                   "strides that are multiples of 8 elements); heads %d, block_size %d", a.heads, a.block_size);
      return B200KV_ERR_INVALID;
    }
    b200kv_decode_args d{};
    d.q = a.q;
    d.q_seq_stride = a.q_seq_stride;
    d.q_head_stride = a.q_head_stride;
    d.pool = a.pool;
    d.block_table = a.block_table;
    d.max_blocks = a.max_blocks;
    d.kv_len = a.kv_len;
    d.batch = a.batch;
    d.heads = a.heads;
    d.block_size = a.block_size;
    d.scale = a.scale;
    d.out = a.out;
    d.lse = a.lse;
    d.workspace = a.workspace;
    d.workspace_bytes = a.workspace_bytes;
    d.flags = a.flags;
    d.out_fp8 = a.out_fp8;
    d.out_scale = a.out_scale;
    return b200kv_mla_decode(&d, stream, status);
  }
  const size_t need = SharedWorkspaceBytes(a.batch);
  if (a.workspace == nullptr || a.workspace_bytes < need || (reinterpret_cast<uintptr_t>(a.workspace) & 15u) != 0) {
    SetLastError("decode_shared: workspace of %zu bytes (16-byte aligned) required, %zu given", need, a.workspace_bytes);
    return a.workspace == nullptr ? B200KV_ERR_NULLPTR : B200KV_ERR_INVALID;
  }
  if (int32_t rc = LaunchShared(a, static_cast<cudaStream_t>(stream), status)) return rc;
  if (a.out_fp8 == nullptr) return B200KV_OK;
  const int64_t cols = static_cast<int64_t>(a.heads) * kLatent;
  return b200kv_mx_quant_e4m3(a.out, cols, a.batch, cols, a.out_fp8, cols, a.out_scale, cols / 32, stream);
}
