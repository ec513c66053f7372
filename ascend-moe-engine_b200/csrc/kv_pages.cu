// Pages of the cache copied inside it, in every layer at once: what a forked sequence's half-filled last block, a write into a
// block that others hold, and a compaction need (b200kv_block_pool_fork, _unshare and _compact say which). The reference keeps
// one sequence and never moves a block (src/memory/static_arena_manager.cpp:298-300).
//
// For layer l and move i = (source block, destination block, rows): rows [0, rows) of the source block become those of the
// destination block, latent and rope. Bytes only, so the bound is HBM: 1,152 read and 1,152 written per row and layer.
//
// A unit of work is up to 16 rows of one move in one layer (18 KB): the units of a single forked block over 43 layers then reach
// more than half of the SMs, and with three stages to a CTA and four CTAs on an SM some 220 KB an SM are in flight, several
// times what latency x bandwidth asks for (four stages and three CTAs: 43.0 us instead of 40.5 for 32 half-filled blocks of 128 rows
// in 43 layers, 0.87 of the measured copy rate; 300 whole blocks of 128 rows in 16 layers 237 us, 0.91). A warp per CTA drives the stages with untiled bulk copies, global -> shared ->
// global; no thread touches the data. Rows that lie one behind the other (the two caches of the arena; the fused 576-wide row)
// go as one copy per array, any other stride row by row, a lane each.
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace b200kv {

int32_t ValidatePoolView(const b200kv_pool_view* pool);

namespace {

constexpr int kUnitRows = 16;
constexpr int kLatentBytes = B200KV_LATENT_DIM * 2;
constexpr int kRopeBytes = B200KV_ROPE_DIM * 2;
constexpr int kRowBytes = kLatentBytes + kRopeBytes;
constexpr int kStageBytes = kUnitRows * kRowBytes;  // 18,432
constexpr int kStages = 3;
constexpr int kAhead = 2;  // units whose loads are in flight before the oldest is stored
constexpr int kSmemBytes = kStages * kStageBytes + 128;
constexpr int kCtasPerSm = 4;

struct PageParams {
  char* latent;
  char* rope;
  int64_t latent_row_bytes;
  int64_t rope_row_bytes;
  int64_t latent_layer_bytes;
  int64_t rope_layer_bytes;
  int64_t blocks;
  int64_t layers;
  const int32_t* moves;  // [n][3]
  int64_t n_moves;
  int64_t units;
  int32_t block_size;
  int32_t chunks;  // units of a whole block
  int32_t fused;   // a row's latent and rope are adjacent and rows follow each other
  int32_t dense;   // each array's rows follow each other
  int32_t* status;
};

// The unit's rows as byte offsets from the arrays' bases; rows 0: nothing to do.
struct Unit {
  int64_t src_latent, dst_latent, src_rope, dst_rope;
  int rows;
};

__device__ __forceinline__ Unit UnitOf(const PageParams& p, int64_t u) {
  Unit unit{};
  if (u >= p.units) return unit;
  const int64_t layer = u % p.layers;
  const int64_t rest = u / p.layers;
  const int chunk = static_cast<int>(rest % p.chunks);
  const int64_t move = rest / p.chunks;
  const int32_t src = p.moves[3 * move], dst = p.moves[3 * move + 1], rows = p.moves[3 * move + 2];
  if (src < 0 || dst < 0 || src == dst || rows == 0) return unit;
  if (src >= p.blocks || dst >= p.blocks || rows < 0 || rows > p.block_size) {
    const int32_t bad = src >= p.blocks ? src : dst >= p.blocks ? dst : rows;
    RecordError(p.status, B200KV_DEV_BAD_BLOCK, static_cast<int32_t>(move), bad);
    return unit;
  }
  const int64_t first = static_cast<int64_t>(chunk) * kUnitRows;
  const int64_t src_row = static_cast<int64_t>(src) * p.block_size + first, dst_row = static_cast<int64_t>(dst) * p.block_size + first;
  unit.rows = max(0, min(kUnitRows, rows - static_cast<int>(first)));
  unit.src_latent = layer * p.latent_layer_bytes + src_row * p.latent_row_bytes;
  unit.dst_latent = layer * p.latent_layer_bytes + dst_row * p.latent_row_bytes;
  unit.src_rope = layer * p.rope_layer_bytes + src_row * p.rope_row_bytes;
  unit.dst_rope = layer * p.rope_layer_bytes + dst_row * p.rope_row_bytes;
  return unit;
}

__device__ __forceinline__ void BulkStore(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

__global__ void __launch_bounds__(32, kCtasPerSm) CopyBlocksKernel(PageParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  const uint32_t stages = ptx::SmemAddr(smem);
  const uint32_t bars = stages + kStages * kStageBytes;
  const int lane = threadIdx.x;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) ptx::MbarInit(bars + 8 * s, 1);
    ptx::FenceBarrierInit();
  }
  __syncwarp();
  GridDependencyTrigger();
  GridDependencyWait();

  // What this lane copies of a unit: one piece of the stage, at `at`, of `bytes` bytes.
  char* dst[kAhead + 1];
  uint32_t bytes[kAhead + 1], at = 0;
  const int row = lane & (kUnitRows - 1);
  const bool is_rope = p.fused != 0 ? false : p.dense != 0 ? lane == 1 : lane >= kUnitRows;
  const bool takes_part = p.fused != 0 ? lane == 0 : p.dense != 0 ? lane < 2 : true;
  if (is_rope) at = kUnitRows * kLatentBytes;
  if (p.fused == 0 && p.dense == 0) at += row * (is_rope ? kRopeBytes : kLatentBytes);

  int loaded = 0, stored = 0;  // units of this CTA
  bool ok = true;
  Unit mine{};
  unsigned pending = 0;  // of the 32 units looked up together: those still to be loaded
  int64_t next = blockIdx.x;
  const int64_t step = gridDim.x;

  // Loads the next unit that has rows; false when there is none left.
  auto load = [&](int slot) -> bool {
    while (pending == 0) {
      if (next >= p.units) return false;
      mine = UnitOf(p, next + lane * step);  // 32 units' moves in one round trip
      next += 32 * step;
      pending = __ballot_sync(0xffffffffu, mine.rows > 0);
    }
    const int from = __ffs(pending) - 1;
    pending &= pending - 1;
    const int rows = __shfl_sync(0xffffffffu, mine.rows, from);
    int64_t src = __shfl_sync(0xffffffffu, mine.src_latent, from), to = __shfl_sync(0xffffffffu, mine.dst_latent, from);
    const int64_t src_rope = __shfl_sync(0xffffffffu, mine.src_rope, from), to_rope = __shfl_sync(0xffffffffu, mine.dst_rope, from);
    const char* base = p.latent;
    uint32_t n = p.fused != 0 ? rows * kRowBytes : rows * kLatentBytes;
    if (is_rope) {
      base = p.rope;
      src = src_rope;
      to = to_rope;
      n = rows * kRopeBytes;
    }
    if (p.fused == 0 && p.dense == 0) {
      const int64_t row_bytes = is_rope ? p.rope_row_bytes : p.latent_row_bytes;
      src += row * row_bytes;
      to += row * row_bytes;
      n = row < rows ? (is_rope ? kRopeBytes : kLatentBytes) : 0;
    }
    if (!takes_part) n = 0;
    const int stage = loaded % kStages;
    if (lane == 0) ptx::MbarArriveExpectTx(bars + 8 * stage, rows * kRowBytes);
    __syncwarp();
    if (n > 0) ptx::BulkLoad(stages + stage * kStageBytes + at, base + src, n, bars + 8 * stage);
    dst[slot] = const_cast<char*>(base) + to;
    bytes[slot] = n;
    ++loaded;
    return true;
  };
  bool more = true;
#pragma unroll
  for (int i = 0; i < kAhead; ++i) more = more && load(i);
  while (ok && (more || stored < loaded)) {
    // The stage that the next load takes was last stored from kStages units before it: all of this lane's stores but the
    // latest kStages - kAhead - 1 have been read out of shared memory.
    ptx::BulkWaitGroupRead<kStages - kAhead - 1>();
    __syncwarp();
    more = more && load(kAhead);
    if (stored == loaded) break;
    const int stage = stored % kStages;
    const uint32_t parity = (stored / kStages) & 1;
    uint64_t start = 0;
    for (uint32_t it = 0; !ptx::MbarTryWait(bars + 8 * stage, parity); ++it) {
      if ((it & 255u) != 255u) continue;
      const uint64_t now = ptx::GlobalTimerNs();
      if (start == 0) start = now;
      if (now - start > 1000000000ull) {
        ok = false;
        break;
      }
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) {
      if (lane == 0) RecordError(p.status, B200KV_DEV_TIMEOUT, 40, static_cast<int32_t>(blockIdx.x), static_cast<int32_t>(parity));
      break;
    }
    if (bytes[0] > 0) BulkStore(dst[0], stages + stage * kStageBytes + at, bytes[0]);
    ptx::BulkCommitGroup();
    ++stored;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      dst[i] = dst[i + 1];
      bytes[i] = bytes[i + 1];
    }
  }
  if (!ok) {  // the loads in flight may still land: wait for them, with a limit
    const uint64_t t0 = ptx::GlobalTimerNs();
    for (int u = stored; u < loaded; ++u) {
      while (!ptx::MbarTryWait(bars + 8 * (u % kStages), (u / kStages) & 1)) {
        if (ptx::GlobalTimerNs() - t0 > 200000000ull) break;
      }
    }
  }
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

}  // namespace
}  // namespace b200kv

using namespace b200kv;

extern "C" int32_t b200kv_copy_blocks(const b200kv_pool_view* pool, int64_t layers, int64_t latent_layer_stride, int64_t rope_layer_stride,
                                      const int32_t* moves, int64_t n_moves, int64_t block_size, void* stream, b200kv_status_word* status) {
  if (int32_t rc = FaultCheck("b200kv_copy_blocks")) return rc;
  if (int32_t rc = ValidatePoolView(pool)) return rc;
  if (n_moves == 0 || layers == 0) return B200KV_OK;
  if (moves == nullptr) {
    SetLastError("copy_blocks: moves is null");
    return B200KV_ERR_NULLPTR;
  }
  if (n_moves < 0 || n_moves > INT32_MAX || layers < 0 || layers > INT32_MAX || block_size <= 0 || block_size > INT32_MAX || pool->pool_rows % block_size != 0 ||
      (layers > 1 && (latent_layer_stride <= 0 || rope_layer_stride <= 0 || latent_layer_stride % 8 != 0 || rope_layer_stride % 8 != 0))) {
    SetLastError("copy_blocks refused: %lld moves, %lld layers at strides %lld / %lld (positive multiples of 8 elements), %lld pool rows in "
                 "blocks of %lld",
                 static_cast<long long>(n_moves), static_cast<long long>(layers), static_cast<long long>(latent_layer_stride),
                 static_cast<long long>(rope_layer_stride), static_cast<long long>(pool->pool_rows), static_cast<long long>(block_size));
    return B200KV_ERR_INVALID;
  }
  PageParams p{};
  p.latent = static_cast<char*>(pool->latent);
  p.rope = static_cast<char*>(pool->rope);
  p.latent_row_bytes = pool->latent_row_stride * 2;
  p.rope_row_bytes = pool->rope_row_stride * 2;
  p.latent_layer_bytes = latent_layer_stride * 2;
  p.rope_layer_bytes = rope_layer_stride * 2;
  p.blocks = pool->pool_rows / block_size;
  p.layers = layers;
  p.moves = moves;
  p.n_moves = n_moves;
  p.block_size = static_cast<int32_t>(block_size);
  p.chunks = static_cast<int32_t>((block_size + kUnitRows - 1) / kUnitRows);
  if (__builtin_mul_overflow(n_moves * layers, static_cast<int64_t>(p.chunks), &p.units)) {
    SetLastError("copy_blocks refused: %lld moves in %lld layers", static_cast<long long>(n_moves), static_cast<long long>(layers));
    return B200KV_ERR_INVALID;
  }
  p.fused = p.rope == p.latent + kLatentBytes && p.latent_row_bytes == kRowBytes && p.rope_row_bytes == kRowBytes &&
            (layers == 1 || p.latent_layer_bytes == p.rope_layer_bytes);
  p.dense = p.latent_row_bytes == kLatentBytes && p.rope_row_bytes == kRopeBytes;
  p.status = status;
  static thread_local int configured_device = -1;
  int device = 0;
  if (int32_t rc = CheckCuda(cudaGetDevice(&device), "cudaGetDevice")) return rc;
  if (device != configured_device) {
    if (int32_t rc = CheckCuda(cudaFuncSetAttribute(CopyBlocksKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes), "copy_blocks smem opt-in"))
      return rc;
    configured_device = device;
  }
  const int64_t cap = static_cast<int64_t>(CurrentDeviceSmCount()) * kCtasPerSm;
  return CheckCuda(LaunchOverlapped(CopyBlocksKernel, dim3(static_cast<unsigned>(p.units < cap ? p.units : cap)), dim3(32), kSmemBytes,
                                    static_cast<cudaStream_t>(stream), p),
                   "copy_blocks launch");
}
