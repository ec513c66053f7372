// The KV path as the engine drives it, batched: what Dsv4Pipeline::Build and ::DecodeStep do for the paged cache
// and the attention stages (src/pipeline/pipeline.cpp:212-258, 496-537), lifted from one sequence and one token
// per step (src/memory/static_arena_manager.cpp:37-39; src/pipeline/pipeline.cpp:40, 515-519) to max_seqs
// sequences and to prefill chunks of many tokens (apps/moe_runner.cpp:434-439 runs the prompt as P single-token
// steps).
//
//   Build      reserve the KV spans and the step's staging in the static arena, note the attention workspace,
//              ONE commit, the workspace, seal; create the block pool; the uploads' pinned staging blocks.
//   step       begin: grow every sequence of the step in the block pool (plan, then commit: a refused growth
//              changes nothing), write the step's table rows, lengths and slots into a pinned block and upload
//              them with ONE copy (the reference's mailbox, :515-519). Then per layer, in the reference's stage
//              order: producer (kv_a_norm + rope + kv_cache_write, stages 6-8), attention (9), MX quantisation of
//              its output (10). end: no allocation happened since begin, as the reference asserts per step
//              (:502-503, 535-536).
//   between steps  fork: a sequence that begins as another's first tokens and shares its whole blocks; trim: rejected
//              drafts are taken back; compact: blocks move towards the pool's start. What has to be copied on the device is
//              enqueued before the tables change for good.
// Every device operation is one of the library's own entry points (b200kv_append_fused, b200kv_mla_decode,
// b200kv_mla_decode_shared, b200kv_copy_blocks); this file is host logic only and allocates nothing after Build.
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>
#include <new>
#include <vector>

#include "b200kv.h"

namespace b200kv {
void SetLastError(const char* fmt, ...);
int32_t CheckCuda(cudaError_t err, const char* what);
int32_t FaultCheck(const char* entry_point);
int64_t StoredTokens(const b200kv_block_pool* pool);
void UndoUnshare(b200kv_block_pool* pool, int32_t seq, int32_t index, const int32_t* move);
bool TakeFromBehind(b200kv_block_pool* pool, int32_t seq, int32_t index, int32_t* move_out);
void UndoTakeFromBehind(b200kv_block_pool* pool, int32_t seq, int32_t index, const int32_t* move);
}  // namespace b200kv

using b200kv::CheckCuda;
using b200kv::SetLastError;

struct b200kv_engine {
  b200kv_engine_config cfg{};
  b200kv_arena* arena = nullptr;
  b200kv_kv_cache cache{};
  b200kv_block_pool* pool = nullptr;
  int64_t status_handle = -1;
  int64_t queries_handle = -1;
  int64_t moves_handle = -1;
  // Device addresses of the step's spans (resolved once, after Commit).
  int32_t* d_table = nullptr;
  int32_t* d_slots = nullptr;
  int32_t* d_lens = nullptr;
  int32_t* d_status = nullptr;
  int32_t* d_queries = nullptr;  // [4][max_step_tokens]: kv_len, leader, shared_len, table_index of the step's queries
  int32_t* d_moves = nullptr;    // [num_blocks][3]
  // Pinned blocks that mirror [queries | table .. lens] of the arena byte for byte: one copy uploads a step (from the
  // table on, when the step's attention needs no queries). The copy reads its block when the stream comes to it, behind the
  // kernels of the steps before, so steps take the blocks in turn and one is written again only when its upload has been made.
  struct Staging {
    unsigned char* at = nullptr;
    cudaEvent_t uploaded = nullptr;
    bool pending = false;
  };
  static constexpr int kStagings = 2;
  Staging stagings[kStagings];
  int at_staging = 0;
  // What an upload that is part of a graph reads when the graph runs: the step begun last, from the first such upload on.
  unsigned char* captured = nullptr;
  bool has_captured = false;
  unsigned char* staging = nullptr;  // of the step in hand
  size_t staging_bytes = 0;
  size_t table_off = 0, slots_off = 0, lens_off = 0;
  // The step in flight.
  bool in_step = false;
  int32_t step_seqs = 0;
  int32_t step_tokens = 0;
  int32_t allocations_at_begin = 0;
  int64_t steps = 0;
  std::vector<int32_t> step_seq_ids;   // sized at Build: the step's sequences and by how much each grew
  std::vector<int32_t> step_grown;
  bool step_shares = false;            // the step's attention is b200kv_mla_decode_shared
  std::vector<int32_t> moves;          // [num_blocks][3], sized at Build
};

namespace {

// From how many common tokens (counted once a pair of neighbours) for each sequence of the step, and from what part of all tokens
// on, attention goes through the entry point for shared rows. Both sides measured, us a layer, b200kv_mla_decode -> _shared, over the
// rows of so many layers that they do not stay in L2; all sequences share the given length and have 100 tokens of their own:
//           256            512            1,024          2,048          4,096          8,192          32,768
//     2      9.3 ->  11.8   11.7 ->  11.9   13.3 ->  12.8   17.0 ->  15.7   20.7 ->  17.3   22.3 ->  20.1   29.7 ->  30.3
//     3      9.3 ->  11.8   11.7 ->  12.1   13.4 ->  14.1   15.2 ->  16.0   16.6 ->  17.6   19.2 ->  21.0   33.6 ->  31.0
//     4      9.6 ->  12.1   12.0 ->  12.4   13.8 ->  14.5   17.6 ->  15.9   19.0 ->  17.9   21.8 ->  21.2   39.1 ->  32.2
//     8     11.3 ->  14.2   13.0 ->  15.3   16.9 ->  16.7   17.9 ->  17.5   21.3 ->  19.6   27.8 ->  23.8   61.4 ->  43.5
//    16     12.7 ->  15.6   15.7 ->  16.8   19.0 ->  18.0   21.0 ->  19.8   27.2 ->  22.9   38.6 ->  29.7   112  ->  70.5
//    32     14.0 ->  19.3   17.2 ->  19.6   21.9 ->  21.4   27.9 ->  25.3   39.2 ->  32.2   61.1 ->  44.8   219  ->  128
//    64     16.8 ->  21.8   20.1 ->  24.9   31.7 ->  27.5   43.3 ->  34.8   66.0 ->  47.3   112  ->  71.0   442  ->  241
//   128     18.0 ->  28.1   41.1 ->  30.3   52.8 ->  37.3   75.6 ->  49.9   120  ->  76.7   230  ->  133
// Two neighbours are common once, so the line lies between the columns of 512 and 1,024. On its shared side three sequences of up
// to 8,192 tokens (one of them is alone) lose 4 to 9 %, 4 x 1,024 5 %, 2 x 32,768 2 %; below it 128 x 512 would gain. With out_fp8,
// which b200kv_mla_decode writes in its merge and the other in a launch of its own, the line would lie higher: 3 x 1,024 .. 8,192 lose 7
// to 13 %, 4, 8 and 16 sequences up to 4,096 tokens 6 % at most (8 x 2,048 18.6 -> 19.5, 16 x 4,096 28.1 -> 25.6, 32 x 1,024 23.7 -> 23.9).
constexpr int64_t kLeastCommon = 512;
constexpr int64_t kCommonPart = 4;

int32_t Refuse(const char* text) {
  SetLastError("%s", text);
  return B200KV_ERR_INVALID;
}

// The queries of the step in the staging block: one per new token, attending over its sequence up to itself. A sequence's tokens
// are a group; so are neighbours of one token each whose table rows begin with the same blocks. True when attention should go
// through the entry point for shared rows: always with several tokens a sequence, else when the common blocks are worth it.
bool PlanQueries(b200kv_engine* e, int32_t n_seqs, int32_t n_tokens) {
  const size_t stride = static_cast<size_t>(e->cfg.max_step_tokens);
  int32_t* kv_len = reinterpret_cast<int32_t*>(e->staging);
  int32_t *leader = kv_len + stride, *shared = leader + stride, *index = shared + stride;
  const int32_t* table = reinterpret_cast<const int32_t*>(e->staging + e->table_off);
  const int32_t* lens = reinterpret_cast<const int32_t*>(e->staging + e->lens_off);
  if (n_tokens != n_seqs) {
    int32_t at = 0;
    for (int32_t i = 0; i < n_seqs; ++i) {
      const int32_t n = e->step_grown[static_cast<size_t>(i)], first = at;
      for (int32_t k = 0; k < n; ++k, ++at) {
        kv_len[at] = lens[i] - n + k + 1;
        leader[at] = first;
        shared[at] = lens[i];
        index[at] = i;
      }
    }
    return true;
  }
  int64_t all = 0;
  for (int32_t i = 0; i < n_seqs; ++i) {
    kv_len[i] = lens[i];
    index[i] = i;
    all += lens[i];
  }
  const int64_t common = b200kv_find_shared(table, e->cfg.max_blocks_per_seq, lens, n_seqs, e->cfg.block_size, leader, shared);
  return common >= kLeastCommon * n_seqs && kCommonPart * common >= all;
}

// The next staging block, once the upload that was last made from it has left it.
int32_t TakeStaging(b200kv_engine* e) {
  b200kv_engine::Staging& block = e->stagings[e->at_staging];
  if (block.pending) {
    // (a capture on this thread does not mind: the event is none of its)
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    const int32_t rc = CheckCuda(cudaEventSynchronize(block.uploaded), "engine staging (the upload before)");
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (rc != B200KV_OK) return rc;
    block.pending = false;
  }
  e->staging = block.at;
  return B200KV_OK;
}

// The block in hand goes to the device, from byte `from` on.
int32_t Upload(b200kv_engine* e, size_t from, cudaStream_t stream) {
  unsigned char* to = reinterpret_cast<unsigned char*>(e->d_queries) + from;
  const size_t bytes = e->staging_bytes - from;
  if (int32_t rc = b200kv::FaultCheck("b200kv_engine_step_upload")) return rc;
  if (e->cfg.backend != B200KV_ARENA_DEVICE) {
    std::memcpy(to, e->staging + from, bytes);
    return B200KV_OK;
  }
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (int32_t rc = CheckCuda(cudaStreamIsCapturing(stream, &capture), "engine step upload")) return rc;
  e->has_captured |= capture != cudaStreamCaptureStatusNone;
  if (e->has_captured) std::memcpy(e->captured, e->staging, e->staging_bytes);
  if (capture != cudaStreamCaptureStatusNone) {
    return CheckCuda(cudaMemcpyAsync(to, e->captured + from, bytes, cudaMemcpyHostToDevice, stream), "engine step upload");
  }
  b200kv_engine::Staging& block = e->stagings[e->at_staging];
  if (int32_t rc = CheckCuda(cudaMemcpyAsync(to, block.at + from, bytes, cudaMemcpyHostToDevice, stream), "engine step upload")) return rc;
  if (int32_t rc = CheckCuda(cudaEventRecord(block.uploaded, stream), "engine step upload")) return rc;
  block.pending = true;
  e->at_staging = (e->at_staging + 1) % b200kv_engine::kStagings;
  return B200KV_OK;
}

// Moves of blocks (pool ids) in every layer, enqueued on the stream.
int32_t CopyMoves(b200kv_engine* e, const int32_t* moves, int32_t n, void* stream) {
  if (n == 0) return B200KV_OK;
  b200kv_pool_view view;
  if (int32_t rc = b200kv_kv_cache_layer_view(e->arena, &e->cache, 0, &view)) return rc;
  const size_t bytes = static_cast<size_t>(n) * 12;
  const int64_t rows = static_cast<int64_t>(e->cfg.num_blocks) * e->cfg.block_size;
  if (e->cfg.backend != B200KV_ARENA_DEVICE) {  // host memory stands for the device's
    if (int32_t rc = b200kv::FaultCheck("b200kv_copy_blocks")) return rc;
    for (int64_t l = 0; l < e->cfg.layers; ++l) {
      for (int32_t i = 0; i < n; ++i) {
        const int64_t from = moves[3 * i] * static_cast<int64_t>(e->cfg.block_size), to = moves[3 * i + 1] * static_cast<int64_t>(e->cfg.block_size);
        auto copy = [&](void* base, int64_t width) {
          auto* layer = static_cast<unsigned char*>(base) + l * rows * width;
          std::memcpy(layer + to * width, layer + from * width, static_cast<size_t>(moves[3 * i + 2] * width));
        };
        copy(view.latent, B200KV_LATENT_DIM * 2);
        copy(view.rope, B200KV_ROPE_DIM * 2);
      }
    }
    return B200KV_OK;
  }
  // (from pageable memory: the list has been read when the call returns, so that the next one may be written)
  if (int32_t rc = CheckCuda(cudaMemcpyAsync(e->d_moves, moves, bytes, cudaMemcpyHostToDevice, static_cast<cudaStream_t>(stream)), "engine moves upload"))
    return rc;
  return b200kv_copy_blocks(&view, e->cfg.layers, rows * B200KV_LATENT_DIM, rows * B200KV_ROPE_DIM, e->d_moves, n, e->cfg.block_size, stream,
                            e->d_status);
}

}  // namespace

extern "C" b200kv_engine* b200kv_engine_create(const b200kv_engine_config* config) {
  if (config == nullptr) {
    SetLastError("engine_create: config is null");
    return nullptr;
  }
  const b200kv_engine_config& c = *config;
  if (c.layers <= 0 || c.max_seqs <= 0 || c.num_blocks <= 0 || c.block_size <= 0 || c.block_size % 64 != 0 ||
      c.max_blocks_per_seq <= 0 || c.max_step_tokens < c.max_seqs || !(c.scale > 0.0f) || !(c.eps >= 0.0f) ||
      (c.backend != B200KV_ARENA_DEVICE && c.backend != B200KV_ARENA_HOST_SIM)) {
    SetLastError("engine_create refused: layers %d, sequences %d, blocks %d x %d rows (a multiple of 64), blocks per "
                 "sequence %d, tokens per step %d (at least one per sequence), scale %g, eps %g, backend %d",
                 c.layers, c.max_seqs, c.num_blocks, c.block_size, c.max_blocks_per_seq, c.max_step_tokens,
                 static_cast<double>(c.scale), static_cast<double>(c.eps), c.backend);
    return nullptr;
  }
  auto* e = new (std::nothrow) b200kv_engine();
  if (e == nullptr) return nullptr;
  e->cfg = c;
  auto fail = [&]() {
    b200kv_engine_destroy(e);
    return static_cast<b200kv_engine*>(nullptr);
  };
  e->arena = b200kv_arena_create(c.backend);
  if (e->arena == nullptr) return fail();
  // RESERVE: the step's queries, the KV spans (table, slots, lengths, the two layer-major caches), then the status word and
  // the moves of a compaction.
  e->queries_handle = b200kv_arena_reserve(e->arena, "kv.queries", static_cast<size_t>(c.max_step_tokens) * 16, 0);
  if (e->queries_handle < 0) return fail();
  if (b200kv_kv_cache_reserve_batched(e->arena, c.num_blocks, c.block_size, c.layers, c.max_seqs, c.max_blocks_per_seq,
                                      c.max_step_tokens, &e->cache) != B200KV_OK) {
    return fail();
  }
  e->status_handle = b200kv_arena_reserve(e->arena, "kv.status", 16, 0);
  if (e->status_handle < 0) return fail();
  e->moves_handle = b200kv_arena_reserve(e->arena, "kv.moves", static_cast<size_t>(c.num_blocks) * 12, 0);
  if (e->moves_handle < 0) return fail();
  // The attention workspace is the only operator workspace of this path (the producer and the quantiser need
  // none): its high-water mark over both attention entry points, one commit, the workspace, the latch.
  size_t workspace = 4096;
  if (c.backend == B200KV_ARENA_DEVICE) {
    workspace = b200kv_mla_decode_shared_workspace_bytes(c.max_step_tokens, B200KV_HEADS);
    const size_t plain = b200kv_mla_decode_workspace_bytes(c.max_seqs, B200KV_HEADS, 0);
    if (plain > workspace) workspace = plain;
  }
  if (b200kv_arena_note_workspace(e->arena, workspace) != B200KV_OK || b200kv_arena_commit(e->arena) != B200KV_OK ||
      b200kv_arena_commit_workspace(e->arena) != B200KV_OK) {
    return fail();
  }
  e->d_table = static_cast<int32_t*>(b200kv_arena_address(e->arena, e->cache.block_table_handle));
  e->d_slots = static_cast<int32_t*>(b200kv_arena_address(e->arena, e->cache.slot_mapping_handle));
  e->d_lens = static_cast<int32_t*>(b200kv_arena_address(e->arena, e->cache.seq_lens_handle));
  e->d_status = static_cast<int32_t*>(b200kv_arena_address(e->arena, e->status_handle));
  e->d_queries = static_cast<int32_t*>(b200kv_arena_address(e->arena, e->queries_handle));
  e->d_moves = static_cast<int32_t*>(b200kv_arena_address(e->arena, e->moves_handle));
  const int64_t first = b200kv_arena_offset(e->arena, e->queries_handle);
  e->table_off = static_cast<size_t>(b200kv_arena_offset(e->arena, e->cache.block_table_handle) - first);
  e->slots_off = static_cast<size_t>(b200kv_arena_offset(e->arena, e->cache.slot_mapping_handle) - first);
  e->lens_off = static_cast<size_t>(b200kv_arena_offset(e->arena, e->cache.seq_lens_handle) - first);
  e->staging_bytes = e->lens_off + static_cast<size_t>(c.max_seqs) * 4;
  auto host_block = [&](unsigned char** at) -> bool {
    if (c.backend == B200KV_ARENA_DEVICE) {
      void* pinned = nullptr;
      if (CheckCuda(cudaMallocHost(&pinned, e->staging_bytes), "engine staging (pinned)") != B200KV_OK) return false;
      *at = static_cast<unsigned char*>(pinned);
    } else {
      *at = new (std::nothrow) unsigned char[e->staging_bytes];
      if (*at == nullptr) return false;
    }
    std::memset(*at, 0, e->staging_bytes);
    return true;
  };
  for (b200kv_engine::Staging& block : e->stagings) {
    if (!host_block(&block.at)) return fail();
    if (c.backend == B200KV_ARENA_DEVICE &&
        CheckCuda(cudaEventCreateWithFlags(&block.uploaded, cudaEventDisableTiming), "engine staging (event)") != B200KV_OK) {
      return fail();
    }
  }
  if (!host_block(&e->captured)) return fail();
  e->pool = b200kv_block_pool_create(c.num_blocks, c.block_size, c.max_seqs, c.max_blocks_per_seq, nullptr);
  if (e->pool == nullptr) return fail();
  e->step_seq_ids.resize(static_cast<size_t>(c.max_seqs));
  e->step_grown.resize(static_cast<size_t>(c.max_seqs));
  e->moves.resize(static_cast<size_t>(c.num_blocks) * 3);
  if (b200kv_arena_seal(e->arena) != B200KV_OK) return fail();
  return e;
}

extern "C" void b200kv_engine_destroy(b200kv_engine* e) {
  if (e == nullptr) return;
  if (e->pool != nullptr) b200kv_block_pool_destroy(e->pool);
  auto free_block = [&](unsigned char* at) {
    if (at == nullptr) return;
    if (e->cfg.backend == B200KV_ARENA_DEVICE) cudaFreeHost(at); else delete[] at;
  };
  for (b200kv_engine::Staging& block : e->stagings) {
    if (block.uploaded != nullptr) cudaEventDestroy(block.uploaded);
    free_block(block.at);
  }
  free_block(e->captured);
  if (e->arena != nullptr) b200kv_arena_destroy(e->arena);
  delete e;
}

extern "C" const b200kv_arena* b200kv_engine_arena(const b200kv_engine* e) { return e ? e->arena : nullptr; }
extern "C" const b200kv_kv_cache* b200kv_engine_cache(const b200kv_engine* e) { return e ? &e->cache : nullptr; }
extern "C" const b200kv_block_pool* b200kv_engine_block_pool(const b200kv_engine* e) { return e ? e->pool : nullptr; }
extern "C" b200kv_status_word* b200kv_engine_status(const b200kv_engine* e) { return e ? e->d_status : nullptr; }

extern "C" int32_t b200kv_engine_admit(b200kv_engine* e, int32_t seq) {
  if (e == nullptr) return B200KV_ERR_NULLPTR;
  if (e->in_step) return Refuse("engine_admit: a step is in flight");
  return b200kv_block_pool_admit(e->pool, seq);
}

extern "C" int32_t b200kv_engine_release(b200kv_engine* e, int32_t seq) {
  if (e == nullptr) return B200KV_ERR_NULLPTR;
  if (e->in_step) return Refuse("engine_release: a step is in flight");
  return b200kv_block_pool_release(e->pool, seq);
}

extern "C" int32_t b200kv_engine_begin_step(b200kv_engine* e, const int32_t* seqs, const int32_t* new_tokens,
                                            int32_t n_seqs, void* stream) {
  if (e == nullptr || seqs == nullptr) {
    SetLastError("engine_begin_step: engine and seqs must be non-null");
    return B200KV_ERR_NULLPTR;
  }
  if (e->in_step) return Refuse("engine_begin_step: the previous step has not ended");
  if (n_seqs <= 0 || n_seqs > e->cfg.max_seqs) {
    SetLastError("engine_begin_step: %d sequences outside [1, %d]", n_seqs, e->cfg.max_seqs);
    return B200KV_ERR_INVALID;
  }
  // PLAN: the whole step must fit (tokens per step, blocks per sequence, free blocks) before anything changes.
  int64_t total_new = 0, blocks_needed = 0;
  for (int32_t i = 0; i < n_seqs; ++i) {
    const int32_t n = new_tokens != nullptr ? new_tokens[i] : 1;
    const int32_t len = b200kv_block_pool_seq_len(e->pool, seqs[i]);
    if (n < 1 || len < 0) {
      SetLastError("engine_begin_step: sequence %d (entry %d) is not admitted, or grows by %d tokens", seqs[i], i, n);
      return B200KV_ERR_INVALID;
    }
    for (int32_t j = 0; j < i; ++j) {
      if (seqs[j] == seqs[i]) {
        SetLastError("engine_begin_step: sequence %d appears twice in the step", seqs[i]);
        return B200KV_ERR_INVALID;
      }
    }
    const int64_t bs = e->cfg.block_size;
    const int64_t have = (len + bs - 1) / bs, want = (static_cast<int64_t>(len) + n + bs - 1) / bs;
    if (want > e->cfg.max_blocks_per_seq) {
      SetLastError("engine_begin_step: sequence %d would need %lld blocks, its table row holds %d", seqs[i],
                   static_cast<long long>(want), e->cfg.max_blocks_per_seq);
      return B200KV_ERR_INVALID;
    }
    blocks_needed += want - have;
    total_new += n;
  }
  if (total_new > e->cfg.max_step_tokens || blocks_needed > b200kv_block_pool_free_count(e->pool)) {
    SetLastError("engine_begin_step: the step appends %lld tokens (at most %d) and needs %lld free blocks (%d free)",
                 static_cast<long long>(total_new), e->cfg.max_step_tokens, static_cast<long long>(blocks_needed),
                 b200kv_block_pool_free_count(e->pool));
    return B200KV_ERR_INVALID;
  }
  if (int32_t rc = TakeStaging(e)) return rc;
  // COMMIT: grow, and mirror the step into the pinned block: table rows in step order, lengths, slots.
  int32_t* s_table = reinterpret_cast<int32_t*>(e->staging + e->table_off);
  int32_t* s_slots = reinterpret_cast<int32_t*>(e->staging + e->slots_off);
  int32_t* s_lens = reinterpret_cast<int32_t*>(e->staging + e->lens_off);
  const int32_t* table = b200kv_block_pool_table(e->pool);
  int32_t at = 0;
  for (int32_t i = 0; i < n_seqs; ++i) {
    const int32_t n = new_tokens != nullptr ? new_tokens[i] : 1;
    if (int32_t rc = b200kv_block_pool_grow(e->pool, seqs[i], n, s_slots + at)) return rc;  // cannot fail after the plan
    at += n;
    std::memcpy(s_table + static_cast<size_t>(i) * e->cfg.max_blocks_per_seq,
                table + static_cast<size_t>(seqs[i]) * e->cfg.max_blocks_per_seq,
                static_cast<size_t>(e->cfg.max_blocks_per_seq) * 4);
    s_lens[i] = b200kv_block_pool_seq_len(e->pool, seqs[i]);
    e->step_seq_ids[static_cast<size_t>(i)] = seqs[i];
    e->step_grown[static_cast<size_t>(i)] = n;
  }
  for (int32_t i = at; i < e->cfg.max_step_tokens; ++i) s_slots[i] = -1;  // padding rows write nothing
  e->step_shares = PlanQueries(e, n_seqs, at);
  e->allocations_at_begin = b200kv_arena_allocations(e->arena);
  e->step_seqs = n_seqs;
  e->step_tokens = at;
  // ONE upload per step: the queries, the table rows, the slots and the lengths lie in the arena in this order. An upload
  // that fails takes the step's growth back: the call changed nothing.
  const int32_t rc = Upload(e, e->step_shares ? 0 : e->table_off, static_cast<cudaStream_t>(stream));
  if (rc != B200KV_OK) {
    for (int32_t i = n_seqs - 1; i >= 0; --i) b200kv_block_pool_ungrow(e->pool, seqs[i], e->step_grown[static_cast<size_t>(i)]);
    return rc;
  }
  e->in_step = true;
  return B200KV_OK;
}

extern "C" int32_t b200kv_engine_abort_step(b200kv_engine* e) {
  if (e == nullptr) return B200KV_ERR_NULLPTR;
  if (!e->in_step) return Refuse("engine_abort_step: no step in flight");
  // The step's growth is taken back newest first, which restores tables, lengths and the free list exactly.
  // Rows the step's launches already wrote lie beyond every sequence's length and mean nothing.
  for (int32_t i = e->step_seqs - 1; i >= 0; --i) {
    if (int32_t rc = b200kv_block_pool_ungrow(e->pool, e->step_seq_ids[static_cast<size_t>(i)], e->step_grown[static_cast<size_t>(i)])) {
      return rc;
    }
  }
  e->in_step = false;
  return b200kv_block_pool_validate(e->pool);
}

extern "C" int32_t b200kv_engine_layer_append(b200kv_engine* e, int32_t layer, const void* kv_a, int64_t kv_a_stride,
                                              const void* gamma, const void* cos, int64_t cos_stride, const void* sin,
                                              int64_t sin_stride, void* q_rope, int64_t q_token_stride,
                                              int64_t q_head_stride, void* stream) {
  if (e == nullptr) return B200KV_ERR_NULLPTR;
  if (!e->in_step) return Refuse("engine_layer_append: no step in flight");
  b200kv_producer_args a{};
  if (int32_t rc = b200kv_kv_cache_layer_view(e->arena, &e->cache, layer, &a.pool)) return rc;
  a.kv_a = kv_a;
  a.kv_a_stride = kv_a_stride;
  a.gamma = gamma;
  a.eps = e->cfg.eps;
  a.cos = cos;
  a.cos_stride = cos_stride;
  a.sin = sin;
  a.sin_stride = sin_stride;
  a.slot_mapping = e->d_slots;
  a.n_tokens = e->step_tokens;
  a.q_rope = q_rope;
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.heads = q_rope != nullptr ? B200KV_HEADS : 0;
  return b200kv_append_fused(&a, stream, e->d_status);
}

extern "C" int32_t b200kv_engine_layer_attend(b200kv_engine* e, int32_t layer, const void* q, int64_t q_seq_stride,
                                              int64_t q_head_stride, void* out, void* out_fp8, void* out_scales,
                                              void* stream) {
  if (e == nullptr) return B200KV_ERR_NULLPTR;
  if (!e->in_step) return Refuse("engine_layer_attend: no step in flight");
  if (out_fp8 != nullptr && out_scales == nullptr) return Refuse("engine_layer_attend: out_fp8 without out_scales");
  // (one token a sequence, and rows that only the other entry point takes: not a reason to refuse the step)
  const bool fits = ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0 && q_seq_stride % 8 == 0 && q_head_stride % 8 == 0;
  if (e->step_shares && (fits || e->step_tokens != e->step_seqs)) {
    b200kv_shared_args a{};
    if (int32_t rc = b200kv_kv_cache_layer_view(e->arena, &e->cache, layer, &a.pool)) return rc;
    const int64_t stride = e->cfg.max_step_tokens;
    a.q = q;
    a.q_seq_stride = q_seq_stride;
    a.q_head_stride = q_head_stride;
    a.block_table = e->d_table;
    a.max_blocks = e->cfg.max_blocks_per_seq;
    a.table_rows = e->cfg.max_seqs;
    a.kv_len = e->d_queries;
    a.leader = e->d_queries + stride;
    a.shared_len = e->d_queries + 2 * stride;
    a.table_index = e->d_queries + 3 * stride;
    a.batch = e->step_tokens;
    a.heads = B200KV_HEADS;
    a.block_size = e->cfg.block_size;
    a.scale = e->cfg.scale;
    a.out = out;
    a.workspace = b200kv_arena_workspace(e->arena);
    a.workspace_bytes = static_cast<size_t>(b200kv_arena_workspace_bytes(e->arena));
    a.flags = B200KV_DECODE_STABLE_TABLES;
    a.out_fp8 = out_fp8;
    a.out_scale = out_fp8 != nullptr ? out_scales : nullptr;
    if (int32_t rc = b200kv_arena_workspace_fits(e->arena, b200kv_mla_decode_shared_workspace_bytes(a.batch, a.heads))) return rc;
    return b200kv_mla_decode_shared(&a, stream, e->d_status);
  }
  b200kv_decode_args a{};
  if (int32_t rc = b200kv_kv_cache_layer_view(e->arena, &e->cache, layer, &a.pool)) return rc;
  a.q = q;
  a.q_seq_stride = q_seq_stride;
  a.q_head_stride = q_head_stride;
  a.block_table = e->d_table;
  a.max_blocks = e->cfg.max_blocks_per_seq;
  a.kv_len = e->d_lens;
  a.batch = e->step_seqs;
  a.heads = B200KV_HEADS;
  a.block_size = e->cfg.block_size;
  a.scale = e->cfg.scale;
  a.out = out;
  a.workspace = b200kv_arena_workspace(e->arena);
  a.workspace_bytes = static_cast<size_t>(b200kv_arena_workspace_bytes(e->arena));
  a.variant = B200KV_DECODE_AUTO;
  // The step's table and lengths were uploaded before the first layer; from the second layer on the kernel
  // before this one on the stream is the producer, which does not write them.
  a.flags = B200KV_DECODE_STABLE_TABLES;
  // Stage 10, the attention output [sequences, 64 x 512] as FP8 E4M3 with one E8M0 scale per 32 values, rides in
  // the attention call: the kernel that writes `out` quantises what it writes.
  a.out_fp8 = out_fp8;
  a.out_scale = out_fp8 != nullptr ? out_scales : nullptr;
  if (int32_t rc = b200kv_arena_workspace_fits(e->arena, b200kv_mla_decode_workspace_bytes(a.batch, a.heads, 0))) return rc;
  return b200kv_mla_decode(&a, stream, e->d_status);
}

extern "C" int32_t b200kv_engine_fork(b200kv_engine* e, int32_t src, int32_t dst, int32_t n_tokens, void* stream) {
  if (e == nullptr) return B200KV_ERR_NULLPTR;
  if (e->in_step) return Refuse("engine_fork: a step is in flight");
  int32_t move[3];
  if (int32_t rc = b200kv_block_pool_fork(e->pool, src, dst, n_tokens, move)) return rc;
  if (move[0] >= 0) {
    if (int32_t rc = CopyMoves(e, move, 1, stream)) {
      b200kv_block_pool_ungrow(e->pool, dst, move[2]);  // (its own block first, to the front of the free list)
      b200kv_block_pool_release(e->pool, dst);
      return rc;
    }
  }
  return B200KV_OK;
}

extern "C" int32_t b200kv_engine_trim(b200kv_engine* e, int32_t seq, int32_t n_tokens, void* stream) {
  if (e == nullptr) return B200KV_ERR_NULLPTR;
  if (e->in_step) return Refuse("engine_trim: a step is in flight");
  const int32_t len = b200kv_block_pool_seq_len(e->pool, seq);
  if (len < 0 || n_tokens < 0 || n_tokens > len) {
    SetLastError("engine_trim: sequence %d holds %d tokens (-1: not admitted), %d to take back", seq, len, n_tokens);
    return B200KV_ERR_INVALID;
  }
  const int32_t left = len - n_tokens;
  if (n_tokens > 0 && left % e->cfg.block_size != 0) {  // the block that will be half filled is the sequence's own from here on
    const int32_t index = left / e->cfg.block_size;
    const int32_t block = b200kv_block_pool_table(e->pool)[static_cast<size_t>(seq) * e->cfg.max_blocks_per_seq + index];
    int32_t move[3];
    // (in a full pool the copy goes into a block that this call empties)
    const bool from_behind = b200kv_block_pool_ref_count(e->pool, block) > 1 && b200kv_block_pool_free_count(e->pool) == 0 &&
                             b200kv::TakeFromBehind(e->pool, seq, index, move);
    if (!from_behind) {
      if (int32_t rc = b200kv_block_pool_unshare(e->pool, seq, index, move)) return rc;
    }
    if (move[0] >= 0) {
      if (move[2] > left % e->cfg.block_size) move[2] = left % e->cfg.block_size;
      if (int32_t rc = CopyMoves(e, move, 1, stream)) {
        (from_behind ? b200kv::UndoTakeFromBehind : b200kv::UndoUnshare)(e->pool, seq, index, move);
        return rc;
      }
    }
  }
  return b200kv_block_pool_ungrow(e->pool, seq, n_tokens);
}

extern "C" int32_t b200kv_engine_compact(b200kv_engine* e, int32_t max_moves, void* stream) {
  if (e == nullptr) return -B200KV_ERR_NULLPTR;
  if (e->in_step) return -Refuse("engine_compact: a step is in flight");
  const int32_t most = max_moves < 0 || max_moves > e->cfg.num_blocks ? e->cfg.num_blocks : max_moves;
  const int32_t n = b200kv_block_pool_plan_compact(e->pool, most, e->moves.data());
  if (n <= 0) return n;
  if (int32_t rc = CopyMoves(e, e->moves.data(), n, stream)) return -rc;
  if (int32_t rc = b200kv_block_pool_apply_moves(e->pool, e->moves.data(), n)) return -rc;  // cannot fail after the plan
  return n;
}

extern "C" int32_t b200kv_engine_end_step(b200kv_engine* e) {
  if (e == nullptr) return B200KV_ERR_NULLPTR;
  if (!e->in_step) return Refuse("engine_end_step: no step in flight");
  e->in_step = false;
  ++e->steps;
  if (b200kv_arena_allocations(e->arena) != e->allocations_at_begin) {
    SetLastError("the step allocated device memory: %d allocations at its start, %d at its end",
                 e->allocations_at_begin, b200kv_arena_allocations(e->arena));
    return B200KV_ERR_INVALID;
  }
  return b200kv_block_pool_validate(e->pool);
}

extern "C" int64_t b200kv_engine_stats_json(const b200kv_engine* e, char* buffer, int64_t capacity) {
  if (e == nullptr) return -1;
  return b200kv_paged_attention_stats_json(e->cfg.num_blocks, e->cfg.layers, b200kv::StoredTokens(e->pool), e->cfg.block_size,
                                           buffer, capacity);
}
