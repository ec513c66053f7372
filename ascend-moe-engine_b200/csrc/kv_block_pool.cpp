// Host bookkeeping for the paged KV pool: a fixed-capacity block allocator with per-sequence block
// tables, plus the reservation arithmetic of the reference arena manager.
//
// Everything is sized at create time and nothing allocates afterwards, the way the reference seals
// its arena before the decode loop (src/memory/static_arena.cpp:301-304, and the zero-allocation
// assertions of src/pipeline/pipeline.cpp:502-503). A call either completes or changes nothing
// (plan, then commit), and Validate() states the failing arithmetic, after the pattern of the
// reference's expert slot pool (src/memory/exclusive_staging.cpp:313-399, 529-572).
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <iomanip>
#include <locale>
#include <mutex>
#include <new>
#include <sstream>
#include <string>

#include "b200kv.h"

namespace b200kv {
void SetLastError(const char* fmt, ...);
}

using b200kv::SetLastError;

struct b200kv_block_pool {
  int32_t num_blocks;
  int32_t block_size;
  int32_t max_seqs;
  int32_t max_blocks_per_seq;
  // Free list: a ring of block ids; [head, head + free_count) modulo num_blocks are free, oldest first.
  int32_t* ring;
  int32_t head;
  int32_t free_count;
  int32_t* table;        // [max_seqs][max_blocks_per_seq], unused entries 0
  int32_t* lens;         // tokens per sequence
  int32_t* used_blocks;  // table entries in use per sequence
  uint8_t* live;
  int32_t* refs;         // [num_blocks] table entries that name the block: more than one once a sequence has been forked
  int32_t* scratch;      // [num_blocks] for Validate, the statistics and compacting, under scratch_mutex: who only looks may be another thread
  mutable std::mutex scratch_mutex;
};

extern "C" b200kv_block_pool* b200kv_block_pool_create(int32_t num_blocks, int32_t block_size, int32_t max_seqs,
                                                       int32_t max_blocks_per_seq, const int32_t* free_order) {
  if (num_blocks <= 0 || block_size <= 0 || max_seqs <= 0 || max_blocks_per_seq <= 0 ||
      static_cast<int64_t>(num_blocks) * block_size > INT32_MAX) {
    SetLastError("block pool refused: blocks %d, block_size %d, max_seqs %d, max_blocks_per_seq %d "
                 "(all > 0, blocks*block_size < 2^31 so slots fit int32)",
                 num_blocks, block_size, max_seqs, max_blocks_per_seq);
    return nullptr;
  }
  auto* pool = new (std::nothrow) b200kv_block_pool();
  if (pool == nullptr) return nullptr;
  pool->num_blocks = num_blocks;
  pool->block_size = block_size;
  pool->max_seqs = max_seqs;
  pool->max_blocks_per_seq = max_blocks_per_seq;
  const size_t table_entries = static_cast<size_t>(max_seqs) * max_blocks_per_seq;
  pool->ring = new (std::nothrow) int32_t[num_blocks];
  pool->table = new (std::nothrow) int32_t[table_entries]();
  pool->lens = new (std::nothrow) int32_t[max_seqs]();
  pool->used_blocks = new (std::nothrow) int32_t[max_seqs]();
  pool->live = new (std::nothrow) uint8_t[max_seqs]();
  pool->refs = new (std::nothrow) int32_t[num_blocks]();
  pool->scratch = new (std::nothrow) int32_t[num_blocks]();
  if (!pool->ring || !pool->table || !pool->lens || !pool->used_blocks || !pool->live || !pool->refs || !pool->scratch) {
    SetLastError("block pool: host allocation failed");
    b200kv_block_pool_destroy(pool);
    return nullptr;
  }
  for (int32_t i = 0; i < num_blocks; ++i) {
    const int32_t id = free_order ? free_order[i] : i;
    if (id < 0 || id >= num_blocks || pool->scratch[id]) {
      SetLastError("block pool: free_order[%d] = %d is out of range or repeated", i, id);
      b200kv_block_pool_destroy(pool);
      return nullptr;
    }
    pool->scratch[id] = 1;
    pool->ring[i] = id;
  }
  pool->head = 0;
  pool->free_count = num_blocks;
  return pool;
}

extern "C" void b200kv_block_pool_destroy(b200kv_block_pool* pool) {
  if (pool == nullptr) return;
  delete[] pool->ring;
  delete[] pool->table;
  delete[] pool->lens;
  delete[] pool->used_blocks;
  delete[] pool->live;
  delete[] pool->refs;
  delete[] pool->scratch;
  delete pool;
}

namespace {
bool SeqInRange(const b200kv_block_pool* pool, int32_t seq, const char* what) {
  if (pool == nullptr) {
    SetLastError("%s: pool is null", what);
    return false;
  }
  if (seq < 0 || seq >= pool->max_seqs) {
    SetLastError("%s: sequence %d outside [0, %d)", what, seq, pool->max_seqs);
    return false;
  }
  return true;
}

int32_t TakeFree(b200kv_block_pool* pool) {
  const int32_t id = pool->ring[pool->head];
  pool->head = pool->head + 1 == pool->num_blocks ? 0 : pool->head + 1;
  --pool->free_count;
  pool->refs[id] = 1;
  return id;
}

// One table entry less for a block; the last one gives it back, to the front of the free list or to its end.
void Drop(b200kv_block_pool* pool, int32_t id, bool to_front) {
  if (--pool->refs[id] > 0) return;
  if (to_front) {
    pool->head = pool->head == 0 ? pool->num_blocks - 1 : pool->head - 1;
    pool->ring[pool->head] = id;
  } else {
    int32_t tail = pool->head + pool->free_count;
    if (tail >= pool->num_blocks) tail -= pool->num_blocks;
    pool->ring[tail] = id;
  }
  ++pool->free_count;
}

int32_t RowsIn(const b200kv_block_pool* pool, int32_t seq, int32_t index) {  // tokens of the sequence in its block `index`
  const int64_t left = pool->lens[seq] - static_cast<int64_t>(index) * pool->block_size;
  return static_cast<int32_t>(left < pool->block_size ? left : pool->block_size);
}

// scratch[block]: the rows that mean something, those of the sequence with the most tokens there. The caller holds scratch_mutex.
void MarkRows(const b200kv_block_pool* pool) {
  std::memset(pool->scratch, 0, static_cast<size_t>(pool->num_blocks) * sizeof(int32_t));
  for (int32_t s = 0; s < pool->max_seqs; ++s) {
    const int32_t* row = pool->table + static_cast<size_t>(s) * pool->max_blocks_per_seq;
    for (int32_t i = 0; i < pool->used_blocks[s]; ++i) {
      const int32_t rows = RowsIn(pool, s, i);
      if (rows > pool->scratch[row[i]]) pool->scratch[row[i]] = rows;
    }
  }
}

void NoMove(int32_t* move) {
  move[0] = move[1] = -1;
  move[2] = 0;
}
}  // namespace

extern "C" int32_t b200kv_block_pool_admit(b200kv_block_pool* pool, int32_t seq) {
  if (!SeqInRange(pool, seq, "admit")) return pool ? B200KV_ERR_INVALID : B200KV_ERR_NULLPTR;
  if (pool->live[seq]) {
    SetLastError("admit: sequence %d is already live with %d tokens", seq, pool->lens[seq]);
    return B200KV_ERR_INVALID;
  }
  pool->live[seq] = 1;
  pool->lens[seq] = 0;
  pool->used_blocks[seq] = 0;
  return B200KV_OK;
}

extern "C" int32_t b200kv_block_pool_grow(b200kv_block_pool* pool, int32_t seq, int32_t n_tokens,
                                          int32_t* slots_out) {
  if (!SeqInRange(pool, seq, "grow")) return pool ? B200KV_ERR_INVALID : B200KV_ERR_NULLPTR;
  if (!pool->live[seq] || n_tokens < 0 || (n_tokens > 0 && slots_out == nullptr)) {
    SetLastError("grow: sequence %d live=%d, n_tokens %d, slots_out %p", seq, static_cast<int>(pool->live[seq]),
                 n_tokens, static_cast<void*>(slots_out));
    return B200KV_ERR_INVALID;
  }
  // Plan: how many blocks the new length needs, refused as a whole when the row or the free list is short.
  const int64_t new_len = static_cast<int64_t>(pool->lens[seq]) + n_tokens;
  const int64_t need = (new_len + pool->block_size - 1) / pool->block_size;
  const int64_t have = pool->used_blocks[seq];
  if (need > pool->max_blocks_per_seq) {
    SetLastError("grow: sequence %d would need %lld blocks for %lld tokens, table row holds %d", seq,
                 static_cast<long long>(need), static_cast<long long>(new_len), pool->max_blocks_per_seq);
    return B200KV_ERR_INVALID;
  }
  if (need - have > pool->free_count) {
    SetLastError("grow: sequence %d needs %lld more blocks, %d free of %d", seq, static_cast<long long>(need - have),
                 pool->free_count, pool->num_blocks);
    return B200KV_ERR_INVALID;
  }
  int32_t* row = pool->table + static_cast<size_t>(seq) * pool->max_blocks_per_seq;
  if (n_tokens > 0 && pool->lens[seq] % pool->block_size != 0 && pool->refs[row[have - 1]] > 1) {
    SetLastError("grow: the last block of sequence %d (%d, half filled) belongs to others too: unshare it first", seq, row[have - 1]);
    return B200KV_ERR_INVALID;
  }
  // Commit.
  for (int64_t i = have; i < need; ++i) row[i] = TakeFree(pool);
  pool->used_blocks[seq] = static_cast<int32_t>(need);
  const int32_t old_len = pool->lens[seq];
  for (int32_t k = 0; k < n_tokens; ++k) {
    const int32_t j = old_len + k;
    slots_out[k] = row[j / pool->block_size] * pool->block_size + j % pool->block_size;
  }
  pool->lens[seq] = static_cast<int32_t>(new_len);
  return B200KV_OK;
}

// Takes back the last n_tokens of a sequence and returns the blocks that empties (and no other sequence holds) to the FRONT of the
// free list, newest first: undoing the most recent grows in reverse order restores tables, lengths and the free
// list exactly (a step that is abandoned half way leaves no trace).
extern "C" int32_t b200kv_block_pool_ungrow(b200kv_block_pool* pool, int32_t seq, int32_t n_tokens) {
  if (!SeqInRange(pool, seq, "ungrow")) return pool ? B200KV_ERR_INVALID : B200KV_ERR_NULLPTR;
  if (!pool->live[seq] || n_tokens < 0 || n_tokens > pool->lens[seq]) {
    SetLastError("ungrow: sequence %d live=%d holds %d tokens, %d to take back", seq, static_cast<int>(pool->live[seq]),
                 pool->lens[seq], n_tokens);
    return B200KV_ERR_INVALID;
  }
  const int32_t new_len = pool->lens[seq] - n_tokens;
  const int32_t keep = (new_len + pool->block_size - 1) / pool->block_size;
  int32_t* row = pool->table + static_cast<size_t>(seq) * pool->max_blocks_per_seq;
  for (int32_t i = pool->used_blocks[seq] - 1; i >= keep; --i) {
    Drop(pool, row[i], true);
    row[i] = 0;
  }
  pool->used_blocks[seq] = keep;
  pool->lens[seq] = new_len;
  return B200KV_OK;
}

extern "C" int32_t b200kv_block_pool_release(b200kv_block_pool* pool, int32_t seq) {
  if (!SeqInRange(pool, seq, "release")) return pool ? B200KV_ERR_INVALID : B200KV_ERR_NULLPTR;
  if (!pool->live[seq]) {
    SetLastError("release: sequence %d is not live", seq);
    return B200KV_ERR_INVALID;
  }
  int32_t* row = pool->table + static_cast<size_t>(seq) * pool->max_blocks_per_seq;
  for (int32_t i = 0; i < pool->used_blocks[seq]; ++i) {
    Drop(pool, row[i], false);
    row[i] = 0;
  }
  pool->used_blocks[seq] = 0;
  pool->lens[seq] = 0;
  pool->live[seq] = 0;
  return B200KV_OK;
}

// A sequence that begins as the first n_tokens of another: whole blocks are held by both, the half-filled one behind them is a block
// of its own, whose rows are the caller's to copy.
extern "C" int32_t b200kv_block_pool_fork(b200kv_block_pool* pool, int32_t src, int32_t dst, int32_t n_tokens, int32_t* move_out) {
  if (!SeqInRange(pool, src, "fork") || !SeqInRange(pool, dst, "fork")) return pool ? B200KV_ERR_INVALID : B200KV_ERR_NULLPTR;
  if (move_out == nullptr) {
    SetLastError("fork: move_out is null");
    return B200KV_ERR_NULLPTR;
  }
  if (!pool->live[src] || pool->live[dst] || n_tokens < -1 || n_tokens > pool->lens[src]) {
    SetLastError("fork: sequence %d live=%d with %d tokens, %d asked for, into sequence %d live=%d", src, static_cast<int>(pool->live[src]),
                 pool->lens[src], n_tokens, dst, static_cast<int>(pool->live[dst]));
    return B200KV_ERR_INVALID;
  }
  const int32_t n = n_tokens < 0 ? pool->lens[src] : n_tokens;
  const int32_t whole = n / pool->block_size, rest = n % pool->block_size;
  if (rest > 0 && pool->free_count == 0) {
    SetLastError("fork: %d tokens end inside a block, and none of %d is free for the copy", n, pool->num_blocks);
    return B200KV_ERR_INVALID;
  }
  const int32_t* from = pool->table + static_cast<size_t>(src) * pool->max_blocks_per_seq;
  int32_t* to = pool->table + static_cast<size_t>(dst) * pool->max_blocks_per_seq;
  for (int32_t i = 0; i < whole; ++i) {
    to[i] = from[i];
    ++pool->refs[from[i]];
  }
  NoMove(move_out);
  if (rest > 0) {
    to[whole] = TakeFree(pool);
    move_out[0] = from[whole];
    move_out[1] = to[whole];
    move_out[2] = rest;
  }
  pool->live[dst] = 1;
  pool->lens[dst] = n;
  pool->used_blocks[dst] = whole + (rest > 0 ? 1 : 0);
  return B200KV_OK;
}

// Gives a sequence a block of its own in place of its block `index`, if others hold that one too; its rows are the caller's to copy.
extern "C" int32_t b200kv_block_pool_unshare(b200kv_block_pool* pool, int32_t seq, int32_t index, int32_t* move_out) {
  if (!SeqInRange(pool, seq, "unshare")) return pool ? B200KV_ERR_INVALID : B200KV_ERR_NULLPTR;
  if (move_out == nullptr) {
    SetLastError("unshare: move_out is null");
    return B200KV_ERR_NULLPTR;
  }
  if (!pool->live[seq] || index < 0 || index >= pool->used_blocks[seq]) {
    SetLastError("unshare: sequence %d live=%d has %d blocks, not one with index %d", seq, static_cast<int>(pool->live[seq]), pool->used_blocks[seq],
                 index);
    return B200KV_ERR_INVALID;
  }
  NoMove(move_out);
  int32_t* entry = pool->table + static_cast<size_t>(seq) * pool->max_blocks_per_seq + index;
  if (pool->refs[*entry] == 1) return B200KV_OK;
  if (pool->free_count == 0) {
    SetLastError("unshare: no block of %d is free for the copy of block %d", pool->num_blocks, *entry);
    return B200KV_ERR_INVALID;
  }
  move_out[0] = *entry;
  move_out[2] = RowsIn(pool, seq, index);
  --pool->refs[*entry];
  *entry = TakeFree(pool);
  move_out[1] = *entry;
  return B200KV_OK;
}

// Not part of the C ABI: for the engine.
namespace b200kv {
// Tokens that the blocks hold, those of several sequences once.
int64_t StoredTokens(const b200kv_block_pool* pool) {
  std::lock_guard<std::mutex> lock(pool->scratch_mutex);
  MarkRows(pool);
  int64_t tokens = 0;
  for (int32_t id = 0; id < pool->num_blocks; ++id) tokens += pool->scratch[id];
  return tokens;
}

// Unshare without a free block, for a sequence that is about to lose its tokens behind block `index`: the last block there that only
// this sequence holds changes places with the common one, which the ungrow that follows lets go of. False: there is none.
bool TakeFromBehind(b200kv_block_pool* pool, int32_t seq, int32_t index, int32_t* move_out) {
  int32_t* row = pool->table + static_cast<size_t>(seq) * pool->max_blocks_per_seq;
  for (int32_t i = pool->used_blocks[seq] - 1; i > index; --i) {
    if (pool->refs[row[i]] != 1) continue;
    move_out[0] = row[index];
    move_out[1] = row[i];
    move_out[2] = RowsIn(pool, seq, index);
    row[index] = move_out[1];
    row[i] = move_out[0];
    return true;
  }
  return false;
}

// Undoes it when its copy could not be made.
void UndoTakeFromBehind(b200kv_block_pool* pool, int32_t seq, int32_t index, const int32_t* move) {
  int32_t* row = pool->table + static_cast<size_t>(seq) * pool->max_blocks_per_seq;
  for (int32_t i = index + 1; i < pool->used_blocks[seq]; ++i) {
    if (row[i] == move[0]) row[i] = move[1];
  }
  row[index] = move[0];
}

// Undoes the unshare that has just been made, when its copy could not be.
void UndoUnshare(b200kv_block_pool* pool, int32_t seq, int32_t index, const int32_t* move) {
  if (move[0] < 0) return;
  Drop(pool, move[1], true);
  pool->table[static_cast<size_t>(seq) * pool->max_blocks_per_seq + index] = move[0];
  ++pool->refs[move[0]];
}
}  // namespace b200kv

// The used blocks with the highest ids, each with the lowest free id below it: done to the end, the used blocks are 0 .. used - 1.
extern "C" int32_t b200kv_block_pool_plan_compact(b200kv_block_pool* pool, int32_t max_moves, int32_t* moves_out) {
  if (pool == nullptr) {
    SetLastError("plan_compact: pool is null");
    return -B200KV_ERR_NULLPTR;
  }
  if (max_moves < 0 || (max_moves > 0 && moves_out == nullptr)) {
    SetLastError("plan_compact: %d moves into %p", max_moves, static_cast<void*>(moves_out));
    return moves_out == nullptr ? -B200KV_ERR_NULLPTR : -B200KV_ERR_INVALID;
  }
  std::lock_guard<std::mutex> lock(pool->scratch_mutex);
  MarkRows(pool);
  int32_t n = 0, to = 0;
  for (int32_t from = pool->num_blocks - 1; n < max_moves; --from) {
    while (from > to && pool->refs[from] == 0) --from;
    while (to < from && pool->refs[to] > 0) ++to;
    if (to >= from) break;
    moves_out[3 * n] = from;
    moves_out[3 * n + 1] = to++;
    moves_out[3 * n + 2] = pool->scratch[from];
    ++n;
  }
  return n;
}

// The tables after the moves: every entry of a source names its destination, the sources are free. The free list is in the order of
// the ids afterwards.
extern "C" int32_t b200kv_block_pool_apply_moves(b200kv_block_pool* pool, const int32_t* moves, int32_t n_moves) {
  if (pool == nullptr || (n_moves > 0 && moves == nullptr)) {
    SetLastError("apply_moves: pool and moves must be non-null");
    return B200KV_ERR_NULLPTR;
  }
  std::lock_guard<std::mutex> lock(pool->scratch_mutex);
  // Plan: sources in use, destinations free, none twice. scratch[id]: 0 untouched, destination + 1 of a source, -1 a destination.
  std::memset(pool->scratch, 0, static_cast<size_t>(pool->num_blocks) * sizeof(int32_t));
  for (int32_t i = 0; i < n_moves; ++i) {
    const int32_t from = moves[3 * i], to = moves[3 * i + 1];
    if (from < 0 || from >= pool->num_blocks || to < 0 || to >= pool->num_blocks || pool->refs[from] == 0 || pool->refs[to] != 0 ||
        pool->scratch[from] != 0 || pool->scratch[to] != 0) {
      SetLastError("apply_moves: move %d from block %d to block %d (a block in use to a free one, no block twice)", i, from, to);
      return B200KV_ERR_INVALID;
    }
    pool->scratch[from] = to + 1;
    pool->scratch[to] = -1;
  }
  if (n_moves < 0) {
    SetLastError("apply_moves: %d moves", n_moves);
    return B200KV_ERR_INVALID;
  }
  if (n_moves == 0) return B200KV_OK;
  for (int32_t s = 0; s < pool->max_seqs; ++s) {
    int32_t* row = pool->table + static_cast<size_t>(s) * pool->max_blocks_per_seq;
    for (int32_t i = 0; i < pool->used_blocks[s]; ++i) {
      if (pool->scratch[row[i]] > 0) row[i] = pool->scratch[row[i]] - 1;
    }
  }
  for (int32_t i = 0; i < n_moves; ++i) {
    pool->refs[moves[3 * i + 1]] = pool->refs[moves[3 * i]];
    pool->refs[moves[3 * i]] = 0;
  }
  pool->head = 0;
  int32_t n = 0;
  for (int32_t id = 0; id < pool->num_blocks; ++id) {
    if (pool->refs[id] == 0) pool->ring[n++] = id;
  }
  return B200KV_OK;
}

// Neighbours, two by two, whose table rows begin with the same blocks. Only whole blocks of both count.
extern "C" int64_t b200kv_find_shared(const int32_t* table, int64_t max_blocks, const int32_t* kv_len, int32_t n_seqs, int32_t block_size,
                                      int32_t* leader_out, int32_t* shared_len_out) {
  if (table == nullptr || kv_len == nullptr || leader_out == nullptr || shared_len_out == nullptr) {
    SetLastError("find_shared: table, kv_len, leader_out and shared_len_out must be non-null");
    return -B200KV_ERR_NULLPTR;
  }
  if (n_seqs < 0 || block_size <= 0 || max_blocks <= 0) {
    SetLastError("find_shared refused: %d sequences, blocks of %d rows, %lld blocks a row", n_seqs, block_size, static_cast<long long>(max_blocks));
    return -B200KV_ERR_INVALID;
  }
  int64_t common = 0;
  for (int32_t i = 0; i < n_seqs; ++i) {
    leader_out[i] = i;
    shared_len_out[i] = 0;
  }
  for (int32_t i = 0; i + 1 < n_seqs; ++i) {
    const int32_t *a = table + i * max_blocks, *b = a + max_blocks;
    const int64_t shorter = (kv_len[i] < kv_len[i + 1] ? kv_len[i] : kv_len[i + 1]) / block_size;
    const int64_t most = shorter < max_blocks ? shorter : max_blocks;
    int64_t blocks = 0;
    while (blocks < most && a[blocks] == b[blocks]) ++blocks;
    if (blocks == 0) continue;
    leader_out[i + 1] = i;
    shared_len_out[i] = shared_len_out[i + 1] = static_cast<int32_t>(blocks * block_size);
    common += shared_len_out[i];
    ++i;  // (the pair is done with)
  }
  return common;
}

extern "C" int32_t b200kv_block_pool_ref_count(const b200kv_block_pool* pool, int32_t block) {
  if (pool == nullptr || block < 0 || block >= pool->num_blocks) {
    SetLastError("ref_count: block %d outside the pool", block);
    return -1;
  }
  return pool->refs[block];
}

extern "C" int32_t b200kv_block_pool_free_count(const b200kv_block_pool* pool) {
  return pool ? pool->free_count : -1;
}

extern "C" int32_t b200kv_block_pool_seq_len(const b200kv_block_pool* pool, int32_t seq) {
  if (!SeqInRange(pool, seq, "seq_len")) return -1;
  return pool->live[seq] ? pool->lens[seq] : -1;
}

extern "C" const int32_t* b200kv_block_pool_table(const b200kv_block_pool* pool) {
  return pool ? pool->table : nullptr;
}

extern "C" const int32_t* b200kv_block_pool_lens(const b200kv_block_pool* pool) { return pool ? pool->lens : nullptr; }

extern "C" int32_t b200kv_block_pool_export_free(const b200kv_block_pool* pool, int32_t* out, int32_t capacity) {
  if (pool == nullptr || out == nullptr) return -1;
  int32_t n = 0;
  int32_t at = pool->head;
  for (; n < pool->free_count && n < capacity; ++n) {
    out[n] = pool->ring[at];
    at = at + 1 == pool->num_blocks ? 0 : at + 1;
  }
  return n;
}

extern "C" int32_t b200kv_block_pool_validate(const b200kv_block_pool* pool) {
  if (pool == nullptr) {
    SetLastError("validate: pool is null");
    return B200KV_ERR_NULLPTR;
  }
  std::lock_guard<std::mutex> lock(pool->scratch_mutex);
  std::memset(pool->scratch, 0, static_cast<size_t>(pool->num_blocks) * sizeof(int32_t));
  int64_t owned = 0;
  int32_t at = pool->head;
  for (int32_t i = 0; i < pool->free_count; ++i) {
    const int32_t id = pool->ring[at];
    if (id < 0 || id >= pool->num_blocks || pool->scratch[id] || pool->refs[id] != 0) {
      SetLastError("validate: free-list entry %d holds block %d (out of range, listed twice or in use)", i, id);
      return B200KV_ERR_INVALID;
    }
    pool->scratch[id] = -1;
    at = at + 1 == pool->num_blocks ? 0 : at + 1;
  }
  for (int32_t s = 0; s < pool->max_seqs; ++s) {
    const int32_t* row = pool->table + static_cast<size_t>(s) * pool->max_blocks_per_seq;
    if (!pool->live[s]) {
      if (pool->lens[s] != 0 || pool->used_blocks[s] != 0) {
        SetLastError("validate: idle sequence %d keeps %d tokens / %d blocks", s, pool->lens[s], pool->used_blocks[s]);
        return B200KV_ERR_INVALID;
      }
      continue;
    }
    const int64_t need = (static_cast<int64_t>(pool->lens[s]) + pool->block_size - 1) / pool->block_size;
    if (need != pool->used_blocks[s]) {
      SetLastError("validate: sequence %d has %d tokens -> ceil(%d/%d) = %lld blocks, table holds %d", s,
                   pool->lens[s], pool->lens[s], pool->block_size, static_cast<long long>(need), pool->used_blocks[s]);
      return B200KV_ERR_INVALID;
    }
    for (int32_t i = 0; i < pool->used_blocks[s]; ++i) {
      const int32_t id = row[i];
      if (id < 0 || id >= pool->num_blocks || pool->scratch[id] < 0) {
        SetLastError("validate: sequence %d entry %d holds block %d (out of range or free)", s, i, id);
        return B200KV_ERR_INVALID;
      }
      if (pool->scratch[id]++ == 0) ++owned;
    }
  }
  for (int32_t id = 0; id < pool->num_blocks; ++id) {
    const int32_t named = pool->scratch[id] < 0 ? 0 : pool->scratch[id];
    if (named != pool->refs[id]) {
      SetLastError("validate: block %d is named by %d table entries, %d are counted", id, named, pool->refs[id]);
      return B200KV_ERR_INVALID;
    }
  }
  if (owned + pool->free_count != pool->num_blocks) {
    SetLastError("validate: %lld blocks in tables + %d free != %d total", static_cast<long long>(owned),
                 pool->free_count, pool->num_blocks);
    return B200KV_ERR_INVALID;
  }
  return B200KV_OK;
}

extern "C" int32_t b200kv_plan_reservation(int64_t max_context, int64_t block_size, int64_t layers, int64_t max_seqs,
                                           int64_t tokens_per_step, b200kv_reservation* out) {
  if (out == nullptr) {
    SetLastError("plan_reservation: out is null");
    return B200KV_ERR_NULLPTR;
  }
  if (max_context <= 0 || block_size <= 0 || layers <= 0 || max_seqs <= 0 || tokens_per_step <= 0) {
    SetLastError("plan_reservation refused: context %lld, block_size %lld, layers %lld, seqs %lld, tokens/step %lld",
                 static_cast<long long>(max_context), static_cast<long long>(block_size),
                 static_cast<long long>(layers), static_cast<long long>(max_seqs),
                 static_cast<long long>(tokens_per_step));
    return B200KV_ERR_INVALID;
  }
  const int64_t blocks = (max_context + block_size - 1) / block_size;
  out->blocks_per_layer = blocks;
  out->total_blocks = blocks * layers;
  out->latent_bytes = layers * blocks * block_size * B200KV_LATENT_DIM * 2;
  out->rope_bytes = layers * blocks * block_size * B200KV_ROPE_DIM * 2;
  out->block_table_bytes = max_seqs * blocks * 4;
  out->slot_mapping_bytes = tokens_per_step * 4;
  return B200KV_OK;
}

extern "C" double b200kv_utilisation(int64_t active_tokens, int64_t blocks_per_layer, int64_t block_size) {
  const int64_t capacity = blocks_per_layer * block_size;
  return capacity > 0 ? static_cast<double>(active_tokens) / static_cast<double>(capacity) : 0.0;
}

// The "paged_attention" object of the reference's diagnostics file, key for key and with its number
// formatting (std::setprecision(12) in the classic locale; src/diagnostics/inference_stats.cpp:22, 42-47).
extern "C" int64_t b200kv_paged_attention_stats_json(int64_t blocks_per_layer, int64_t layers, int64_t active_tokens,
                                                     int64_t block_size, char* buffer, int64_t capacity) {
  std::ostringstream out;
  out.imbue(std::locale::classic());
  out << std::setprecision(12);
  out << "\"paged_attention\": {\n"
      << "    \"total_blocks_allocated\": " << blocks_per_layer * layers << ",\n"
      << "    \"active_context_tokens\": " << active_tokens << ",\n"
      << "    \"block_size\": " << block_size << ",\n"
      << "    \"kv_cache_utilization\": " << b200kv_utilisation(active_tokens, blocks_per_layer, block_size) << "\n  }";
  const std::string text = out.str();
  if (buffer != nullptr && capacity > 0) {
    const size_t n = text.size() < static_cast<size_t>(capacity - 1) ? text.size() : static_cast<size_t>(capacity - 1);
    std::memcpy(buffer, text.data(), n);
    buffer[n] = '\0';
  }
  return static_cast<int64_t>(text.size());
}
