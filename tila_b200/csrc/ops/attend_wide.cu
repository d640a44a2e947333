// Attention over a paged cache with a shared prefix: the wide form, for more
// than 16 rows of queries that see the same prefix, or 32 that see the same sequence.
//
// Up to 256 rows against one chunk of keys: GEMM-shaped, on the 5th-generation
// tensor cores.  A block has
//
//   * one or two softmax warpgroups, one row a thread (a row is a TMEM lane), each with
//     its own scores S (128 columns) and its own sums O in tensor memory;
//   * a copy warp that streams tiles of 128 keys, then of their values, through
//     one ring in shared memory: a TMA box for each page and each 64 elements of
//     the heads, so that a tile takes its pages from anywhere in the pool;
//   * an MMA warp that issues S = Q K^T and O += P V;
//   * two warps that look through the values of the tiles where some rows see keys
//     that others do not (new tokens): a value that is no number must not reach the
//     others through its weight of 0, so it is cleared there and put into the rows
//     that see it at the end.
//
// The prefix: two softmax warpgroups and one block a multiprocessor.  With more than
// 128 rows they hold two row tiles and share every tile of keys (half the traffic
// from L2, which at 128 rows a tile would bound: 64 KB for every 1024 cycles of MMA);
// with fewer, both hold the same rows and take the tiles in turn, and their results
// are joined at the end.  Either way the tensor core works for one while the other is
// in its softmax.  Sequences' own tokens: many blocks of few tiles, so one warpgroup
// and 128 rows a block, two blocks a multiprocessor, which also hide each other's
// beginnings and ends (11 us of a block's 15 at 4 tiles); where that is faster, they go
// through the prefix first and write the result itself.  Weights P (rounded to the
// values' type) go through tensor memory in the place of S.
//
// tcgen05 operations of one thread run in order: S of a warpgroup's next tile,
// issued behind P V of its last, overwrites P only after that was read, and its
// arrival means that P V is done, so that the warpgroup may scale O in place.  O
// is scaled only when a row's maximum grew by more than 2^8 (weights reach 256
// then; sums stay in 32 bits and f16 weights in range), rarely after the first
// tiles.
//
// Keys behind the end read whatever the page holds (even NaN): their scores are
// replaced before use, P V covers whole groups of 16 keys, and the MMA warp
// clears the values behind the end in the last group.

#include "attend.cuh"
#include "attend_wide.cuh"

#include <atomic>
#include <type_traits>

namespace tila_ops {
namespace {

using tila::TensorMap;

constexpr int kTile = 128;                       // keys of a tile, rows of a row tile
constexpr int kHalf = kTile * 128;               // bytes of 64 elements of a tile
constexpr float kGrowth = 8.f;                   // log2 of what weights may reach before O is scaled

// G softmax warpgroups: two, one block a multiprocessor, for the prefix; one, two blocks
// a multiprocessor, for sequences' own tokens.
template <int DP, int G> struct Wide {
  static constexpr int kThreads = G * 128 + 128;
  static constexpr int kBlocks = G == 2 ? 1 : 2;            // of a multiprocessor
  // Registers a thread at launch (65536 / (kBlocks * kThreads) in steps of 8), and what
  // the warpgroups keep of them: the softmax holds a whole row of scores.  The shares
  // add up to at most the total at launch (256 * 216 + 128 * 64 = 63488 of 384 * 168 =
  // 64512; 128 * 200 + 128 * 56 = 256 * 128); the host checks that the compiler gave the
  // kernel exactly those, since a warpgroup would otherwise wait for registers that do
  // not exist, and leaves the rows to the narrow form where it did not.
  static constexpr int kLaunchRegisters = G == 2 ? 168 : 128;
  static constexpr int kSoftmaxRegisters = G == 2 ? 216 : 200, kOtherRegisters = G == 2 ? 64 : 56;
  static_assert(G * 128 * kSoftmaxRegisters + 128 * kOtherRegisters <= kThreads * kLaunchRegisters, "registers");
  // Tensor memory: S, P and O of each warpgroup.  At 64 elements there is room for P
  // beside S: S of the next tile is issued as soon as the warpgroup has read S, and is
  // there when it comes back.
  static constexpr bool kEarly = DP == 64;
  static constexpr u32 kColumns = 256 * G;
  static constexpr u32 kWeightsAt = kEarly ? 128 * G : 0, kWeightsStep = kEarly ? 64 : 128;   // columns of P
  static constexpr u32 kSumsAt = kEarly ? 192 * G : 128 * G;                                  // columns of O
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kStages = G == 2 ? (DP == 128 ? 5 : 9) : (DP == 128 ? 2 : 5);
  static constexpr int kRing = G * kTileBytes;   // behind the query tiles
  static constexpr int kBytes = kRing + kStages * kTileBytes + 1024;   // 1024: alignment of swizzled tiles
  static constexpr int kRowFloats = DP + 4;      // of a staged result row: no two rows start in one bank
  static_assert(G * kTile * kRowFloats * 4 <= kRing + kStages * kTileBytes, "results are staged in queries and ring");
  static_assert(kBytes <= (G == 2 ? 226 : 112) * 1024, "shared memory of a block");
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// One lane of the warp, the same one each time, in a form that the compiler knows
// to be one: what it feeds to tcgen05 instructions stays in uniform registers.
__device__ __forceinline__ bool elected() {
  u32 one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

// A value that all lanes hold, as one that the compiler knows to be uniform.
__device__ __forceinline__ u32 uniform(u32 x) { return __shfl_sync(0xffffffffu, x, 0); }

// A bounded wait by a whole warp: all lanes go on, or none.
__device__ __forceinline__ bool warp_wait(u64 *bar, u32 parity, u32 *err, u32 where, int *dead) {
  return __all_sync(0xffffffffu, tila::mbar_wait(bar, parity, err, where, dead));
}

// First key of the tiles looked through whose value at an element is not a number,
// +inf, -inf.
constexpr int kNever = 0x7fffffff;
template <int DP> struct OddValues {
  int first[3][DP];
  int any;
};

// A row of O from tensor memory (zeros where nothing was added to it) times `mine`,
// plus `other` times the partner's row, to shared memory.
template <int DP>
__device__ __forceinline__ void write_row(u32 o_col, bool any, float mine, float other, const float *partner,
                                          float *dst) {
#pragma unroll 1
  for (int c = 0; c < DP; c += 32) {
    float o[32];
    tila::tmem_ld32(o_col + c, o);
    tila::tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (any) x = make_float4(o[i] * mine, o[i + 1] * mine, o[i + 2] * mine, o[i + 3] * mine);
      if (partner != nullptr) {
        const float4 y = *reinterpret_cast<const float4 *>(partner + c + i);
        x = make_float4(x.x + other * y.x, x.y + other * y.y, x.z + other * y.z, x.w + other * y.w);
      }
      *reinterpret_cast<float4 *>(dst + c + i) = x;
    }
  }
}

// The values cleared from the tiles, into the row of a token that sees `limit` keys.
template <int DP>
__device__ __noinline__ void put_odd(float *dst, const OddValues<DP> &odd, int limit) {
  for (int i = 0; i < DP; ++i) {
    const bool nan = odd.first[0][i] < limit, up = odd.first[1][i] < limit, down = odd.first[2][i] < limit;
    if (nan || (up && down)) dst[i] = __int_as_float(0x7fffffff);
    else if (up || down) dst[i] += up ? __builtin_huge_valf() : -__builtin_huge_valf();
  }
}

struct Barriers {
  u64 full[9], empty[9];
  u64 scores[2];      // S of a warpgroup's tile is there (and P V of its tile before)
  u64 taken[2];       // S has been read (kEarly)
  u64 weights[2];     // P is in tensor memory
  u64 summed[2];      // P V of a warpgroup's tile is done (kEarly)
  u64 loaded[4], checked[4];   // values of the n-th tile that rows see differently: there, looked through
  u64 queries, done;
};

// `kOwn`: sequences' own tokens, each of which sees its own number of keys; else the
// shared prefix, which all rows of the batch see.
template <typename T, int DP, bool kOwn>
__device__ __forceinline__ void wide_block(const AttendParams &p, const TensorMap &kmap, const TensorMap &vmap,
                                           const WideGrid &grid) {
  constexpr int G = kOwn ? 1 : 2;                            // softmax warpgroups
  using W = Wide<DP, G>;
  constexpr int kCopies = 4 * G, kMmas = 4 * G + 1, kLooks = 4 * G + 2;   // first warps of the other roles
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) Barriers bars;
  __shared__ OddValues<kOwn ? DP : 1> odd;
  __shared__ u32 tmem_slot;
  __shared__ volatile int dead;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char *smem = smem_raw + ((1024 - (tila::smem_u32(smem_raw) & 1023)) & 1023);

  // ---- which rows and keys ------------------------------------------------------
  i64 token0;
  int rows, head, begin, end, limit0, slot, pair;
  const i32 *pages;
  {
    int i = blockIdx.x;
    if constexpr (!kOwn) {
      pair = i % grid.pairs;
      i /= grid.pairs;
      head = i % p.kv_heads;
      slot = i / p.kv_heads;
      token0 = 0;
      const i64 all = p.offsets == nullptr ? p.batch : min(max(static_cast<i64>(p.offsets[p.batch]), static_cast<i64>(0)), p.tokens);
      rows = static_cast<int>(all * p.group);
      begin = slot * p.prefix_chunk;
      end = min(begin + p.prefix_chunk, p.prefix);
      limit0 = p.prefix;
      pages = p.prefix_pages;
    } else {
      pair = i % grid.pairs;
      i /= grid.pairs;
      head = i % p.kv_heads;
      i /= p.kv_heads;
      const int chunk = i % p.own_chunks, b = i / p.own_chunks;
      slot = p.prefix_chunks + chunk;
      int count;
      sequence_rows(p, b, token0, count);
      const int length = own_length(p, b);
      rows = count * p.group;
      limit0 = length - count + 1;
      const int keys = own_chunk(p, length);
      begin = chunk * keys;
      // the last token of the block's rows sees furthest
      const int last = min((pair + 1) * G * kTile, rows) - 1;
      end = min(begin + keys, limit0 + last / p.group);
      pages = p.table + b * p.table_stride;
    }
  }
  const int row0 = pair * G * kTile;
  if (row0 >= rows || (begin >= end && !p.direct)) return;
  // own tokens: tiles of the prefix before them, where the block takes it too
  const int before = kOwn && p.prefix_inside ? (p.prefix + kTile - 1) / kTile : 0;
  const auto first_key = [&](int tile) { return tile < before ? tile * kTile : begin + (tile - before) * kTile; };
  const auto keys_end = [&](int tile) { return tile < before ? p.prefix : end; };
  const bool shared_rows = G == 2 && rows - row0 <= kTile;   // one row tile: the warpgroups take tiles in turn
  const int tiles = before + (end > begin ? (end - begin + kTile - 1) / kTile : 0);
  const int ahead = shared_rows ? 2 : 1;             // S is issued so many tiles ahead of P V
  // tiles from here on hold keys that some rows see and others do not (2 at most: a
  // block's tokens are 128 or fewer)
  const int least = kOwn ? limit0 + row0 / p.group : end;
  const int mixed = least >= end ? tiles : before + max(0, least - begin) / kTile;

  if (threadIdx.x == 0) {
    for (int i = 0; i < W::kStages; ++i) {
      tila::mbar_init(&bars.full[i], 1);
      tila::mbar_init(&bars.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tila::mbar_init(&bars.scores[i], 1);
      tila::mbar_init(&bars.weights[i], kTile);
      tila::mbar_init(&bars.taken[i], kTile);
      tila::mbar_init(&bars.summed[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      tila::mbar_init(&bars.loaded[i], 1);
      tila::mbar_init(&bars.checked[i], 2);
    }
    tila::mbar_init(&bars.queries, G * kTile);
    tila::mbar_init(&bars.done, 1);
    dead = 0;
    odd.any = 0;
    tila::mbar_fence_init();
  }
  if (kOwn && warp >= kLooks && mixed < tiles)
    for (int i = threadIdx.x - 32 * kLooks; i < 3 * DP; i += 64) odd.first[i / DP][i % DP] = kNever;
  if (warp == kMmas) tila::tmem_alloc(&tmem_slot, W::kColumns);
  tila::tc_fence_before();
  __syncthreads();
  tila::tc_fence_after();
  const u32 tmem = tmem_slot;
  int *const dead_ptr = const_cast<int *>(&dead);

  // Ring order: keys of the first `ahead` tiles, then values of tile j and keys of
  // tile j + ahead.
  const int first_keys = min(ahead, tiles);

  if (warp >= kCopies) tila::reg_dealloc<W::kOtherRegisters>();
  if (warp == kCopies) {
    // ---- copies -----------------------------------------------------------------
    // A lane copies one box: 64 elements of one page's rows in the tile.  Its page
    // is looked up one tile ahead.
    constexpr int kHalves = DP / 64;
    const int box_rows = min(p.page_size, kTile);
    const int box = lane / kHalves, half = lane % kHalves;
    auto look_up = [&](int tile) {
      const int key = first_key(tile) + box * box_rows;
      if (box * box_rows >= kTile || key >= keys_end(tile)) return 0;
      int page, row;
      split_key(p, key, page, row);
      return tile < before ? p.prefix_pages[page] : pages[page];
    };
    auto copy = [&](int item, int tile, int page, const TensorMap *map) -> bool {
      const int stage = item % W::kStages;
      const int key0 = first_key(tile);
      const int boxes = (min(kTile, keys_end(tile) - key0) + box_rows - 1) / box_rows;   // pages that hold seen keys
      int index, row;
      split_key(p, key0 + box * box_rows, index, row);
      if (item >= W::kStages &&
          !warp_wait(&bars.empty[stage], (item / W::kStages - 1) & 1, p.err, __LINE__, dead_ptr))
        return false;
      if (lane == 0) tila::mbar_arrive_expect_tx(&bars.full[stage], boxes * kHalves * box_rows * 128);
      __syncwarp();
      if (box < boxes) {
        if (page < 0 || page >= p.num_pages) {
          tila::report_error(p.err, kErrIndex, index);
          page = p.num_pages;                               // outside the tensor: reads as zeros
        }
        tila::tma_load_4d(smem + W::kRing + stage * W::kTileBytes + half * kHalf + box * box_rows * 128, map,
                          &bars.full[stage], half * 64, row, head, page);
      }
      return true;
    };
    int item = 0;
    bool ok = true;
    for (int j = 0; ok && j < first_keys; ++j) ok = copy(item++, j, look_up(j), &kmap);
    int values = look_up(0), keys = look_up(ahead);
    for (int j = 0; ok && j < tiles; ++j) {
      const int next_values = look_up(j + 1), next_keys = look_up(j + 1 + ahead);
      ok = copy(item++, j, values, &vmap);
      if (ok && j + ahead < tiles) ok = copy(item++, j + ahead, keys, &kmap);
      values = next_values;
      keys = next_keys;
    }
    // (where a wait gave up nobody else waits for the copies in flight: they land before
    // the block leaves its shared memory)
    const int issued = ok ? item : item - 1;
    for (int i = max(0, issued - W::kStages); i < issued; ++i)
      warp_wait(&bars.full[i % W::kStages], (i / W::kStages) & 1, p.err, __LINE__, nullptr);
  } else if (warp == kMmas) {
    // ---- MMAs -------------------------------------------------------------------
    const u32 base4 = uniform(tila::smem_u32(smem)) >> 4, tm = uniform(tmem);
    const int n_tiles = static_cast<int>(uniform(tiles));
    const bool turns = uniform(shared_rows) != 0;                 // the warpgroups take tiles in turn
    const bool second = G == 2 && uniform(rows - row0 > kTile) != 0;        // the second row tile exists
    const int lead = turns ? 2 : 1, first_mixed = static_cast<int>(uniform(mixed));
    constexpr u32 kFormat = __is_same(T, __half) ? 0u : (1u << 7) | (1u << 10);
    constexpr u32 kScoresDesc = tila::idesc_f16_f32(128, 128, 0, 0) | kFormat;
    constexpr u32 kValuesDesc = tila::idesc_f16_f32(128, DP, 0, 1) | kFormat;
    auto wait_full = [&](int item) {
      return warp_wait(&bars.full[item % W::kStages], (item / W::kStages) & 1, p.err, __LINE__, dead_ptr);
    };
    auto stage_at = [&](int item) -> u32 { return W::kRing + (item % W::kStages) * W::kTileBytes; };
    auto scores = [&](int w, int item) {
      const u32 q = turns ? 0 : w * W::kTileBytes, k = stage_at(item);
      if (elected()) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const u32 off = (kk / 4) * kHalf + (kk % 4) * 32;
          tila::mma_f16_ss(tm + w * 128, tila::sdesc<16, 1024, 2>(base4, q + off),
                           tila::sdesc<16, 1024, 2>(base4, k + off), kScoresDesc, kk > 0);
        }
        tila::mma_commit(&bars.scores[w]);
      }
      __syncwarp();
    };
    bool ok = n_tiles == 0 || warp_wait(&bars.queries, 0, p.err, __LINE__, dead_ptr);
    int item = 0;
    for (int j = 0; ok && j < min(lead, n_tiles); ++j, ++item) {
      ok = wait_full(item);
      if (!ok) break;
      tila::tc_fence_after();
      if (turns) {
        scores(j, item);
      } else {
        scores(0, item);
        if (second) scores(1, item);
      }
      if (elected()) tila::mma_commit(&bars.empty[item % W::kStages]);
      __syncwarp();
    }
    for (int j = 0; ok && j < n_tiles; ++j) {
      const int values = item++;
      const bool more = j + lead < n_tiles;
      const int keys = more ? item++ : 0;
      ok = wait_full(values) && (!more || wait_full(keys));
      if (!ok) break;
      if (kOwn && j >= first_mixed && elected()) tila::mbar_arrive(&bars.loaded[j - first_mixed]);
      const int seen = static_cast<int>(uniform(min(kTile, keys_end(j) - first_key(j))));
      const int steps = static_cast<int>(uniform((seen + 15) >> 4));
      if (seen & 15) {
        // values behind the end, up to the group of 16 that P V covers
        unsigned char *v = smem + stage_at(values);
        for (int i = lane; i < (steps * 16 - seen) * (DP / 8); i += 32) {
          const int r = seen + i / (DP / 8), c = i % (DP / 8);
          *reinterpret_cast<uint4 *>(v + (c / 8) * kHalf + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
        }
        tila::fence_proxy_async_smem();
        __syncwarp();
      }
      const int w_first = turns ? (j & 1) : 0, w_last = turns ? (j & 1) : (second ? 1 : 0);
      const int turn = turns ? j >> 1 : j;
      for (int w = w_first; ok && w <= w_last; ++w) {
        if (W::kEarly && more) {
          ok = warp_wait(&bars.taken[w], turn & 1, p.err, __LINE__, dead_ptr);
          if (!ok) break;
          tila::tc_fence_after();
          scores(w, keys);
        }
        ok = warp_wait(&bars.weights[w], turn & 1, p.err, __LINE__, dead_ptr);
        if (!ok) break;
        tila::tc_fence_after();
        const u32 v = stage_at(values);
        if (elected()) {
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk)
            if (kk < steps)
              tila::mma_f16_ts(tm + W::kSumsAt + w * DP, tm + W::kWeightsAt + w * W::kWeightsStep + kk * 8,
                               tila::sdesc<kHalf, 1024, 2>(base4, v + kk * 2048), kValuesDesc, turn > 0 || kk > 0);
          if (W::kEarly) tila::mma_commit(&bars.summed[w]);
        }
        __syncwarp();
        if (!W::kEarly && more) scores(w, keys);
      }
      if (ok && elected()) {
        tila::mma_commit(&bars.empty[values % W::kStages]);
        if (more) tila::mma_commit(&bars.empty[keys % W::kStages]);
      }
      __syncwarp();
    }
    // (also where a wait gave up: products in flight end before tensor memory is given back)
    if (n_tiles > 0) {
      if (elected()) tila::mma_commit(&bars.done);
      __syncwarp();
      warp_wait(&bars.done, 0, p.err, __LINE__, nullptr);
    }
  } else if (warp >= kLooks) {
    if constexpr (kOwn) {
      // ---- values of mixed tiles -----------------------------------------------------
      bool ok = true;
      for (int j = mixed; ok && j < tiles; ++j) {
        const int item = first_keys + j + min(j, tiles - first_keys);
        unsigned char *v = smem + W::kRing + (item % W::kStages) * W::kTileBytes;
        // (not the ring's own barrier, whose phases this warp does not follow)
        ok = warp_wait(&bars.loaded[j - mixed], 0, p.err, __LINE__, dead_ptr);
        const int key0 = first_key(j), seen = min(kTile, end - key0);
        for (int i = threadIdx.x - 32 * kLooks; ok && i < seen * (DP / 8); i += 64) {
          const int r = i / (DP / 8), c = i % (DP / 8);
          unsigned char *at = v + (c / 8) * kHalf + r * 128 + (((c % 8) ^ (r & 7)) << 4);
          if (any_odd<T>(*reinterpret_cast<const uint4 *>(at))) {
            T *e = reinterpret_cast<T *>(at);
  #pragma unroll 1
            for (int k = 0; k < 8; ++k) {
              const float x = Elem<T>::get(e[k]);
              if (fabsf(x) < __builtin_huge_valf()) continue;
              atomicMin(&odd.first[x != x ? 0 : x > 0.f ? 1 : 2][c * 8 + k], key0 + r);
              odd.any = 1;
              e[k] = Elem<T>::put(0.f);
            }
          }
        }
        tila::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tila::mbar_arrive(&bars.checked[j - mixed]);
      }
    }
  } else {
    // ---- softmax: warpgroup w, one row a thread ------------------------------------
    tila::reg_alloc<W::kSoftmaxRegisters>();
    const int w = warp >> 2, r = threadIdx.x & (kTile - 1);
    const int row = row0 + (shared_rows ? 0 : w * kTile) + r;
    const bool valid = row < rows;
    const int token = valid ? row / p.group : 0;
    const int limit = !valid ? 0 : kOwn ? limit0 + token : limit0;
    const int out_head = head * p.group + (valid ? row - token * p.group : 0);
    if (!shared_rows || w == 0) {
      // the warp's 32 rows of queries, whole rows at a time, swizzled as TMA would
      // leave them
      constexpr int kPieces = DP / 8, kRows = 32 / kPieces;  // 16-byte pieces of a row; rows of one access
      // (rows that are not there read the first one, so that no load is conditional and
      // all are in flight together; they are cleared below)
      const i64 from = (token0 + token) * p.q_stride[0] + out_head * p.q_stride[1];
      const int c = lane % kPieces;
      const bool in = c * 8 < p.dim;
      const T *q = static_cast<const T *>(p.q) + (in ? c * 8 : 0);
      uint4 x[32 / kRows];
      if (p.q_vectors) {
#pragma unroll
        for (int i = 0; i < 32 / kRows; ++i)
          x[i] = *reinterpret_cast<const uint4 *>(q + __shfl_sync(0xffffffffu, from, i * kRows + lane / kPieces));
      } else {
#pragma unroll
        for (int i = 0; i < 32 / kRows; ++i) {
          const unsigned short *e = reinterpret_cast<const unsigned short *>(
              q + __shfl_sync(0xffffffffu, from, i * kRows + lane / kPieces));
          x[i] = make_uint4(e[0] | static_cast<u32>(e[1]) << 16, e[2] | static_cast<u32>(e[3]) << 16,
                            e[4] | static_cast<u32>(e[5]) << 16, e[6] | static_cast<u32>(e[7]) << 16);
        }
      }
      const u32 there = __ballot_sync(0xffffffffu, valid);
      const u32 flip = p.scale2 < 0.f ? 0x80008000u : 0u;    // scores are scaled by |scale|
#pragma unroll
      for (int i = 0; i < 32 / kRows; ++i) {
        const int q_row = (warp & 3) * 32 + i * kRows + lane / kPieces;
        x[i].x ^= flip, x[i].y ^= flip, x[i].z ^= flip, x[i].w ^= flip;
        if (!in || !(there >> (q_row & 31) & 1)) x[i] = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4 *>(smem + w * W::kTileBytes + q_row * 128 + (c / 8) * kHalf +
                                   (((c % 8) ^ (q_row & 7)) << 4)) = x[i];
      }
      tila::fence_proxy_async_smem();
    }
    tila::mbar_arrive(&bars.queries);

    const u32 lanes = tmem + ((warp & 3) << 21);            // this warp's 32 lanes
    const u32 s_col = lanes + w * 128, o_col = lanes + W::kSumsAt + w * DP;
    const u32 p_col = lanes + W::kWeightsAt + w * W::kWeightsStep;
    const float scale = fmaxf(fabsf(p.scale2), 1e-30f);     // above 0, so that -inf stays what it is
    float top = kNegInf, sum = 0.f;
    const bool works = shared_rows || row0 + w * kTile < rows;
    bool ok = true;
    int turn = 0;
    for (int j = shared_rows ? w : 0; works && j < tiles; j += ahead, ++turn) {
      ok = warp_wait(&bars.scores[w], turn & 1, p.err, __LINE__, dead_ptr);
      if (!ok) break;
      tila::tc_fence_after();
      float s[kTile];
      tila::tmem_load_row<kTile>(s_col, s);
      if (W::kEarly) {
        tila::tc_fence_before();
        tila::mbar_arrive(&bars.taken[w]);
      }
      const int seen = (j < before ? p.prefix : min(end, limit)) - first_key(j);   // columns that the row sees
      if (__any_sync(0xffffffffu, seen < kTile)) {
#pragma unroll
        for (int i = 0; i < kTile; ++i) s[i] = i < seen ? s[i] : kNegInf;
      }
      float best[2] = {s[0], s[1]};
#pragma unroll
      for (int i = 2; i < kTile; i += 4)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (i + e + 2 < kTile) best[e] = max3(best[e], s[i + e], s[i + e + 2]);
          else best[e] = fmaxf(best[e], s[i + e]);
        }
      const float high = fmaxf(best[0], best[1]) * scale;
      const bool grew = high > top + kGrowth || (top == kNegInf && high > kNegInf);
      const float factor = grew ? exp2f(top - high) : 1.f;
      if (grew) top = high;
      sum *= factor;
      if (W::kEarly && turn > 0) {
        // P V of the tile before reads P, and adds to O
        ok = warp_wait(&bars.summed[w], (turn - 1) & 1, p.err, __LINE__, dead_ptr);
        if (!ok) break;
        tila::tc_fence_after();
      }
      if (turn > 0 && __any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int c = 0; c < DP; c += 32) {
          float o[32];
          tila::tmem_ld32(o_col + c, o);
          tila::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= factor;
          tila::tmem_st32(o_col + c, o);
        }
      }
      const float base = top == kNegInf ? 0.f : top;
      const u64 scale_2 = tila::pk2(scale, scale), base_2 = tila::pk2(-base, -base);
      u64 sums[2] = {0, 0};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float packed[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int k = half * 64 + i * 2;
          const u64 x = tila::fma2(tila::pk2(s[k], s[k + 1]), scale_2, base_2);
          const float a = tila::exp2_ftz(tila::lo2(x)), b = tila::exp2_ftz(tila::hi2(x));
          sums[i & 1] = tila::add2(sums[i & 1], tila::pk2(a, b));
          packed[i] = __uint_as_float(pack_pair<T>(a, b));
        }
        tila::tmem_st32(p_col + half * 32, packed);
      }
      const u64 both = tila::add2(sums[0], sums[1]);
      sum += tila::lo2(both) + tila::hi2(both);
      tila::tmem_wait_st();
      tila::tc_fence_before();
      if (kOwn && j >= mixed) {
        // P V waits for the weights, and they for the look through the values
        ok = warp_wait(&bars.checked[j - mixed], 0, p.err, __LINE__, dead_ptr);
        if (!ok) break;
      }
      tila::mbar_arrive(&bars.weights[w]);
    }

    // ---- results: normalised, staged in queries and ring (free by now) --------
    if (tiles > 0) ok = warp_wait(&bars.done, 0, p.err, __LINE__, dead_ptr) && ok;
    tila::tc_fence_after();
    float *staged = reinterpret_cast<float *>(smem) + (w * kTile + r) * W::kRowFloats;
    float lse = sum == 0.f ? kNegInf : top + log2f(sum);
    float mine = sum == 0.f ? 0.f : 1.f / sum, other = 0.f;   // factors of the two warpgroups' sums
    const float *partner = staged + kTile * W::kRowFloats;
    if (shared_rows) {
      // both warpgroups saw a part of the keys: the second leaves its sums, the first joins
      if (w == 1) {
        write_row<DP>(o_col, turn > 0, mine, 0.f, nullptr, staged);
        staged[DP] = lse;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (w == 0) {
        const float second = partner[DP];
        const float high = fmaxf(lse, second), b = high == kNegInf ? 0.f : high;
        const float e0 = exp2f(lse - b), e1 = exp2f(second - b), all = e0 + e1;
        const float inverse = all == 0.f ? 0.f : 1.f / all;
        mine *= e0 * inverse;
        other = e1 * inverse;
        lse = all == 0.f ? kNegInf : b + log2f(all);
      }
    }
    if (!shared_rows || w == 0) {
      write_row<DP>(o_col, turn > 0, mine, other, shared_rows ? partner : nullptr, staged);
      if constexpr (kOwn)
        if (odd.any) put_odd<DP>(staged, odd, limit);
      const int at = valid && ok ? static_cast<int>((token0 + token) * p.heads + out_head) : -1;
      const i64 first = slot * p.tokens * p.heads;
      if (at >= 0) {
        if (!p.direct) p.partial_lse[first + at] = lse;
        else if (p.lse != nullptr) p.lse[at] = lse * 0.6931471805599453f;
      }
      __syncwarp();
      // the warp writes its 32 rows, a whole row at a time
      const float *from = staged - lane * W::kRowFloats + lane * 4;
      const bool in = lane * 4 < p.dim;
      if (!p.direct) {
        float *to = p.partial + first * p.dim + lane * 4;
#pragma unroll 8
        for (int i = 0; i < 32; ++i) {
          const int row_at = __shfl_sync(0xffffffffu, at, i);
          if (row_at >= 0 && in)
            *reinterpret_cast<float4 *>(to + static_cast<i64>(row_at) * p.dim) =
                *reinterpret_cast<const float4 *>(from + i * W::kRowFloats);
        }
      } else {
        const i64 out_at = (token0 + token) * p.out_stride[0] + out_head * p.out_stride[1];
#pragma unroll 4
        for (int i = 0; i < 32; ++i) {
          const i64 row_at = __shfl_sync(0xffffffffu, at >= 0 ? out_at : -1, i);
          if (row_at >= 0 && in) {
            const float4 x = *reinterpret_cast<const float4 *>(from + i * W::kRowFloats);
            T *to = static_cast<T *>(p.out) + row_at + lane * 4;
            if (p.out_vectors) {
              *reinterpret_cast<uint2 *>(to) = make_uint2(pack_pair<T>(x.x, x.y), pack_pair<T>(x.z, x.w));
            } else {
              to[0] = Elem<T>::put(x.x);
              to[1] = Elem<T>::put(x.y);
              to[2] = Elem<T>::put(x.z);
              to[3] = Elem<T>::put(x.w);
            }
          }
        }
      }
    }
    tila::tc_fence_before();
  }
  __syncthreads();
  if (warp == kMmas) tila::tmem_dealloc(tmem, W::kColumns);
}

// The first block ends after the previous kernel, beside which this one may run, so
// that what waits for this grid waits for both.
template <typename T, int DP, bool kOwn>
__global__ void __launch_bounds__(Wide<DP, kOwn ? 1 : 2>::kThreads, Wide<DP, kOwn ? 1 : 2>::kBlocks)
attend_wide_kernel(const __grid_constant__ AttendParams p, const __grid_constant__ TensorMap kmap,
                   const __grid_constant__ TensorMap vmap, const __grid_constant__ WideGrid grid) {
  tila::grid_dep_release();
  wide_block<T, DP, kOwn>(p, kmap, vmap, grid);
  if (blockIdx.x == 0 && threadIdx.x == 0) tila::grid_dep_wait();
}

int encode(TensorMap *map, const tila_attend_args &a, int rows, u64 address, const int64_t *stride, char *log,
           size_t cap) {
  const uint64_t dims[4] = {static_cast<u64>(a.dim), static_cast<u64>(a.page_size), static_cast<u64>(a.kv_heads),
                            static_cast<u64>(a.num_pages)};
  const uint64_t strides[3] = {static_cast<u64>(stride[1]) * 2, static_cast<u64>(stride[2]) * 2,
                               static_cast<u64>(stride[0]) * 2};
  const uint32_t box[4] = {64, static_cast<u32>(rows), 1, 1};
  // CUtensorMapDataType: 6 = f16, 9 = bf16; swizzle 3 = 128 bytes
  return tila_encode_tensor_map(map, a.dtype == TILA_F16 ? 6 : 9, 4, address, dims, strides, box, 3, log, cap);
}

// Whether the kernel was given the registers that its warpgroups share out.  What the
// compiler did is looked up once; a lookup that fails is made again at the next call.
template <typename T, int DP, bool kOwn> cudaError_t registers_fit(bool &fit) {
  static std::atomic<int> registers{0};
  int n = registers.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaFuncAttributes attr;
    const cudaError_t e = cudaFuncGetAttributes(&attr, attend_wide_kernel<T, DP, kOwn>);
    if (e != cudaSuccess) return e;
    registers.store(n = attr.numRegs, std::memory_order_relaxed);
  }
  fit = n == Wide<DP, kOwn ? 1 : 2>::kLaunchRegisters;
  return cudaSuccess;
}

template <typename T, int DP, bool kOwn>
cudaError_t launch_form(const AttendParams &p, const TensorMap &k, const TensorMap &v, const WideGrid &grid,
                        unsigned blocks, bool after_previous, cudaStream_t stream) {
  using W = Wide<DP, kOwn ? 1 : 2>;
  bool fit = false;
  cudaError_t e = registers_fit<T, DP, kOwn>(fit);
  if (e == cudaSuccess && !fit) e = cudaErrorLaunchOutOfResources;
  if (e == cudaSuccess) e = allow_shared_memory<attend_wide_kernel<T, DP, kOwn>>(W::kBytes);
  if (e != cudaSuccess) return e;
  return launch_kernel(attend_wide_kernel<T, DP, kOwn>, blocks, W::kThreads, W::kBytes, stream, after_previous, p, k, v,
                       grid);
}

}  // namespace

bool tma_possible(const tila_attend_args &a) {
  if (a.num_pages < 1) return false;
  // a dimension of one element may have any stride in torch; a tensor map's are positive and below 2^40 bytes
  const int64_t *strides[2] = {a.k_stride, a.v_stride};
  for (const int64_t *s : strides)
    for (int i = 0; i < 3; ++i)
      if (s[i] <= 0 || s[i] >= (1ll << 39)) return false;
  return true;
}

bool wide_possible(const tila_attend_args &a) {
  return tma_possible(a) && a.dim <= 128 && a.page_size % 8 == 0 &&
         (a.page_size < kTile ? kTile % a.page_size == 0 : a.page_size % kTile == 0);
}

namespace {
template <typename T> cudaError_t form_fits(const tila_attend_args &a, bool own, bool &fit) {
  if (a.dim <= 64) return own ? registers_fit<T, 64, true>(fit) : registers_fit<T, 64, false>(fit);
  return own ? registers_fit<T, 128, true>(fit) : registers_fit<T, 128, false>(fit);
}
}  // namespace

bool wide_fits(const tila_attend_args &a, bool own) {
  bool fit = true;
  const cudaError_t e = a.dtype == TILA_F16 ? form_fits<__half>(a, own, fit) : form_fits<__nv_bfloat16>(a, own, fit);
  if (e != cudaSuccess) cudaGetLastError();                 // the launch asks again, and reports it
  return fit;
}

int encode_caches(const tila_attend_args &a, int rows, tila::TensorMap *k, tila::TensorMap *v, char *log, size_t cap) {
  const int st = encode(k, a, rows, a.k_cache, a.k_stride, log, cap);
  return st == TILA_OK ? encode(v, a, rows, a.v_cache, a.v_stride, log, cap) : st;
}

int launch_wide(const tila_attend_args &a, const AttendParams &p, bool prefix, bool after_previous, cudaStream_t stream,
                char *log, size_t cap) {
  TensorMap k, v;
  const int st = encode_caches(a, a.page_size < kTile ? a.page_size : kTile, &k, &v, log, cap);
  if (st != TILA_OK) return st;
  WideGrid grid{};
  const i64 rows = static_cast<i64>(prefix ? (a.query_offsets == 0 ? a.batch : a.tokens) : p.max_queries) * p.group;
  const int each = (prefix ? 2 : 1) * kTile;                // rows of a block
  grid.pairs = static_cast<int>((rows + each - 1) / each);
  const i64 blocks = static_cast<i64>(grid.pairs) * p.kv_heads *
                     (prefix ? p.prefix_chunks : static_cast<i64>(p.own_chunks) * p.batch);
  if (blocks > 0x7fffffff) return fail(TILA_ERR_ARGUMENT, log, cap, "tila_attend_shared_prefix: too many blocks");
  const unsigned n = static_cast<unsigned>(blocks);
  const auto launch = [&](auto type, auto own) {
    using T = decltype(type);
    constexpr bool kOwn = decltype(own)::value;
    return a.dim <= 64 ? launch_form<T, 64, kOwn>(p, k, v, grid, n, after_previous, stream)
                       : launch_form<T, 128, kOwn>(p, k, v, grid, n, after_previous, stream);
  };
  const auto of_type = [&](auto own) {
    return a.dtype == TILA_F16 ? launch(__half{}, own) : launch(__nv_bfloat16{}, own);
  };
  const cudaError_t e = prefix ? of_type(std::false_type{}) : of_type(std::true_type{});
  return launch_status(e, "tila_attend_shared_prefix", log, cap);
}

}  // namespace tila_ops
