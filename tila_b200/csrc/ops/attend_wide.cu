// Attention over a paged cache with a shared prefix: the wide form, for more
// than 16 rows of queries that see the same keys.
//
// Up to 256 rows against one chunk of keys: GEMM-shaped, on the 5th-generation
// tensor cores.  One block a multiprocessor:
//
//   * two softmax warpgroups, one row a thread (a row is a TMEM lane), each with
//     its own scores S (128 columns) and its own sums O in tensor memory;
//   * a copy warp that streams tiles of 128 keys, then of their values, through
//     one ring in shared memory: a TMA box for each page and each 64 elements of
//     the heads, so that a tile takes its pages from anywhere in the pool;
//   * an MMA warp that issues S = Q K^T and O += P V.
//
// With more than 128 rows the warpgroups hold two row tiles and share every
// tile of keys (half the traffic from L2, which at 128 rows a tile would bound:
// 64 KB for every 1024 cycles of MMA); with fewer, both hold the same rows and
// take the tiles in turn, and their results are joined at the end.  Either way
// the tensor core works for one while the other is in its softmax.  Weights P
// (rounded to the values' type) go through tensor memory in the place of S.
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

namespace tila_ops {
namespace {

using tila::TensorMap;

constexpr int kThreads = 384;
// Registers a thread at launch (65536 / 384 in steps of 8), and what the
// warpgroups keep of them: the softmax holds a whole row of scores.  The shares add up to
// 256 * 216 + 128 * 64 = 63488, below the 384 * 168 = 64512 at launch; the host
// checks that the compiler gave the kernel exactly those, since a warpgroup
// would otherwise wait for registers that do not exist.
constexpr int kLaunchRegisters = 168;
constexpr int kTile = 128;                       // keys of a tile, rows of a row tile
constexpr float kGrowth = 8.f;                   // log2 of what weights may reach before O is scaled

template <int DP> struct Wide {
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kStages = DP == 128 ? 5 : 9;
  static constexpr int kRing = 2 * kTileBytes;   // behind the two query tiles
  static constexpr int kBytes = kRing + kStages * kTileBytes + 1024;   // 1024: alignment of swizzled tiles
  static constexpr int kRowFloats = DP + 4;      // of a staged result row: no two rows start in one bank
  static_assert(2 * kTile * kRowFloats * 4 <= kStages * kTileBytes, "results are staged in the ring");
  static_assert(kBytes <= 227 * 1024, "shared memory of a block");
};

// A bounded wait by a whole warp: all lanes go on, or none.
__device__ __forceinline__ bool warp_wait(u64 *bar, u32 parity, u32 *err, u32 where, int *dead) {
  return __all_sync(0xffffffffu, tila::mbar_wait(bar, parity, err, where, dead));
}

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

struct Barriers {
  u64 full[9], empty[9];
  u64 scores[2];      // S of a warpgroup's tile is there (and P V of its tile before)
  u64 weights[2];     // P is in tensor memory
  u64 queries, done;
};

template <typename T, int DP>
__device__ __forceinline__ void wide_block(const AttendParams &p, const TensorMap &kmap, const TensorMap &vmap,
                                           const WideGrid &grid) {
  using W = Wide<DP>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) Barriers bars;
  __shared__ u32 tmem_slot;
  __shared__ volatile int dead;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char *smem = smem_raw + ((1024 - (tila::smem_u32(smem_raw) & 1023)) & 1023);

  // ---- which rows and keys ------------------------------------------------------
  i64 token0;
  int rows, head, begin, end, limit0, slot, pair;
  const i32 *pages;
  bool causal = false;
  {
    int i = blockIdx.x;
    if (grid.prefix) {
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
      begin = chunk * p.own_chunk;
      // the last token of the block's rows sees furthest
      const int last = min((pair + 1) * 2 * kTile, rows) - 1;
      end = min(begin + p.own_chunk, limit0 + last / p.group);
      pages = p.table + b * p.table_stride;
      causal = true;
    }
  }
  const int row0 = pair * 2 * kTile;
  if (row0 >= rows || (begin >= end && !p.direct)) return;
  const bool shared_rows = rows - row0 <= kTile;     // one row tile: the warpgroups take tiles in turn
  const int tiles = end > begin ? (end - begin + kTile - 1) / kTile : 0;
  const int ahead = shared_rows ? 2 : 1;             // S is issued so many tiles ahead of P V

  if (threadIdx.x == 0) {
    for (int i = 0; i < W::kStages; ++i) {
      tila::mbar_init(&bars.full[i], 1);
      tila::mbar_init(&bars.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tila::mbar_init(&bars.scores[i], 1);
      tila::mbar_init(&bars.weights[i], kTile);
    }
    tila::mbar_init(&bars.queries, 2 * kTile);
    tila::mbar_init(&bars.done, 1);
    dead = 0;
    tila::mbar_fence_init();
  }
  if (warp == 9) tila::tmem_alloc(&tmem_slot, 512);
  tila::tc_fence_before();
  __syncthreads();
  tila::tc_fence_after();
  const u32 tmem = tmem_slot;
  int *const dead_ptr = const_cast<int *>(&dead);

  // Ring order: keys of the first `ahead` tiles, then values of tile j and keys of
  // tile j + ahead.
  const int first_keys = min(ahead, tiles);

  if (warp >= 8) tila::reg_dealloc<64>();
  if (warp == 8) {
    // ---- copies -----------------------------------------------------------------
    constexpr int kHalves = DP / 64;
    const int box_rows = min(p.page_size, kTile);
    auto copy = [&](int item, int tile, const TensorMap *map) -> bool {
      const int stage = item % W::kStages;
      if (item >= W::kStages &&
          !warp_wait(&bars.empty[stage], (item / W::kStages - 1) & 1, p.err, __LINE__, dead_ptr))
        return false;
      const int key0 = begin + tile * kTile;
      const int boxes = (min(kTile, end - key0) + box_rows - 1) / box_rows;   // pages that hold seen keys
      if (lane == 0) tila::mbar_arrive_expect_tx(&bars.full[stage], boxes * kHalves * box_rows * 128);
      __syncwarp();
      unsigned char *dst = smem + W::kRing + stage * W::kTileBytes;
      if (lane < boxes * kHalves) {
        const int i = lane / kHalves, half = lane % kHalves;
        int page, row;
        split_key(p, key0 + i * box_rows, page, row);
        page = checked_page(p, pages, page);
        if (page < 0) page = p.num_pages;                   // outside the tensor: reads as zeros
        tila::tma_load_4d(dst + half * (kTile * 128) + i * box_rows * 128, map, &bars.full[stage], half * 64, row,
                          head, page);
      }
      return true;
    };
    int item = 0;
    bool ok = true;
    for (int j = 0; ok && j < first_keys; ++j) ok = copy(item++, j, &kmap);
    for (int j = 0; ok && j < tiles; ++j) {
      ok = copy(item++, j, &vmap);
      if (ok && j + ahead < tiles) ok = copy(item++, j + ahead, &kmap);
    }
  } else if (warp == 9) {
    // ---- MMAs -------------------------------------------------------------------
    const u32 base4 = tila::smem_u32(smem) >> 4;
    constexpr u32 kFormat = __is_same(T, __half) ? 0u : (1u << 7) | (1u << 10);
    constexpr u32 kScoresDesc = tila::idesc_f16_f32(128, 128, 0, 0) | kFormat;
    constexpr u32 kValuesDesc = tila::idesc_f16_f32(128, DP, 0, 1) | kFormat;
    auto stage_of = [&](int item) { return W::kRing + (item % W::kStages) * W::kTileBytes; };
    auto wait_full = [&](int item) {
      return warp_wait(&bars.full[item % W::kStages], (item / W::kStages) & 1, p.err, __LINE__, dead_ptr);
    };
    auto scores = [&](int w, int item) {
      if (lane == 0) {
        const u32 q = shared_rows ? 0 : w * W::kTileBytes, k = stage_of(item);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const u32 off = (kk / 4) * (kTile * 128) + (kk % 4) * 32;
          tila::mma_f16_ss(tmem + w * 128, tila::sdesc<16, 1024, 2>(base4, q + off),
                           tila::sdesc<16, 1024, 2>(base4, k + off), kScoresDesc, kk > 0);
        }
        tila::mma_commit(&bars.scores[w]);
      }
      __syncwarp();
    };
    bool ok = tiles == 0 || warp_wait(&bars.queries, 0, p.err, __LINE__, dead_ptr);
    const bool second = !shared_rows && rows - row0 > kTile;      // the second row tile exists
    int item = 0;
    for (int j = 0; ok && j < first_keys; ++j, ++item) {
      ok = wait_full(item);
      if (!ok) break;
      tila::tc_fence_after();
      if (shared_rows) {
        scores(j, item);
      } else {
        scores(0, item);
        if (second) scores(1, item);
      }
      if (lane == 0) tila::mma_commit(&bars.empty[item % W::kStages]);
    }
    for (int j = 0; ok && j < tiles; ++j) {
      const int values = item++;
      const bool more = j + ahead < tiles;
      const int keys = more ? item++ : 0;
      ok = wait_full(values) && (!more || wait_full(keys));
      if (!ok) break;
      const int seen = min(kTile, end - (begin + j * kTile));
      const int steps = (seen + 15) >> 4;
      if (seen & 15) {
        // values behind the end, up to the group of 16 that P V covers
        unsigned char *v = smem + stage_of(values);
        for (int i = lane; i < (steps * 16 - seen) * (DP / 8); i += 32) {
          const int r = seen + i / (DP / 8), c = i % (DP / 8);
          *reinterpret_cast<uint4 *>(v + (c / 8) * (kTile * 128) + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
        }
        tila::fence_proxy_async_smem();
        __syncwarp();
      }
      for (int w = shared_rows ? (j & 1) : 0; ok && w <= (shared_rows ? (j & 1) : (second ? 1 : 0)); ++w) {
        const int turn = shared_rows ? j >> 1 : j;
        ok = warp_wait(&bars.weights[w], turn & 1, p.err, __LINE__, dead_ptr);
        if (!ok) break;
        tila::tc_fence_after();
        if (lane == 0) {
          const u32 v = stage_of(values);
          for (int kk = 0; kk < steps; ++kk)
            tila::mma_f16_ts(tmem + 256 + w * DP, tmem + w * 128 + kk * 8,
                             tila::sdesc<kTile * 128, 1024, 2>(base4, v + kk * 2048), kValuesDesc, turn > 0 || kk > 0);
        }
        __syncwarp();
        if (more) scores(w, keys);
      }
      if (ok && lane == 0) {
        tila::mma_commit(&bars.empty[values % W::kStages]);
        if (more) tila::mma_commit(&bars.empty[keys % W::kStages]);
      }
      __syncwarp();
    }
    if (ok && tiles > 0 && lane == 0) tila::mma_commit(&bars.done);
    __syncwarp();
  } else if (warp < 8) {
    // ---- softmax: warpgroup w, one row a thread ------------------------------------
    tila::reg_alloc<216>();
    const int w = warp >> 2, r = threadIdx.x & (kTile - 1);
    const int row = row0 + (shared_rows ? 0 : w * kTile) + r;
    const bool valid = row < rows;
    const int token = valid ? row / p.group : 0;
    const int limit = !valid ? 0 : causal ? limit0 + token : limit0;
    const int out_head = head * p.group + (valid ? row - token * p.group : 0);
    if (!shared_rows || w == 0) {
      // the warp's 32 rows of queries, whole rows at a time, swizzled as TMA would
      // leave them
      constexpr int kPieces = DP / 8, kRows = 32 / kPieces;  // 16-byte pieces of a row; rows of one access
      const i64 from = valid ? (token0 + token) * p.q_stride[0] + out_head * p.q_stride[1] : -1;
      const int c = lane % kPieces;
      uint4 x[32 / kRows];
#pragma unroll
      for (int i = 0; i < 32 / kRows; ++i) {
        const i64 at = __shfl_sync(0xffffffffu, from, i * kRows + lane / kPieces);
        x[i] = make_uint4(0, 0, 0, 0);
        if (at >= 0 && c * 8 < p.dim) {
          const T *q = static_cast<const T *>(p.q) + at + c * 8;
          if (p.q_vectors) {
            x[i] = *reinterpret_cast<const uint4 *>(q);
          } else {
            const unsigned short *e = reinterpret_cast<const unsigned short *>(q);
            x[i] = make_uint4(e[0] | static_cast<u32>(e[1]) << 16, e[2] | static_cast<u32>(e[3]) << 16,
                              e[4] | static_cast<u32>(e[5]) << 16, e[6] | static_cast<u32>(e[7]) << 16);
          }
        }
      }
      const u32 flip = p.scale2 < 0.f ? 0x80008000u : 0u;    // scores are scaled by |scale|
#pragma unroll
      for (int i = 0; i < 32 / kRows; ++i) {
        const int q_row = (warp & 3) * 32 + i * kRows + lane / kPieces;
        x[i].x ^= flip, x[i].y ^= flip, x[i].z ^= flip, x[i].w ^= flip;
        *reinterpret_cast<uint4 *>(smem + w * W::kTileBytes + q_row * 128 + (c / 8) * (kTile * 128) +
                                   (((c % 8) ^ (q_row & 7)) << 4)) = x[i];
      }
      tila::fence_proxy_async_smem();
    }
    tila::mbar_arrive(&bars.queries);

    const u32 lanes = tmem + ((warp & 3) << 21);            // this warp's 32 lanes
    const u32 s_col = lanes + w * 128, o_col = lanes + 256 + w * DP;
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
      const int key0 = begin + j * kTile;
      const int seen = min(end, limit) - key0;              // columns that the row sees
      if (__any_sync(0xffffffffu, seen < kTile)) {
#pragma unroll
        for (int i = 0; i < kTile; ++i) s[i] = i < seen ? s[i] : kNegInf;
      }
      float best[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int i = 4; i < kTile; i += 4)
#pragma unroll
        for (int e = 0; e < 4; ++e) best[e] = fmaxf(best[e], s[i + e]);
      const float high = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3])) * scale;
      const bool grew = high > top + kGrowth || (top == kNegInf && high > kNegInf);
      const float factor = grew ? exp2f(top - high) : 1.f;
      if (grew) top = high;
      sum *= factor;
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
          const float a = tila::exp2_fast(tila::lo2(x)), b = tila::exp2_fast(tila::hi2(x));
          sums[i & 1] = tila::add2(sums[i & 1], tila::pk2(a, b));
          packed[i] = __uint_as_float(wide_pack<T>(a, b));
        }
        tila::tmem_st32(s_col + half * 32, packed);
      }
      const u64 both = tila::add2(sums[0], sums[1]);
      sum += tila::lo2(both) + tila::hi2(both);
      tila::tmem_wait_st();
      tila::tc_fence_before();
      tila::mbar_arrive(&bars.weights[w]);
    }

    // ---- results: normalised, staged in the ring (free by now), a bulk copy a row -----
    if (tiles > 0) ok = warp_wait(&bars.done, 0, p.err, __LINE__, dead_ptr) && ok;
    tila::tc_fence_after();
    float *staged = reinterpret_cast<float *>(smem + W::kRing) + (w * kTile + r) * W::kRowFloats;
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
      if (valid && ok) {
        const i64 at = (token0 + token) * p.heads + out_head;
        const i64 place = slot * p.tokens * p.heads + at;
        if (p.direct) {
          T *out = static_cast<T *>(p.out) + (token0 + token) * p.out_stride[0] + out_head * p.out_stride[1];
          for (int d = 0; d < p.dim; ++d) out[d] = Elem<T>::put(staged[d]);
          if (p.lse != nullptr) p.lse[at] = lse * 0.6931471805599453f;
        } else {
          p.partial_lse[place] = lse;
          tila::fence_proxy_async_smem();
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(p.partial + place * p.dim),
                       "r"(tila::smem_u32(staged)), "r"(p.dim * 4) : "memory");
          tila::bulk_commit();
          tila::bulk_wait_read();
        }
      }
    }
    tila::tc_fence_before();
  }
  __syncthreads();
  if (warp == 9) tila::tmem_dealloc(tmem, 512);
}

// The first block ends after the previous kernel, beside which this one may run, so
// that what waits for this grid waits for both.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
attend_wide_kernel(const __grid_constant__ AttendParams p, const __grid_constant__ TensorMap kmap,
                   const __grid_constant__ TensorMap vmap, const __grid_constant__ WideGrid grid) {
  tila::grid_dep_release();
  wide_block<T, DP>(p, kmap, vmap, grid);
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

template <typename T, int DP>
cudaError_t launch_form(const AttendParams &p, const TensorMap &k, const TensorMap &v, const WideGrid &grid,
                        unsigned blocks, bool after_previous, cudaStream_t stream) {
  static const cudaError_t registers = [] {
    cudaFuncAttributes attr;
    const cudaError_t e = cudaFuncGetAttributes(&attr, attend_wide_kernel<T, DP>);
    return e != cudaSuccess ? e : attr.numRegs == kLaunchRegisters ? cudaSuccess : cudaErrorLaunchOutOfResources;
  }();
  if (registers != cudaSuccess) return registers;
  cudaError_t e = cudaFuncSetAttribute(attend_wide_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Wide<DP>::kBytes);
  if (e != cudaSuccess) return e;
  return launch_kernel(attend_wide_kernel<T, DP>, blocks, kThreads, Wide<DP>::kBytes, stream, after_previous, p, k, v,
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
  grid.prefix = prefix;
  grid.pairs = static_cast<int>((rows + 2 * kTile - 1) / (2 * kTile));
  const i64 blocks = static_cast<i64>(grid.pairs) * p.kv_heads *
                     (prefix ? p.prefix_chunks : static_cast<i64>(p.own_chunks) * p.batch);
  if (blocks > 0x7fffffff) return fail(TILA_ERR_ARGUMENT, log, cap, "tila_attend_shared_prefix: too many blocks");
  const unsigned n = static_cast<unsigned>(blocks);
  const auto launch = [&](auto form) { return form(p, k, v, grid, n, after_previous, stream); };
  const cudaError_t e = a.dtype == TILA_F16
                            ? (a.dim <= 64 ? launch(launch_form<__half, 64>) : launch(launch_form<__half, 128>))
                            : (a.dim <= 64 ? launch(launch_form<__nv_bfloat16, 64>) : launch(launch_form<__nv_bfloat16, 128>));
  return launch_status(e, "tila_attend_shared_prefix", log, cap);
}

}  // namespace tila_ops
