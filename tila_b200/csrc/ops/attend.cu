// Attention over a paged cache with a shared prefix: the narrow form for up to
// 16 rows of queries a block, the join of partial results, and the host side
// (the wide form, for more rows, is attend_wide.cu).
//
// Narrow form.  Few rows against many keys: bound by reading the keys and
// values once.  A block takes 8 or 16 rows (a sequence's new tokens times the heads
// that share its key head) and one chunk of keys.  Each warp runs on its own: it
// brings 16 keys and values at a time into its own ring of shared memory and needs
// no barrier with the others, so that loads never wait for arithmetic.  Where pages
// are multiples of 16 rows a step's keys lie in one page and one lane fetches them
// with TMA (a box for 64 elements of 16 rows); for other pages each lane looks up
// rows and copies 16-byte pieces with cp.async, whose 32 instructions a step cost a
// warp 1500 of its 2500 cycles where TMA costs it about 100.
//
// Scores and sums go through m16n8k16 matrix instructions with 32-bit sums, keys
// and values as the 16-row operand and the queries as the 8 columns: S^T = K Q^T and
// O^T += V^T P^T.  Groups of up to 8 heads waste none of that, where 16 rows of queries
// would take twice the instructions and registers (these rows do not fill a tcgen05
// tile, and the instruction rate is not what bounds).  Weights p are rounded to the
// values' type for the product with the values and summed as they are in 32 bits:
// the sum is also a result (lse), and a rounding of p moves it by 2^-9 of a weight.

#include "attend.cuh"
#include "attend_wide.cuh"

#include <algorithm>
#include <cmath>

namespace {

using namespace tila_ops;

constexpr int kWarps = 4;
constexpr int kSlice = 16;                 // keys of one warp's step
constexpr int kStep = kWarps * kSlice;     // keys of one block's step
constexpr int kStages = 2;                 // 64 KB a block at 128 elements: three blocks a multiprocessor

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const u32 (&a)[4], u32 b0, u32 b1) {
  if constexpr (sizeof(T) == 2 && __is_same(T, __half))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix4(u32 (&r)[4], u32 addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// The transpose of an 8x8 block of 16-bit elements across the warp.
__device__ __forceinline__ u32 transposed(u32 x) {
  u32 r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void ldmatrix4t(u32 (&r)[4], u32 addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// 16 bytes into shared memory, zeros where `bytes` is 0 (nothing is read then).
__device__ __forceinline__ void copy16(u32 dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Where a block's rows and keys are.
struct Item {
  i64 token0;          // first row of q
  int rows;            // rows of the segment: tokens * group
  int row0;            // first row of this block
  int head;            // key head
  int begin, end;      // keys of the chunk
  int limit0;          // keys that the segment's first token sees (token i sees limit0 + i)
  int slot;            // of the partial result
  const i32 *pages;
};

template <int DP> struct Narrow {
  static constexpr int kHalf = kSlice * 128;                 // 64 elements of 16 rows, swizzled
  static constexpr int kValues = DP / 64 * kHalf;            // of a stage: keys, then values
  static constexpr int kStage = 2 * kValues;
  static constexpr int kWarpBytes = kStages * kStage;
  static constexpr int kBytes = kWarps * kWarpBytes + 1024;  // 1024: alignment of swizzled tiles
  static constexpr int kJoin = DP + 8;                        // floats of a row in the join of the warps
  static_assert(kWarpBytes >= 16 * kJoin * 4, "the join of the warps reuses the ring");
};

// Where 16 bytes (piece `ch` of row r) lie in a swizzled tile.
__device__ __forceinline__ u32 piece(int r, int ch) {
  return (ch >> 3) * (kSlice * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
}

template <typename T, int DP, int NT, bool kTma>
__device__ __forceinline__ void narrow_block(const AttendParams &p, const tila::TensorMap &kmap,
                                             const tila::TensorMap &vmap, int prefix_items, int prefix_tiles,
                                             int own_tiles) {
  using N = Narrow<DP>;
  constexpr int kRows = 8 * NT;                              // of queries
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = smem_raw + ((1024 - (tila::smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ __align__(8) u64 full[kWarps][kStages];
  __shared__ float row_max[kWarps][kRows], row_sum[kWarps][kRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  // which rows and keys: neighbouring blocks take the heads of the same pages
  Item it;
  {
    int i = blockIdx.x;
    if (i < prefix_items) {
      const int tile = i % prefix_tiles;
      i /= prefix_tiles;
      it.head = i % p.kv_heads;
      it.slot = i / p.kv_heads;
      it.token0 = 0;
      const i64 all = p.offsets == nullptr ? p.batch : min(max(static_cast<i64>(p.offsets[p.batch]), static_cast<i64>(0)), p.tokens);
      it.rows = static_cast<int>(all * p.group);
      it.row0 = tile * kRows;
      it.begin = it.slot * p.prefix_chunk;
      it.end = min(it.begin + p.prefix_chunk, p.prefix);
      it.limit0 = p.prefix;
      it.pages = p.prefix_pages;
      if (it.row0 >= it.rows) return;
    } else {
      i -= prefix_items;
      const int tile = i % own_tiles;
      i /= own_tiles;
      it.head = i % p.kv_heads;
      i /= p.kv_heads;
      const int chunk = i % p.own_chunks, b = i / p.own_chunks;
      it.slot = p.prefix_chunks + chunk;
      int count;
      sequence_rows(p, b, it.token0, count);
      const int length = own_length(p, b);
      it.rows = count * p.group;
      it.row0 = tile * kRows;
      if (it.row0 >= it.rows) return;
      it.limit0 = length - count + 1;
      const int last = (min(it.row0 + kRows, it.rows) - 1) / p.group;
      const int keys = own_chunk(p, length);
      it.begin = chunk * keys;
      it.end = min(it.begin + keys, it.limit0 + last);
      it.pages = p.table + b * p.table_stride;
      // nothing of this chunk is seen: only the sole chunk writes (zeros) then
      if (it.begin >= it.end && !p.direct) return;
    }
  }
  const bool causal = it.slot >= p.prefix_chunks;

  // the warp's ring of keys and values
  unsigned char *ring = smem + warp * N::kWarpBytes;
  const u32 ring_at = tila::smem_u32(ring);
  const int begin = it.begin + warp * kSlice;
  const int steps = it.end > begin ? (it.end - begin + kStep - 1) / kStep : 0;
  if constexpr (kTma) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < kStages; ++i) tila::mbar_init(&full[warp][i], 1);
      tila::mbar_fence_init();
    }
    __syncwarp();
  }
  // The page of a step's key is read one step ahead, and looked at when it is
  // used: that of the step's first key, or each lane's of key lane & 15.
  const int page_key = kTma ? 0 : lane & 15;
  auto look_up = [&](int step) {
    const int key = begin + step * kStep + page_key;
    if (key >= it.end) return 0;
    int page, row;
    split_key(p, key, page, row);
    return it.pages[page];
  };
  int page_ahead = kTma && lane != 0 ? 0 : look_up(0);
  auto issue = [&](int step) {
    if (step < steps && (!kTma || lane == 0)) {
      const int key0 = begin + step * kStep;
      int index, row;
      split_key(p, key0 + page_key, index, row);
      const int page = page_ahead;
      page_ahead = look_up(step + 1);
      bool ok = key0 + page_key < it.end;
      if (ok && (page < 0 || page >= p.num_pages)) {
        tila::report_error(p.err, kErrIndex, index);
        ok = false;
      }
      if constexpr (kTma) {
        u64 *bar = &full[warp][step % kStages];
        unsigned char *stage = ring + (step % kStages) * N::kStage;
        const int from = ok ? page : p.num_pages;            // outside the tensor: reads as zeros
        tila::mbar_arrive_expect_tx(bar, N::kStage);
#pragma unroll
        for (int i = 0; i < DP / 64; ++i) {
          tila::tma_load_4d(stage + i * N::kHalf, &kmap, bar, i * 64, row, it.head, from);
          tila::tma_load_4d(stage + N::kValues + i * N::kHalf, &vmap, bar, i * 64, row, it.head, from);
        }
      } else {
        constexpr int kChunks = DP / 8;                      // 16-byte pieces of a row
        const i64 koff = ok ? page * p.k_stride[0] + row * p.k_stride[1] + it.head * p.k_stride[2] : -1;
        const i64 voff = ok ? page * p.v_stride[0] + row * p.v_stride[1] + it.head * p.v_stride[2] : 0;
        const u32 stage = ring_at + (step % kStages) * N::kStage;
#pragma unroll
        for (int i = 0; i < kSlice * kChunks / 32; ++i) {
          const int r = (i * 32 + lane) / kChunks, ch = (i * 32 + lane) % kChunks;
          const i64 ko = __shfl_sync(0xffffffffu, koff, r), vo = __shfl_sync(0xffffffffu, voff, r);
          const bool in = ko >= 0 && ch * 8 < p.dim;
          const T *k = static_cast<const T *>(p.k), *v = static_cast<const T *>(p.v);
          copy16(stage + piece(r, ch), in ? k + ko + ch * 8 : k, in ? 16 : 0);
          copy16(stage + N::kValues + piece(r, ch), in ? v + vo + ch * 8 : v, in ? 16 : 0);
        }
      }
    }
    if constexpr (!kTma) copy_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) issue(s);

  // queries: columns g of 8, as B fragments
  const int g = lane >> 2, c = lane & 3;
  u32 qf[NT][DP / 16][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = it.row0 + t * 8 + g;
    const int token = row / p.group;
    const T *q = static_cast<const T *>(p.q) + (it.token0 + token) * p.q_stride[0] +
                 (it.head * p.group + row - token * p.group) * p.q_stride[1];
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int d = k * 16 + half * 8 + c * 2;
        u32 w = 0;
        if (row < it.rows && d < p.dim) {
          if (p.q_words) w = *reinterpret_cast<const u32 *>(q + d);
          else w = reinterpret_cast<const unsigned short *>(q)[d] |
                   static_cast<u32>(reinterpret_cast<const unsigned short *>(q)[d + 1]) << 16;
        }
        qf[t][k][half] = w;
      }
  }
  // keys that the rows of this lane's sums (2 c and 2 c + 1 of each 8) see
  int limit[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = it.row0 + t * 8 + c * 2 + e;
      limit[t][e] = row < it.rows ? min(it.end, causal ? it.limit0 + row / p.group : it.limit0) : 0;
    }

  // keys up to here are seen by all rows or by none
  const int sees_least = causal && it.limit0 + it.row0 / p.group < it.end ? it.limit0 + it.row0 / p.group : 0x7fffffff;
  float o[NT][DP / 16][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t][0] = m[t][1] = kNegInf;
    l[t][0] = l[t][1] = 0.f;
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.f;
  }

  for (int step = 0; step < steps; ++step) {
    const u32 stage = ring_at + (step % kStages) * N::kStage;
    const int key0 = begin + step * kStep;
    if constexpr (kTma) {
      if (!__all_sync(0xffffffffu, tila::mbar_wait(&full[warp][step % kStages], (step / kStages) & 1, p.err, __LINE__,
                                                   nullptr))) {
        // the copies behind it land before their places are used for the join
        for (int s = step; s < min(step + kStages, steps); ++s)
          tila::mbar_wait(&full[warp][s % kStages], (s / kStages) & 1, p.err, __LINE__, nullptr);
        break;
      }
      if (key0 + kSlice > it.end) {
        // values behind the end: whatever the page holds there, for a weight of 0
        for (int i = lane; i < (key0 + kSlice - it.end) * (DP / 8); i += 32)
          *reinterpret_cast<uint4 *>(ring + (step % kStages) * N::kStage + N::kValues +
                                     piece(it.end - key0 + i / (DP / 8), i % (DP / 8))) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
    } else {
      copy_wait<kStages - 1>();
      __syncwarp();
    }
    // S^T: keys g and g + 8 in rows, two chains of sums
    float s[NT][2][4] = {};
    {
      const int r = lane & 15, ch = lane >> 4;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        u32 a[4];
        ldmatrix4(a, stage + piece(r, k * 2 + ch));
#pragma unroll
        for (int t = 0; t < NT; ++t) mma16816<T>(s[t][k & 1], a, qf[t][k][0], qf[t][k][1]);
      }
    }
    u32 pf[NT][2];
    float scale[NT][2], weights[NT][2][2];                   // [key g, key g + 8][row]
    bool moved = false;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float (&w)[2][2] = weights[t];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          w[h][e] = key0 + g + h * 8 < limit[t][e] ? (s[t][0][h * 2 + e] + s[t][1][h * 2 + e]) * p.scale2 : kNegInf;
        float best = fmaxf(w[0][e], w[1][e]);
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 4));
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 8));
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 16));
        const float top = fmaxf(m[t][e], best);
        const float base = top == kNegInf ? 0.f : top;       // nothing seen yet: all weights 0
        scale[t][e] = tila::exp2_ftz(m[t][e] - base);
        moved = moved || top != m[t][e];
        m[t][e] = top;
        w[0][e] = tila::exp2_ftz(w[0][e] - base);
        w[1][e] = tila::exp2_ftz(w[1][e] - base);
        l[t][e] = l[t][e] * scale[t][e] + (w[0][e] + w[1][e]);
      }
      // P^T as the B operand: keys in rows there, so each 8x8 block turned around
      pf[t][0] = transposed(pack_pair<T>(w[0][0], w[0][1]));
      pf[t][1] = transposed(pack_pair<T>(w[1][0], w[1][1]));
    }
    // the sums follow the maximum only when it moved
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
          o[t][n][0] *= scale[t][0];
          o[t][n][1] *= scale[t][1];
          o[t][n][2] *= scale[t][0];
          o[t][n][3] *= scale[t][1];
        }
    }
    // Where some rows see keys that others do not, a value that is no number must
    // not reach the others through its weight of 0: such slices (new tokens' own,
    // and of them only those with such values) are summed one key at a time.
    bool odd = false;
    if (key0 + kSlice > sees_least)
      for (int i = lane; i < kSlice * (DP / 8); i += 32)
        odd = odd || any_odd<T>(*reinterpret_cast<const uint4 *>(ring + (step % kStages) * N::kStage + N::kValues + i * 16));
    if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
      for (int j = 0; j < kSlice; ++j) {
        const T *v = reinterpret_cast<const T *>(ring + (step % kStages) * N::kStage + N::kValues);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float w = Elem<T>::get(Elem<T>::put(
                __shfl_sync(0xffffffffu, j < 8 ? weights[t][0][e] : weights[t][1][e], (j & 7) * 4 + c)));
            if (key0 + j < limit[t][e])
#pragma unroll
              for (int n = 0; n < DP / 16; ++n) {
                o[t][n][e] += w * Elem<T>::get(v[piece(j, n * 2) / 2 + g]);
                o[t][n][2 + e] += w * Elem<T>::get(v[piece(j, n * 2 + 1) / 2 + g]);
              }
          }
      }
    } else {
      const int r = (lane & 7) + ((lane >> 4) << 3), ch = (lane >> 3) & 1;
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        u32 a[4];
        ldmatrix4t(a, stage + N::kValues + piece(r, n * 2 + ch));
#pragma unroll
        for (int t = 0; t < NT; ++t) mma16816<T>(o[t][n], a, pf[t][0], pf[t][1]);
      }
    }
    __syncwarp();                                            // all lanes have read the stage
    issue(step + kStages);
  }

  // join the warps: maxima, sums, then the scaled results through shared memory
  if constexpr (!kTma) copy_wait<0>();
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 4);
      l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 8);
      l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 16);
      if (g == 0) {
        row_max[warp][t * 8 + c * 2 + e] = m[t][e];
        row_sum[warp][t * 8 + c * 2 + e] = l[t][e];
      }
    }
  __syncthreads();
  float *joined = reinterpret_cast<float *>(smem) + warp * kRows * N::kJoin;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = t * 8 + c * 2 + e;
      float top = kNegInf;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, row_max[w][r]);
      const float f = m[t][e] == kNegInf ? 1.f : exp2f(m[t][e] - top);   // nothing seen: 0 times 1
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        joined[r * N::kJoin + n * 16 + g] = o[t][n][e] * f;
        joined[r * N::kJoin + n * 16 + 8 + g] = o[t][n][2 + e] * f;
      }
    }
  __syncthreads();
  const float *all = reinterpret_cast<const float *>(smem);
  for (int r = warp; r < kRows; r += kWarps) {
    const int row = it.row0 + r;
    if (row >= it.rows) continue;
    float top = kNegInf, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, row_max[w][r]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += row_max[w][r] == kNegInf ? row_sum[w][r] : row_sum[w][r] * exp2f(row_max[w][r] - top);
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
    const float lse2 = sum == 0.f ? kNegInf : top + log2f(sum);
    const i64 token = it.token0 + row / p.group;
    const int head = it.head * p.group + row % p.group;
    const i64 at = token * p.heads + head;
    if (p.direct) {
      T *out = static_cast<T *>(p.out) + token * p.out_stride[0] + head * p.out_stride[1];
      for (int d = lane; d < p.dim; d += 32) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += all[(w * kRows + r) * N::kJoin + d];
        out[d] = Elem<T>::put(v * inverse);
      }
      if (lane == 0 && p.lse != nullptr) p.lse[at] = lse2 * 0.6931471805599453f;
    } else {
      const i64 slot = it.slot * p.tokens * p.heads + at;
      for (int d = lane * 4; d < p.dim; d += 128) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 x = *reinterpret_cast<const float4 *>(all + (w * kRows + r) * N::kJoin + d);
          v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        v.x *= inverse, v.y *= inverse, v.z *= inverse, v.w *= inverse;
        *reinterpret_cast<float4 *>(p.partial + slot * p.dim + d) = v;
      }
      if (lane == 0) p.partial_lse[slot] = lse2;
    }
  }
}

// Launched behind the wide form, whose results it does not read, it may run beside
// it; the first block ends after it, so that what waits for this grid waits for
// both.
template <typename T, int DP, int NT, bool kTma>
__global__ void __launch_bounds__(kWarps * 32)
attend_narrow_kernel(const __grid_constant__ AttendParams p, const __grid_constant__ tila::TensorMap kmap,
                     const __grid_constant__ tila::TensorMap vmap, int prefix_items, int prefix_tiles, int own_tiles) {
  tila::grid_dep_release();
  narrow_block<T, DP, NT, kTma>(p, kmap, vmap, prefix_items, prefix_tiles, own_tiles);
  if (blockIdx.x == 0 && threadIdx.x == 0) tila::grid_dep_wait();
}

// The weighted sum of a row's partial results, N slots in flight at a time: the
// running maximum lets rows be loaded beside their weights.  With short rows no load
// is conditional (slots behind the last read the last one, with no weight): 16000 rows
// of 3 slots of 64 elements take 6 us so and 10 us otherwise; with longer rows, of which
// there are fewer with more slots, it costs 2 us.
template <int I> struct Joined { float top = kNegInf, sum = 0.f, acc[I * 4] = {}; };
// Slots `from`, `from` + `by` and so on.
template <int L, int I, int N>
__device__ __forceinline__ void join_slots(const AttendParams &p, i64 at, i64 step, int slots, int from, int by, int lane,
                                           Joined<I> &j) {
  constexpr bool kAlways = L == 16;
  for (int s0 = from; s0 < slots; s0 += N * by) {
    float lse[N];
    float4 row[N][I];
#pragma unroll
    for (int s = 0; s < N; ++s) {
      lse[s] = kNegInf;
      const int slot = s0 + s * by;
      if (!kAlways && slot >= slots) continue;
      const i64 place = (kAlways ? min(slot, slots - 1) : slot) * step + at;
      lse[s] = p.partial_lse[place];
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int d = lane * 4 + i * 4 * L;
        row[s][i] = *reinterpret_cast<const float4 *>(p.partial + place * p.dim + (d < p.dim ? d : 0));
      }
    }
    float high = j.top;
#pragma unroll
    for (int s = 0; s < N; ++s) {
      if (s0 + s * by >= slots) lse[s] = kNegInf;
      high = fmaxf(high, lse[s]);
    }
    const float base = high == kNegInf ? 0.f : high;
    const float f = exp2f(j.top - base);
    j.top = high;
    j.sum *= f;
#pragma unroll
    for (int i = 0; i < I * 4; ++i) j.acc[i] *= f;
#pragma unroll
    for (int s = 0; s < N; ++s) {
      const float w = exp2f(lse[s] - base);
      j.sum += w;
      if (w != 0.f)                                          // (a slot that nothing was seen in may hold anything)
#pragma unroll
        for (int i = 0; i < I; ++i) {
          j.acc[i * 4] = fmaf(w, row[s][i].x, j.acc[i * 4]);
          j.acc[i * 4 + 1] = fmaf(w, row[s][i].y, j.acc[i * 4 + 1]);
          j.acc[i * 4 + 2] = fmaf(w, row[s][i].z, j.acc[i * 4 + 2]);
          j.acc[i * 4 + 3] = fmaf(w, row[s][i].w, j.acc[i * 4 + 3]);
        }
    }
  }
}

// out = sum over slots of 2^(lse_s - lse) * partial_s, lse = log2 sum 2^lse_s: L lanes
// for each row of q and head.  Bound by reading the partial results, which the
// blocks before left in L2.  Which row, sequence and chunks is found out before the
// wait for them: lengths and offsets are older than the kernels waited for.
// `kBlock`: a whole block for each row, its groups of L lanes take the slots in turn:
// few rows of many slots, which would wait for one another's loads.
template <typename T, int L, int I, bool kBlock>
__global__ void __launch_bounds__(256) attend_join_kernel(const __grid_constant__ AttendParams p) {
  constexpr int kParts = kBlock ? 256 / L : 1;
  const int lane = threadIdx.x % L, part = kBlock ? threadIdx.x / L : 0;
  const i64 at = kBlock ? blockIdx.x : static_cast<i64>(blockIdx.x) * (256 / L) + threadIdx.x / L;
  const bool there = at < p.tokens * p.heads;
  const int token = there ? static_cast<int>(at) / p.heads : 0;
  const int head = static_cast<int>(at) - token * p.heads;
  // the row's sequence, and the chunks of its own tokens that it saw
  int b = token;
  if (p.offsets != nullptr && p.batch <= 8 * L) {
    // the last b with offsets[b] <= token, all looked at in one go by the row's lanes
    int before = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      before += lane + i * L < p.batch && p.offsets[min(lane + i * L, p.batch)] <= token;
#pragma unroll
    for (int x = L / 2; x > 0; x >>= 1) before += __shfl_xor_sync(0xffffffffu, before, x);
    b = max(before - 1, 0);
  } else if (p.offsets != nullptr) {
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      (p.offsets[mid] <= token ? lo : hi) = mid;
    }
    b = lo;
  }
  i64 first = 0;
  int count = 0, slots = 0;
  if (there && b < p.batch) {
    sequence_rows(p, b, first, count);
    const int length = own_length(p, b), keys = own_chunk(p, length);
    const int limit = length - count + 1 + static_cast<int>(token - first);
    slots = p.prefix_chunks + (limit <= 0 ? 0 : min((limit + keys - 1) / keys, p.own_chunks));
  }
  tila::grid_dep_wait();
  if (!there || token < first || token >= first + count) return;
  const i64 step = p.tokens * p.heads;
  Joined<I> j;
  join_slots<L, I, kBlock || L == 16 ? 4 : 8>(p, at, step, slots, part, kParts, lane, j);
  if constexpr (kBlock) {
    // the groups' sums, by the first group
    __shared__ float2 seen[kParts];
    __shared__ float4 sums[kParts][L * I];
    if (lane == 0) seen[part] = make_float2(j.top, j.sum);
#pragma unroll
    for (int i = 0; i < I; ++i)
      sums[part][lane + i * L] = make_float4(j.acc[i * 4], j.acc[i * 4 + 1], j.acc[i * 4 + 2], j.acc[i * 4 + 3]);
    __syncthreads();
    if (part != 0) return;
    j = Joined<I>{};
#pragma unroll
    for (int k = 0; k < kParts; ++k) j.top = fmaxf(j.top, seen[k].x);
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      // (a group that saw nothing has sums of 0, or not a number)
      const float f = seen[k].x == kNegInf ? 1.f : exp2f(seen[k].x - j.top);
      j.sum += seen[k].y * f;
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const float4 x = sums[k][lane + i * L];
        j.acc[i * 4] = fmaf(f, x.x, j.acc[i * 4]);
        j.acc[i * 4 + 1] = fmaf(f, x.y, j.acc[i * 4 + 1]);
        j.acc[i * 4 + 2] = fmaf(f, x.z, j.acc[i * 4 + 2]);
        j.acc[i * 4 + 3] = fmaf(f, x.w, j.acc[i * 4 + 3]);
      }
    }
  }
  const float top = j.top, sum = j.sum;
  const float (&acc)[I * 4] = j.acc;
  const float inverse = sum == 0.f ? 0.f : 1.f / sum;
  T *out = static_cast<T *>(p.out) + static_cast<i64>(token) * p.out_stride[0] + head * p.out_stride[1];
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int d = lane * 4 + i * 4 * L;
    if (d < p.dim) {
      if (p.out_vectors)
        *reinterpret_cast<uint2 *>(out + d) = make_uint2(pack_pair<T>(acc[i * 4] * inverse, acc[i * 4 + 1] * inverse),
                                                         pack_pair<T>(acc[i * 4 + 2] * inverse, acc[i * 4 + 3] * inverse));
      else
#pragma unroll
        for (int e = 0; e < 4; ++e) out[d + e] = Elem<T>::put(acc[i * 4 + e] * inverse);
    }
  }
  if (lane == 0 && p.lse != nullptr) p.lse[at] = sum == 0.f ? kNegInf : (top + log2f(sum)) * 0.6931471805599453f;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

int check(const tila_attend_args *a, char *log, size_t cap) {
  const char *who = "tila_attend_shared_prefix";
  if (a == nullptr || a->size != sizeof(tila_attend_args) || a->reserved != 0 || a->max_length < 0)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: args.size is not that of this library's structure", who);
  if (a->dtype != TILA_F16 && a->dtype != TILA_BF16)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: dtype must be TILA_F16 or TILA_BF16", who);
  if (a->tokens < 0 || a->batch < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: heads must be a multiple of kv_heads", who);
  if (a->dim < 8 || a->dim > 256 || a->dim % 8 != 0)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: dim must be a multiple of 8 up to 256", who);
  if (!std::isfinite(a->scale * 1.4426950408889634f))
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: scale must be finite", who);
  if (a->page_size < 1 || a->table_width < 0 || a->max_queries < 1 || a->num_pages < 0 || a->prefix_length < 0)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: a size is out of range", who);
  constexpr i64 most = 1ll << 30;
  if (a->num_pages > 0x7fffffff || a->prefix_length > most || a->tokens > most ||
      static_cast<i64>(a->table_width) * a->page_size > most || a->tokens * a->heads > most ||
      static_cast<i64>(a->max_queries) * a->heads > most)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: more than 2^30 tokens or rows", who);
  if (a->query_offsets == 0 && a->tokens < a->batch)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: q has fewer rows than the batch", who);
  if (a->tokens > 0 && a->batch > 0) {
    if (a->q == 0 || a->out == 0 || a->q % 2 != 0 || a->out % 2 != 0 || a->lse % 4 != 0)
      return fail(TILA_ERR_ARGUMENT, log, cap, "%s: an address is missing or not aligned to its elements", who);
    if (a->lengths == 0 || (a->table_width > 0 && a->page_table == 0) || (a->prefix_length > 0 && a->prefix_pages == 0))
      return fail(TILA_ERR_ARGUMENT, log, cap, "%s: lengths or pages are missing", who);
    if ((a->lengths | a->page_table | a->query_offsets | a->prefix_pages) % 4 != 0 || a->err % 8 != 0)
      return fail(TILA_ERR_ARGUMENT, log, cap, "%s: lengths, offsets, pages or err are not aligned to their elements", who);
    bool ok = a->k_cache % 16 == 0 && a->v_cache % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && a->k_stride[i] % 8 == 0 && a->v_stride[i] % 8 == 0;
    if (!ok || (a->num_pages > 0 && (a->k_cache == 0 || a->v_cache == 0)))
      return fail(TILA_ERR_ARGUMENT, log, cap, "%s: cache rows must start on 16-byte boundaries", who);
  }
  return TILA_OK;
}

struct Plan {
  AttendParams p;
  int narrow_rows;               // of a block: 8 or 16
  int prefix_tiles, own_tiles;   // of as many rows
  bool prefix_wide, own_wide, narrow_tma;
  i64 slots;
};

// Chunks of the wide form, one block a multiprocessor.  A block takes about 2.1 us
// for a tile of 128 keys and 9.5 us beside that (queries, filling the ring, results).
// That is the tile at 128 elements and the price at any size: at 64, where a tile takes
// 1.4, that price would split most calls alike and some better (16 of 128 new tokens on
// 4096, 16 heads 94.1 us with either; 64 on 8192, 8 key heads 46.7 us with 2.1, 45.2 with
// 1.4).
// Where the narrow form follows (`narrow_bytes`, half of what the longest sequences
// would be), it starts beside the wide form on the multiprocessors that are left,
// which fetch about 58 GB/s each, 6.7 TB/s in all, and takes 8 us beside that: the
// split that ends both first (of those that give the wide form 48 multiprocessors at
// least, since lengths may be far below what the table could hold).  128 sequences of up
// to 4096 own tokens on 32768 shared ones: 199 us so, 237 us with the wide form on
// every multiprocessor first; 64 of up to 1024 on 8192: 40 and 46 us.
int wide_chunk_of(i64 keys, i64 blocks, double narrow_bytes, int &chunks) {
  const i64 tiles = (keys + 127) / 128;
  const i64 most = std::min<i64>(tiles, 64);
  i64 best = 0;
  double least = 0;
  for (i64 n = 1; n <= most; ++n) {
    if (narrow_bytes > 0 && blocks * n < 48 && n < most) continue;
    const double wide = ((blocks * n + kSms - 1) / kSms) * (9.5e-6 + 2.1e-6 * ((tiles + n - 1) / n));
    const double beside = std::min(6.7e12, 58e9 * std::max<i64>(0, kSms - blocks * n));
    const double left = std::max(0., narrow_bytes - beside * wide);
    const double narrow = narrow_bytes <= 0 ? 0. : 8e-6 + (left > 0 ? wide + left / 6.7e12 : narrow_bytes / beside);
    const double cost = std::max(wide, narrow);
    if (best == 0 || cost < least) best = n, least = cost;
  }
  const i64 each = (tiles + best - 1) / best;
  chunks = static_cast<int>((tiles + each - 1) / each);
  return static_cast<int>(each * 128);
}

// Chunks of the prefix in the narrow form: enough blocks for four a multiprocessor,
// and none longer than 512 keys while there are at most 4096 blocks (nine waves): with
// more, shorter chunks even out nothing, and each leaves a partial result for every row
// (64 sequences of 128 new tokens of 32 heads on 32768 keys in pages of 48: 270 MB of
// workspace in one chunk, 8.8 GB in 64; on 8192 keys in pages of 1 7.8 ms in one chunk,
// 11.7 in 16; 128 single tokens, heads of 256 elements, on 32768 2.2 ms in 16, 2.8 in 64).
int chunk_of(i64 keys, i64 blocks, int &chunks) {
  if (keys <= 0) {
    chunks = 0;
    return kStep;
  }
  const i64 want = std::max<i64>(1, (4 * kSms + blocks - 1) / std::max<i64>(1, blocks));
  const i64 even = std::max<i64>(1, 4096 / blocks);          // chunks of that many blocks
  i64 chunk = std::min(std::max<i64>(512, (keys + even - 1) / even), (keys + want - 1) / want);
  chunk = std::max<i64>(chunk, (keys + 255) / 256);          // at most 256 slots
  chunk = (chunk + kStep - 1) / kStep * kStep;
  chunks = static_cast<int>((keys + chunk - 1) / chunk);
  return static_cast<int>(chunk);
}

// Chunks of each sequence in the narrow form: enough blocks for four a
// multiprocessor, and up to 8 of 512 keys beyond that, since
// sequences end at different lengths and the longest chunk is what the last block
// waits for; not more than 16384 blocks for it, since those of short sequences start in
// vain (0.7 us each).  A chunk's partial result costs 8 bytes an element beside 4 bytes
// a key for every row.
int own_chunks_of(i64 keys, i64 blocks) {
  const i64 fill = (4 * kSms + blocks - 1) / blocks;
  const i64 even = std::min<i64>({8, (keys + 511) / 512, std::max<i64>(1, 16384 / blocks)});
  return static_cast<int>(std::max<i64>(1, std::min<i64>({(keys + kStep - 1) / kStep, 256, std::max(fill, even)})));
}

// Whether blocks of own tokens (wide, one chunk a sequence) should go through the prefix
// too: then there are no partial results and no join, but a tile of keys serves 128
// rows of one sequence where the prefix's own blocks fill 256 from all.  Estimates in us;
// a tile takes 2.1 either way (at 64 elements 2.0 and 1.4), a wave of the prefix's blocks
// 9.5 beside that, partial results are written and read at about 5 TB/s.  Measured so and
// apart: 110 sequences of 42 tokens on 13 shared, 40 heads 82 and 200 us; 34 of up to 104 on
// 1000, 56 heads 128 and 235, on 4000 302 and 378; 8 of 512 on 1000 87 and 173; 16 of 128
// on 4096, 16 heads of 64 elements 88 and 68; 87 of 40 on 1000, 4 heads 59 and 44.
bool inside_is_faster(const AttendParams &p, i64 rows, i64 own_blocks) {
  const double tiles = (p.prefix + 127) / 128, chunks = p.prefix_chunks;
  const i64 blocks = std::min<i64>(own_blocks, (rows / 128 + p.batch) * p.kv_heads);   // that have rows
  double waves = blocks / (2. * kSms);
  if (waves < 2) waves = std::ceil(waves);
  const double inside = waves * tiles * (p.dim <= 64 ? 2.0 : 2.1);
  const double prefix_waves = std::ceil((rows + 255) / 256 * p.kv_heads * chunks / kSms);
  const double apart = prefix_waves * (9.5 + std::ceil(tiles / chunks) * (p.dim <= 64 ? 1.4 : 2.1));
  const double join = 3 + 8. * (chunks + 1) * rows * p.kv_heads * p.dim / 5e6;
  return inside < 0.9 * (apart + join);
}

Plan plan(const tila_attend_args &a) {
  Plan r{};
  AttendParams &p = r.p;
  p.q = reinterpret_cast<const void *>(a.q);
  p.k = reinterpret_cast<const void *>(a.k_cache);
  p.v = reinterpret_cast<const void *>(a.v_cache);
  p.out = reinterpret_cast<void *>(a.out);
  p.lse = reinterpret_cast<float *>(a.lse);
  for (int i = 0; i < 2; ++i) {
    p.q_stride[i] = a.q_stride[i];
    p.out_stride[i] = a.out_stride[i];
  }
  for (int i = 0; i < 3; ++i) {
    p.k_stride[i] = a.k_stride[i];
    p.v_stride[i] = a.v_stride[i];
  }
  p.table = reinterpret_cast<const i32 *>(a.page_table);
  p.table_stride = a.table_stride;
  p.lengths = reinterpret_cast<const i32 *>(a.lengths);
  p.offsets = reinterpret_cast<const i32 *>(a.query_offsets);
  p.prefix_pages = reinterpret_cast<const i32 *>(a.prefix_pages);
  p.tokens = a.tokens;
  p.err = reinterpret_cast<u32 *>(a.err);
  p.batch = a.batch;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.group = a.heads / a.kv_heads;
  p.dim = a.dim;
  p.page_size = a.page_size;
  p.page_shift = -1;
  for (int s = 0; s < 30; ++s)
    if (a.page_size == 1 << s) p.page_shift = s;
  p.table_width = a.table_width;
  p.num_pages = static_cast<int>(a.num_pages);
  p.max_queries = a.query_offsets == 0 ? 1 : a.max_queries;
  p.prefix = static_cast<int>(a.prefix_length);
  p.scale2 = a.scale * 1.4426950408889634f;
  p.q_words = a.q % 4 == 0 && a.q_stride[0] % 2 == 0 && a.q_stride[1] % 2 == 0;
  const i64 rows = (a.query_offsets == 0 ? a.batch : a.tokens) * p.group;
  p.q_vectors = a.q % 16 == 0 && a.q_stride[0] % 8 == 0 && a.q_stride[1] % 8 == 0;
  p.out_vectors = a.out % 8 == 0 && a.out_stride[0] % 4 == 0 && a.out_stride[1] % 4 == 0;
  const i64 own_rows = static_cast<i64>(p.max_queries) * p.group;
  const i64 table_keys = static_cast<i64>(a.table_width) * a.page_size;
  const i64 own_keys = a.max_length > 0 ? std::min<i64>(a.max_length, table_keys) : table_keys;
  const bool wide = wide_possible(a);
  r.narrow_tma = tma_possible(a) && a.page_size % kSlice == 0;
  // The prefix: the narrow form would take longer, however few keys (256 rows a head on 512
  // keys 32 us, wide 23; on 2048 44 and 27; 28 rows on 425 19 and 17).  Own tokens:
  // up to 32 rows fill a quarter of a row tile, and two blocks of 16 that read the keys
  // twice, once from L2, are faster (28 rows, 21 sequences of up to 3462 tokens: 32 us, wide
  // 39; 20 rows, 64 of up to 1000: 34 and 48; 64 rows 43 either way).
  r.prefix_wide = wide && p.prefix > 0 && rows > 16 && wide_fits(a, false);
  r.own_wide = wide && own_keys > 0 && own_rows > 32 && wide_fits(a, true);
  r.narrow_rows = (r.own_wide || own_rows <= 8) && (r.prefix_wide || rows <= 8) ? 8 : 16;
  r.prefix_tiles = static_cast<int>((rows + r.narrow_rows - 1) / r.narrow_rows);
  r.own_tiles = static_cast<int>((own_rows + r.narrow_rows - 1) / r.narrow_rows);
  p.prefix_chunk = r.prefix_wide
                       ? wide_chunk_of(p.prefix, (rows + 255) / 256 * p.kv_heads,
                                       r.own_wide ? 0. : 2. * own_keys * p.batch * p.kv_heads * p.dim, p.prefix_chunks)
                       : chunk_of(p.prefix, static_cast<i64>(r.prefix_tiles) * p.kv_heads, p.prefix_chunks);
  const i64 own_blocks = r.own_wide ? (own_rows + 127) / 128 * p.kv_heads * p.batch
                                    : static_cast<i64>(r.own_tiles) * p.kv_heads * p.batch;
  p.own_unit = r.own_wide ? 128 : kStep;
  // wide: two blocks a multiprocessor, or up to four while a chunk has 8 tiles, since the
  // longest sequence is what the last block waits for (168 blocks of up to 27 tiles: 72 us
  // in three chunks, 99 in one; 256 of up to 8: 68 us in one, 73 in two)
  p.own_chunks = own_keys == 0 ? 0
                 : r.own_wide  ? static_cast<int>(std::max<i64>({1, std::min<i64>(2 * kSms / own_blocks, (own_keys + 127) / 128),
                                                                  std::min<i64>(4 * kSms / own_blocks, (own_keys + 1023) / 1024)}))
                               : own_chunks_of(own_keys, own_blocks);
  p.own_least = p.own_unit;
  // where there are blocks enough, shorter sequences are not cut as finely as the longest:
  // 128 of up to 4096 tokens in chunks of 512 201 us, in eighths 217 us
  if (!r.own_wide && p.own_chunks > 0 && own_blocks >= 2 * kSms)
    p.own_least = static_cast<int>(std::min<i64>(512, (own_keys / p.own_chunks + kStep - 1) / kStep * kStep));
  p.own_least = std::max(p.own_least, p.own_unit);
  if (p.own_chunks == 0 && p.prefix_chunks == 0) p.own_chunks = 1;   // no keys at all: a block writes the zeros
  if (r.own_wide && r.prefix_wide && p.own_chunks == 1 && inside_is_faster(p, rows, own_blocks)) {
    p.prefix_inside = 1;
    p.prefix_chunks = 0;
    r.prefix_wide = false;
  }
  r.slots = p.prefix_chunks + p.own_chunks;
  p.direct = r.slots == 1 && p.prefix_chunks == 0;
  return r;
}

u64 workspace_of(const Plan &r) {
  return r.p.direct ? 0 : static_cast<u64>(r.slots) * r.p.tokens * r.p.heads * (r.p.dim + 1) * sizeof(float);
}

template <typename T, int DP, int NT, bool kTma>
cudaError_t launch_narrow(const Plan &r, const tila::TensorMap &k, const tila::TensorMap &v, cudaStream_t stream) {
  const i64 prefix_items = r.prefix_wide ? 0 : static_cast<i64>(r.prefix_tiles) * r.p.kv_heads * r.p.prefix_chunks;
  const i64 own_items = r.own_wide ? 0 : static_cast<i64>(r.own_tiles) * r.p.kv_heads * r.p.own_chunks * r.p.batch;
  if (prefix_items + own_items == 0) return cudaSuccess;
  if (prefix_items + own_items > 0x7fffffff) return cudaErrorInvalidValue;
  constexpr auto kernel = attend_narrow_kernel<T, DP, NT, kTma>;
  const cudaError_t e = allow_shared_memory<kernel>(Narrow<DP>::kBytes);
  if (e != cudaSuccess) return e;
  return launch_kernel(kernel, static_cast<unsigned>(prefix_items + own_items), kWarps * 32, Narrow<DP>::kBytes,
                       stream, r.prefix_wide || r.own_wide, r.p, k, v, static_cast<int>(prefix_items), r.prefix_tiles, r.own_tiles);
}

template <typename T, int DP>
cudaError_t launch_narrow(const Plan &r, const tila::TensorMap &k, const tila::TensorMap &v, cudaStream_t stream) {
  if (r.narrow_rows == 8)
    return r.narrow_tma ? launch_narrow<T, DP, 1, true>(r, k, v, stream) : launch_narrow<T, DP, 1, false>(r, k, v, stream);
  return r.narrow_tma ? launch_narrow<T, DP, 2, true>(r, k, v, stream) : launch_narrow<T, DP, 2, false>(r, k, v, stream);
}

template <typename T>
cudaError_t launch(const Plan &r, const tila::TensorMap &k, const tila::TensorMap &v, cudaStream_t stream) {
  cudaError_t e = r.p.dim <= 64    ? launch_narrow<T, 64>(r, k, v, stream)
                  : r.p.dim <= 128 ? launch_narrow<T, 128>(r, k, v, stream)
                                   : launch_narrow<T, 256>(r, k, v, stream);
  if (e != cudaSuccess || r.p.direct) return e;
  const int lanes = r.p.dim <= 64 ? 16 : 32;
  const unsigned blocks = static_cast<unsigned>((r.p.tokens * r.p.heads * lanes + 255) / 256);
  const i64 rows = r.p.tokens * r.p.heads;
  if (rows <= 4 * kSms && r.slots > 8)                        // 2048 rows of 20 slots take 5 us more so, 24 of 71 3 less
    return launch_kernel(r.p.dim <= 64    ? attend_join_kernel<T, 16, 1, true>
                         : r.p.dim <= 128 ? attend_join_kernel<T, 32, 1, true>
                                          : attend_join_kernel<T, 32, 2, true>,
                         static_cast<unsigned>(rows), 256, 0, stream, true, r.p);
  return launch_kernel(r.p.dim <= 64    ? attend_join_kernel<T, 16, 1, false>
                       : r.p.dim <= 128 ? attend_join_kernel<T, 32, 1, false>
                                        : attend_join_kernel<T, 32, 2, false>,
                       blocks, 256, 0, stream, true, r.p);
}

}  // namespace

extern "C" int tila_attend_shared_prefix(const tila_attend_args *args, char *log, size_t log_cap) {
  int st = check(args, log, log_cap);
  if (st != TILA_OK) return st;
  if (args->tokens == 0 || args->batch == 0) return TILA_OK;
  Plan r = plan(*args);
  const u64 need = workspace_of(r);
  if (need > 0) {
    if (args->workspace == 0 || args->workspace % 16 != 0 || args->workspace_bytes < need)
      return fail(TILA_ERR_ARGUMENT, log, log_cap,
                  "tila_attend_shared_prefix: workspace is too small or not 16-byte aligned");
    r.p.partial = reinterpret_cast<float *>(args->workspace);
    r.p.partial_lse = r.p.partial + static_cast<u64>(r.slots) * r.p.tokens * r.p.heads * r.p.dim;
  }
  const cudaStream_t stream = reinterpret_cast<cudaStream_t>(args->stream);
  if (r.prefix_wide) st = launch_wide(*args, r.p, true, false, stream, log, log_cap);
  if (st == TILA_OK && r.own_wide) st = launch_wide(*args, r.p, false, r.prefix_wide, stream, log, log_cap);
  if (st != TILA_OK) return st;
  tila::TensorMap k{}, v{};
  if (r.narrow_tma) st = encode_caches(*args, kSlice, &k, &v, log, log_cap);
  if (st != TILA_OK) return st;
  const cudaError_t e =
      args->dtype == TILA_F16 ? launch<__half>(r, k, v, stream) : launch<__nv_bfloat16>(r, k, v, stream);
  return launch_status(e, "tila_attend_shared_prefix", log, log_cap);
}

extern "C" uint64_t tila_attend_workspace(const tila_attend_args *args) {
  if (check(args, nullptr, 0) != TILA_OK || args->tokens == 0 || args->batch == 0) return 0;
  return workspace_of(plan(*args));
}
