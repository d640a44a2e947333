// Attention over a paged cache with a shared prefix: the narrow form for up to
// 16 rows of queries a block, the join of partial results, and the host side
// (the wide form, for more rows, is attend_wide.cu).
//
// Narrow form.  Few rows against many keys: bound by reading the keys and
// values once.  A block of 4 warps takes 16 rows (a sequence's new tokens times
// the heads that share its key head) and one chunk of keys.  Each warp runs on
// its own: it brings 16 keys and values at a time into its own ring of shared
// memory with cp.async (pages may have any size: each lane looks up rows) and
// needs no barrier with the others, so that loads never wait for arithmetic.
// Scores and values go through m16n8k16 matrix instructions with 32-bit sums
// (16 rows do not fill a tcgen05 tile; at these rows the instruction rate is not
// what bounds).  Weights p are rounded to the values' type for the product with
// the values and summed as they are in 32 bits: the sum is also a result (lse),
// and a rounding of p moves it by 2^-9 of a weight.

#include "attend.cuh"
#include "attend_wide.cuh"

#include <algorithm>

namespace {

using namespace tila_ops;

constexpr int kWarps = 4;
constexpr int kSlice = 16;                 // keys of one warp's step
constexpr int kStep = kWarps * kSlice;     // keys of one block's step
constexpr int kStages = 3;

template <typename T> __device__ __forceinline__ u32 pack2(float lo, float hi);
template <> __device__ __forceinline__ u32 pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const u32 *>(&h);
}
template <> __device__ __forceinline__ u32 pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const u32 *>(&h);
}

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
  static constexpr int kRow = DP * 2;                        // bytes of a row in shared memory
  static constexpr int kStage = 2 * kSlice * kRow;           // keys and values of one step
  static constexpr int kWarpBytes = kStages * kStage;
  static constexpr int kBytes = kWarps * kWarpBytes;
  static_assert(kBytes >= kWarps * 16 * DP * 4, "the join of the warps reuses the ring");
};

template <typename T, int DP>
__global__ void __launch_bounds__(kWarps * 32) attend_narrow_kernel(const __grid_constant__ AttendParams p,
                                                                    int prefix_items, int prefix_tiles,
                                                                    int own_tiles) {
  using N = Narrow<DP>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float row_max[kWarps][16], row_sum[kWarps][16];
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
      it.row0 = tile * 16;
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
      it.row0 = tile * 16;
      if (it.row0 >= it.rows) return;
      it.limit0 = length - count + 1;
      const int last = min(it.row0 + 15, it.rows - 1) / p.group;
      it.begin = chunk * p.own_chunk;
      it.end = min(it.begin + p.own_chunk, it.limit0 + last);
      it.pages = p.table + b * p.table_stride;
      // nothing of this chunk is seen: only the sole chunk writes (zeros) then
      if (it.begin >= it.end && !p.direct) return;
    }
  }
  const bool causal = it.slot >= p.prefix_chunks;

  // queries: A fragments of 16 rows, rows g and g + 8 of each lane
  const int g = lane >> 2, c = lane & 3;
  u32 qf[DP / 16][4];
  int limit[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = it.row0 + g + 8 * h;
    const int token = row / p.group;
    limit[h] = row < it.rows ? (causal ? it.limit0 + token : it.limit0) : 0;
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
        qf[k][half * 2 + h] = w;
      }
  }

  // the warp's ring of keys and values
  const u32 ring = tila::smem_u32(smem) + warp * N::kWarpBytes;
  constexpr int kChunks = DP / 8;                            // 16-byte pieces of a row
  const int begin = it.begin + warp * kSlice;
  const int steps = it.end > begin ? (it.end - begin + kStep - 1) / kStep : 0;
  const T *kbase = static_cast<const T *>(p.k) + it.head * p.k_stride[2];
  const T *vbase = static_cast<const T *>(p.v) + it.head * p.v_stride[2];
  // the page of this lane's key (lane & 15) of a step, looked up one step ahead
  auto look_up = [&](int step) {
    const int key = begin + step * kStep + (lane & 15);
    if (key >= it.end) return -1;
    int page, row;
    split_key(p, key, page, row);
    return checked_page(p, it.pages, page);
  };
  int page_ahead = steps > 0 ? look_up(0) : -1;
  auto issue = [&](int step) {
    if (step < steps) {
      const int key = begin + step * kStep + (lane & 15);
      int unused, row;
      split_key(p, key, unused, row);
      const int page = page_ahead;
      i64 koff = -1, voff = 0;
      if (page >= 0) {
        koff = page * p.k_stride[0] + row * p.k_stride[1];
        voff = page * p.v_stride[0] + row * p.v_stride[1];
      }
      page_ahead = look_up(step + 1);
      const u32 stage = ring + (step % kStages) * N::kStage;
#pragma unroll
      for (int i = 0; i < kSlice * kChunks / 32; ++i) {
        const int r = (i * 32 + lane) / kChunks, ch = (i * 32 + lane) % kChunks;
        const i64 ko = __shfl_sync(0xffffffffu, koff, r), vo = __shfl_sync(0xffffffffu, voff, r);
        const int bytes = ko >= 0 && ch * 8 < p.dim ? 16 : 0;
        const u32 at = stage + r * N::kRow + ((ch ^ (r & 7)) << 4);
        copy16(at, bytes ? kbase + ko + ch * 8 : kbase, bytes);
        copy16(at + kSlice * N::kRow, bytes ? vbase + vo + ch * 8 : vbase, bytes);
      }
    }
    copy_commit();
  };

  float o[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};

#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(s);
  for (int step = 0; step < steps; ++step) {
    copy_wait<kStages - 2>();
    __syncwarp();
    issue(step + kStages - 1);
    const u32 stage = ring + (step % kStages) * N::kStage;
    float s[2][4] = {};
    {
      const int r = (lane & 7) + ((lane >> 4) << 3), ch = (lane >> 3) & 1;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        u32 b[4];
        ldmatrix4(b, stage + r * N::kRow + (((k * 2 + ch) ^ (r & 7)) << 4));
        mma16816<T>(s[0], qf[k], b[0], b[1]);
        mma16816<T>(s[1], qf[k], b[2], b[3]);
      }
    }
    const int key0 = begin + step * kStep;
    u32 pf[4];
    float scale[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int end = min(it.end, limit[h]);
      float best = kNegInf;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float &x = s[n][h * 2 + e];
          x = key0 + n * 8 + c * 2 + e < end ? x * p.scale2 : kNegInf;
          best = fmaxf(best, x);
        }
      best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
      best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
      const float top = fmaxf(m[h], best);
      const float base = top == kNegInf ? 0.f : top;         // nothing seen yet: all weights 0
      scale[h] = exp2f(m[h] - base);
      m[h] = top;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float x = tila::exp2_fast(s[n][h * 2] - base), y = tila::exp2_fast(s[n][h * 2 + 1] - base);
        sum += x + y;
        pf[n * 2 + h] = pack2<T>(x, y);
      }
      l[h] = l[h] * scale[h] + sum;
    }
    // the sums follow the maximum only when it moved
    if (__any_sync(0xffffffffu, scale[0] != 1.f || scale[1] != 1.f)) {
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        o[n][0] *= scale[0];
        o[n][1] *= scale[0];
        o[n][2] *= scale[1];
        o[n][3] *= scale[1];
      }
    }
    {
      const int r = (lane & 7) + (((lane >> 3) & 1) << 3), ch = lane >> 4;
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        u32 b[4];
        ldmatrix4t(b, stage + kSlice * N::kRow + r * N::kRow + (((n * 2 + ch) ^ (r & 7)) << 4));
        mma16816<T>(o[2 * n], pf, b[0], b[1]);
        mma16816<T>(o[2 * n + 1], pf, b[2], b[3]);
      }
    }
  }

  // join the warps: maxima, sums, then the scaled results through shared memory
  copy_wait<0>();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (c == 0) {
      row_max[warp][g + 8 * h] = m[h];
      row_sum[warp][g + 8 * h] = l[h];
    }
  }
  __syncthreads();
  float *joined = reinterpret_cast<float *>(smem) + warp * 16 * DP;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h;
    float top = kNegInf;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, row_max[w][r]);
    const float f = m[h] == kNegInf ? 1.f : exp2f(m[h] - top);   // nothing seen: 0 times 1
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
      float2 v = make_float2(o[n][h * 2] * f, o[n][h * 2 + 1] * f);
      *reinterpret_cast<float2 *>(joined + r * DP + n * 8 + c * 2) = v;
    }
  }
  __syncthreads();
  const float *all = reinterpret_cast<const float *>(smem);
  for (int r = warp; r < 16; r += kWarps) {
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
        for (int w = 0; w < kWarps; ++w) v += all[(w * 16 + r) * DP + d];
        out[d] = Elem<T>::put(v * inverse);
      }
      if (lane == 0 && p.lse != nullptr) p.lse[at] = lse2 * 0.6931471805599453f;
    } else {
      const i64 slot = it.slot * p.tokens * p.heads + at;
      for (int d = lane * 4; d < p.dim; d += 128) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 x = *reinterpret_cast<const float4 *>(all + (w * 16 + r) * DP + d);
          v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
        v.x *= inverse, v.y *= inverse, v.z *= inverse, v.w *= inverse;
        *reinterpret_cast<float4 *>(p.partial + slot * p.dim + d) = v;
      }
      if (lane == 0) p.partial_lse[slot] = lse2;
    }
  }
}

// out = sum over slots of 2^(lse_s - lse) * partial_s, lse = log2 sum 2^lse_s: one
// warp for each row of q and head.  Bound by reading the partial results, which
// the blocks before left in L2.
template <typename T>
__global__ void __launch_bounds__(256) attend_join_kernel(const __grid_constant__ AttendParams p) {
  const int lane = threadIdx.x & 31;
  const i64 at = static_cast<i64>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (at >= p.tokens * p.heads) return;
  const i64 token = at / p.heads;
  const int head = static_cast<int>(at - token * p.heads);
  // the row's sequence, and the chunks of its own tokens that it saw
  int b = static_cast<int>(token);
  if (p.offsets != nullptr) {
    int lo = 0, hi = p.batch;                 // the last b with offsets[b] <= token
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      (p.offsets[mid] <= token ? lo : hi) = mid;
    }
    b = lo;
  }
  if (b >= p.batch) return;
  i64 first;
  int count;
  sequence_rows(p, b, first, count);
  if (token < first || token >= first + count) return;
  const int limit = own_length(p, b) - count + 1 + static_cast<int>(token - first);
  const int own = limit <= 0 ? 0 : min((limit + p.own_chunk - 1) / p.own_chunk, p.own_chunks);
  const int slots = p.prefix_chunks + own;
  const i64 step = p.tokens * p.heads;
  float top = kNegInf;
  for (int s = lane; s < slots; s += 32) top = fmaxf(top, p.partial_lse[s * step + at]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  const float base = top == kNegInf ? 0.f : top;
  float sum = 0.f;
  float acc[8] = {};
  for (int s0 = 0; s0 < slots; s0 += 32) {
    const float w = s0 + lane < slots ? exp2f(p.partial_lse[(s0 + lane) * step + at] - base) : 0.f;
    sum += w;
    const int n = min(32, slots - s0);
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float ws = __shfl_sync(0xffffffffu, w, s);
      const float *row = p.partial + ((s0 + s) * step + at) * p.dim;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int d = lane * 4 + i * 128;
        if (d < p.dim) {
          const float4 x = *reinterpret_cast<const float4 *>(row + d);
          acc[i * 4] = fmaf(ws, x.x, acc[i * 4]);
          acc[i * 4 + 1] = fmaf(ws, x.y, acc[i * 4 + 1]);
          acc[i * 4 + 2] = fmaf(ws, x.z, acc[i * 4 + 2]);
          acc[i * 4 + 3] = fmaf(ws, x.w, acc[i * 4 + 3]);
        }
      }
    }
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
  const float inverse = sum == 0.f ? 0.f : 1.f / sum;
  T *out = static_cast<T *>(p.out) + token * p.out_stride[0] + head * p.out_stride[1];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = lane * 4 + i * 128;
    if (d < p.dim)
#pragma unroll
      for (int e = 0; e < 4; ++e) out[d + e] = Elem<T>::put(acc[i * 4 + e] * inverse);
  }
  if (lane == 0 && p.lse != nullptr) p.lse[at] = sum == 0.f ? kNegInf : (base + log2f(sum)) * 0.6931471805599453f;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

int check(const tila_attend_args *a, char *log, size_t cap) {
  const char *who = "tila_attend_shared_prefix";
  if (a == nullptr || a->size != sizeof(tila_attend_args))
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: args.size is not that of this library's structure", who);
  if (a->dtype != TILA_F16 && a->dtype != TILA_BF16)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: dtype must be TILA_F16 or TILA_BF16", who);
  if (a->tokens < 0 || a->batch < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: heads must be a multiple of kv_heads", who);
  if (a->dim < 8 || a->dim > 256 || a->dim % 8 != 0)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: dim must be a multiple of 8 up to 256", who);
  if (a->page_size < 1 || a->table_width < 0 || a->max_queries < 1 || a->num_pages < 0 || a->prefix_length < 0)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: a size is out of range", who);
  constexpr i64 most = 1ll << 30;
  if (a->num_pages > 0x7fffffff || a->prefix_length > most ||
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
    bool ok = a->k_cache % 16 == 0 && a->v_cache % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && a->k_stride[i] % 8 == 0 && a->v_stride[i] % 8 == 0;
    if (!ok || (a->num_pages > 0 && (a->k_cache == 0 || a->v_cache == 0)))
      return fail(TILA_ERR_ARGUMENT, log, cap, "%s: cache rows must start on 16-byte boundaries", who);
  }
  return TILA_OK;
}

struct Plan {
  AttendParams p;
  int prefix_tiles, own_tiles;   // 16 rows each
  bool prefix_wide, own_wide;
  i64 slots;
};

// Chunks of the wide form: one block a multiprocessor, so that the blocks of all
// chunks fill whole waves; a block costs about 4 tiles of keys beside its own
// (filling the ring, the results).
int wide_chunk_of(i64 keys, i64 blocks, int &chunks) {
  const i64 tiles = (keys + 127) / 128;
  i64 best = 1, cost = 0;
  for (i64 n = 1; n <= std::min<i64>(tiles, 64); ++n) {
    const i64 c = ((blocks * n + kSms - 1) / kSms) * ((tiles + n - 1) / n + 4);
    if (n == 1 || c < cost) best = n, cost = c;
  }
  const i64 each = (tiles + best - 1) / best;
  chunks = static_cast<int>((tiles + each - 1) / each);
  return static_cast<int>(each * 128);
}

// Chunks: enough blocks for two a multiprocessor and twice that many again, and
// none longer than 512 keys beyond that, since sequences end at different
// lengths and the longest chunk is what the last block waits for.  A chunk's
// partial result costs 8 bytes an element beside 4 bytes a key for every row.
int chunk_of(i64 keys, i64 blocks, int &chunks) {
  if (keys <= 0) {
    chunks = 0;
    return kStep;
  }
  const i64 want = std::max<i64>(1, (4 * kSms + blocks - 1) / std::max<i64>(1, blocks));
  i64 chunk = std::min<i64>(512, (keys + want - 1) / want);
  chunk = std::max<i64>(chunk, (keys + 255) / 256);          // at most 256 slots
  chunk = (chunk + kStep - 1) / kStep * kStep;
  chunks = static_cast<int>((keys + chunk - 1) / chunk);
  return static_cast<int>(chunk);
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
  r.prefix_tiles = static_cast<int>((rows + 15) / 16);
  r.own_tiles = (p.max_queries * p.group + 15) / 16;
  p.q_vectors = a.q % 16 == 0 && a.q_stride[0] % 8 == 0 && a.q_stride[1] % 8 == 0;
  const i64 own_rows = static_cast<i64>(p.max_queries) * p.group;
  const i64 own_keys = static_cast<i64>(a.table_width) * a.page_size;
  const bool wide = wide_possible(a);
  r.prefix_wide = wide && p.prefix > 0 && rows > 16;
  r.own_wide = wide && own_keys > 0 && own_rows > 16;
  p.prefix_chunk = r.prefix_wide
                       ? wide_chunk_of(p.prefix, (rows + 255) / 256 * p.kv_heads, p.prefix_chunks)
                       : chunk_of(p.prefix, static_cast<i64>(r.prefix_tiles) * p.kv_heads, p.prefix_chunks);
  p.own_chunk = r.own_wide
                    ? wide_chunk_of(own_keys, (own_rows + 255) / 256 * p.kv_heads * p.batch, p.own_chunks)
                    : chunk_of(own_keys, static_cast<i64>(r.own_tiles) * p.kv_heads * p.batch, p.own_chunks);
  if (p.own_chunks == 0 && p.prefix_chunks == 0) p.own_chunks = 1;   // no keys at all: a block writes the zeros
  r.slots = p.prefix_chunks + p.own_chunks;
  p.direct = r.slots == 1 && p.prefix_chunks == 0;
  return r;
}

u64 workspace_of(const Plan &r) {
  return r.p.direct ? 0 : static_cast<u64>(r.slots) * r.p.tokens * r.p.heads * (r.p.dim + 1) * sizeof(float);
}

template <typename T, int DP>
cudaError_t launch_narrow(const Plan &r, cudaStream_t stream) {
  const i64 prefix_items = r.prefix_wide ? 0 : static_cast<i64>(r.prefix_tiles) * r.p.kv_heads * r.p.prefix_chunks;
  const i64 own_items = r.own_wide ? 0 : static_cast<i64>(r.own_tiles) * r.p.kv_heads * r.p.own_chunks * r.p.batch;
  if (prefix_items + own_items == 0) return cudaSuccess;
  if (prefix_items + own_items > 0x7fffffff) return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(attend_narrow_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Narrow<DP>::kBytes);
  if (e != cudaSuccess) return e;
  attend_narrow_kernel<T, DP><<<static_cast<unsigned>(prefix_items + own_items), kWarps * 32, Narrow<DP>::kBytes,
                                stream>>>(r.p, static_cast<int>(prefix_items), r.prefix_tiles, r.own_tiles);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch(const Plan &r, cudaStream_t stream) {
  cudaError_t e = r.p.dim <= 64    ? launch_narrow<T, 64>(r, stream)
                  : r.p.dim <= 128 ? launch_narrow<T, 128>(r, stream)
                                   : launch_narrow<T, 256>(r, stream);
  if (e != cudaSuccess || r.p.direct) return e;
  attend_join_kernel<T><<<static_cast<unsigned>((r.p.tokens * r.p.heads + 7) / 8), 256, 0, stream>>>(r.p);
  return cudaGetLastError();
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
  if (r.prefix_wide) st = launch_wide(*args, r.p, true, stream, log, log_cap);
  if (st == TILA_OK && r.own_wide) st = launch_wide(*args, r.p, false, stream, log, log_cap);
  if (st != TILA_OK) return st;
  const cudaError_t e = args->dtype == TILA_F16 ? launch<__half>(r, stream) : launch<__nv_bfloat16>(r, stream);
  return launch_status(e, "tila_attend_shared_prefix", log, log_cap);
}

extern "C" uint64_t tila_attend_workspace(const tila_attend_args *args) {
  if (check(args, nullptr, 0) != TILA_OK || args->tokens == 0 || args->batch == 0) return 0;
  return workspace_of(plan(*args));
}
