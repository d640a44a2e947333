// Rotary positions over rows of heads, alone, after a norm of each row, and on
// the way into a paged cache; and the gradients of the normed form.
//
// A row x (one head of one token, `dim` elements) becomes
//     y = a * R(p) * n,    n = x  or  n_j = w_j * x_j / sqrt(mean(x^2) + eps)
// where R turns each pair (n_i, n_p) by the angle p * inv_freq_i and leaves the
// elements behind `rotary` as they are.  The angle is reduced to a part of one
// turn in 64 bits (positions in the millions keep 1e-10 of a turn there, where
// 32 bits would lose the angle), and only that part goes through sincospi in 32
// bits.  All products and sums are 32-bit; a result is rounded once, when it is
// stored.
//
// Bound by memory: a row is read once and written once.  One block takes a few
// tokens with all their heads, of every tensor of the call, so that the sines
// of a token are computed once and shared through shared memory.  A row is
// spread over as many lanes as it has units; a unit is the two V-element vectors
// that hold both halves of V pairs, so that neither layout moves data between
// lanes, and V elements are one 16-byte access where sizes, strides and
// addresses allow it.  The first row's loads are issued before the sines.

#include "ops_common.cuh"

#include <algorithm>

namespace {

using namespace tila_ops;

struct Rows {
  const void *src;
  void *dst;
  const void *weight;
  const void *grad;
  i64 src_stride[3], dst_stride[3], grad_stride[3];
  int heads;
  u32 flags;
};

struct Params {
  Rows rows[3];
  int heads;             // of all tensors
  int num_rows;
  i64 tokens_all, tokens;
  int dim, half, interleaved;
  int lanes;             // lanes of a row, a power of two
  int units;
  int tokens_per_block;
  int any_norm, any_paged;
  float sign;            // -1 rotates back
  float amplitude, eps, inv_dim;
  const void *positions;
  i64 position_stride[2];
  const double *inv_freq;
  const void *slots;
  i64 slot_stride, num_slots;
  int page_size, index64;
  u32 *err;
  float *partial;        // backward: blocks x 2 x dim sums of the weights' gradients
};

__device__ __forceinline__ i64 index_at(const void *p, i64 i, int wide) {
  return wide ? static_cast<const i64 *>(p)[i] : static_cast<i64>(static_cast<const i32 *>(p)[i]);
}

// Offsets of a unit's two vectors inside a row.
template <int V>
__device__ __forceinline__ void unit_at(const Params &p, int u, int &first, int &second) {
  const int pairs = p.half / V;                 // units that rotate
  if (u < pairs && !p.interleaved) {
    first = u * V;
    second = p.half + u * V;
  } else {
    first = 2 * V * u;                          // also the tail: it starts at 2 * V * pairs
    second = first + V;
  }
}

template <typename T, int V, int K>
struct Raw { Vec<T, V> a[K], b[K]; };

template <typename T, int V, int K>
__device__ __forceinline__ void load_row(const Params &p, const T *row, int lane, Raw<T, V, K> &r) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int u = lane + k * p.lanes;
    if (u < p.units) {
      int first, second;
      unit_at<V>(p, u, first, second);
      r.a[k] = *reinterpret_cast<const Vec<T, V> *>(row + first);
      if (second < p.dim) r.b[k] = *reinterpret_cast<const Vec<T, V> *>(row + second);
      else
#pragma unroll
        for (int i = 0; i < V; ++i) r.b[k].e[i] = Elem<T>::put(0.f);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) r.a[k].e[i] = r.b[k].e[i] = Elem<T>::put(0.f);
    }
  }
}

template <typename T, int V, int K>
__device__ __forceinline__ void unpack(const Raw<T, V, K> &r, float (&x)[K][2 * V]) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[k][i] = Elem<T>::get(r.a[k].e[i]);
      x[k][V + i] = Elem<T>::get(r.b[k].e[i]);
    }
}

template <typename T, int V, int K>
__device__ __forceinline__ void store_row(const Params &p, T *row, int lane, const float (&x)[K][2 * V]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int u = lane + k * p.lanes;
    if (u < p.units) {
      int first, second;
      unit_at<V>(p, u, first, second);
      Vec<T, V> a, b;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        a.e[i] = Elem<T>::put(x[k][i]);
        b.e[i] = Elem<T>::put(x[k][V + i]);
      }
      *reinterpret_cast<Vec<T, V> *>(row + first) = a;
      if (second < p.dim) *reinterpret_cast<Vec<T, V> *>(row + second) = b;
    }
  }
}

// Turns the pairs of a row; `tab` holds (cos, sin) of the row's token, the
// amplitude in both.
template <int V, int K>
__device__ __forceinline__ void turn(const Params &p, const float2 *tab, int lane, float (&x)[K][2 * V]) {
  const int pairs = p.half / V;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int u = lane + k * p.lanes;
    if (u < pairs) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 cs = tab[u * V + i];
        const int m = p.interleaved ? 1 : 0;
        // both layouts with constant register indices
        const float a0 = m ? x[k][2 * i] : x[k][i];
        const float b0 = m ? x[k][2 * i + 1] : x[k][V + i];
        const float a1 = a0 * cs.x - b0 * cs.y, b1 = b0 * cs.x + a0 * cs.y;
        if (m) {
          x[k][2 * i] = a1;
          x[k][2 * i + 1] = b1;
        } else {
          x[k][i] = a1;
          x[k][V + i] = b1;
        }
      }
    }
  }
}

// (cos, sin) of the block's tokens, and the norm weights, into shared memory.
template <typename T>
__device__ __forceinline__ void fill_tables(const Params &p, i64 token0, int tokens, float2 *tab) {
  for (int i = threadIdx.x; i < tokens * p.half; i += blockDim.x) {
    const int t = i / p.half, j = i - t * p.half;
    const i64 token = token0 + t;
    const i64 b = token / p.tokens;
    const i64 pos = index_at(p.positions, b * p.position_stride[0] + (token - b * p.tokens) * p.position_stride[1],
                             p.index64 & 1);
    double turns = static_cast<double>(pos) * p.inv_freq[j] * 0.15915494309189535;
    turns -= rint(turns);
    float s, c;
    sincospif(static_cast<float>(2.0 * turns), &s, &c);
    tab[i] = make_float2(c * p.amplitude, s * p.amplitude * p.sign);
  }
}

template <typename T>
__device__ __forceinline__ void fill_weights(const Params &p, float *weights, int count) {
  for (int i = threadIdx.x; i < count * p.dim; i += blockDim.x) {
    const int r = i / p.dim, j = i - r * p.dim;
    const Rows &rows = p.rows[r];
    if (rows.flags & TILA_ROWS_NORM)
      weights[i] = (rows.flags & TILA_ROWS_WEIGHT_F32) ? static_cast<const float *>(rows.weight)[j]
                                                       : Elem<T>::get(static_cast<const T *>(rows.weight)[j]);
  }
}

template <int V, int K>
__device__ __forceinline__ float row_sum(const Params &p, const float (&x)[K][2 * V], const float (&y)[K][2 * V]) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) s = fmaf(x[k][i], y[k][i], s);
  for (int m = p.lanes >> 1; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
  return s;
}

// w of the elements that a lane holds (0 behind the row's end).
template <int V, int K>
__device__ __forceinline__ void times_weight(const Params &p, const float *w, float scale, int lane,
                                             float (&x)[K][2 * V]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int u = lane + k * p.lanes;
    if (u < p.units) {
      int first, second;
      unit_at<V>(p, u, first, second);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x[k][i] = x[k][i] * scale * w[first + i];
        if (second < p.dim) x[k][V + i] = x[k][V + i] * scale * w[second + i];
      }
    }
  }
}

// Which row a job of a block is: jobs run over the heads of all tensors of one
// token, then over the tokens.
struct Job {
  int tensor, head;
  int t;          // token within the block
  bool valid;
};

__device__ __forceinline__ Job job_at(const Params &p, int j, int jobs) {
  Job job;
  job.valid = j < jobs;
  j = min(j, jobs - 1);
  job.t = j / p.heads;
  int h = j - job.t * p.heads;
  job.tensor = 0;
  if (h >= p.rows[0].heads) {
    h -= p.rows[0].heads;
    job.tensor = 1;
    if (h >= p.rows[1].heads) {
      h -= p.rows[1].heads;
      job.tensor = 2;
    }
  }
  job.head = h;
  return job;
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(512) rotary_rows_kernel(const __grid_constant__ Params p) {
  extern __shared__ float2 tab[];
  float *weights = reinterpret_cast<float *>(tab + p.tokens_per_block * p.half);
  const i64 token0 = static_cast<i64>(blockIdx.x) * p.tokens_per_block;
  const int tokens = static_cast<int>(min(static_cast<i64>(p.tokens_per_block), p.tokens_all - token0));
  const int jobs = tokens * p.heads;
  const int groups = blockDim.x / p.lanes;
  const int lane = threadIdx.x & (p.lanes - 1);
  const int group = threadIdx.x / p.lanes;

  auto row_of = [&](const Job &job) -> const T * {
    const Rows &r = p.rows[job.tensor];
    const i64 token = token0 + job.t, b = token / p.tokens;
    return static_cast<const T *>(r.src) + b * r.src_stride[0] + (token - b * p.tokens) * r.src_stride[1] +
           job.head * r.src_stride[2];
  };

  Job job = job_at(p, group, jobs);
  Raw<T, V, K> raw;
  load_row<T, V, K>(p, row_of(job), lane, raw);
  fill_tables<T>(p, token0, tokens, tab);
  if (p.any_norm) fill_weights<T>(p, weights, p.num_rows);
  __syncthreads();

  // every warp runs the same number of times: the norm's sum is over its lanes
  for (int first = 0; first < jobs; first += groups) {
    const Job next = job_at(p, group + first + groups, jobs);
    Raw<T, V, K> ahead;
    if (first + groups < jobs) load_row<T, V, K>(p, row_of(next), lane, ahead);
    float x[K][2 * V];
    unpack<T, V, K>(raw, x);
    const Rows &r = p.rows[job.tensor];
    if (p.any_norm) {
      const float ss = row_sum<V, K>(p, x, x);
      if (r.flags & TILA_ROWS_NORM)
        times_weight<V, K>(p, weights + job.tensor * p.dim, rsqrtf(ss * p.inv_dim + p.eps), lane, x);
    }
    if (r.flags & TILA_ROWS_ROTATE) turn<V, K>(p, tab + job.t * p.half, lane, x);
    if (job.valid) {
      const i64 token = token0 + job.t;
      T *dst = static_cast<T *>(r.dst) + job.head * r.dst_stride[2];
      if (r.flags & TILA_ROWS_PAGED) {
        const i64 slot = index_at(p.slots, token * p.slot_stride, p.index64 & 2);
        if (slot >= p.num_slots) {
          tila::report_error(p.err, kErrIndex, static_cast<u32>(token));
        } else if (slot >= 0) {
          const i64 page = slot / p.page_size;
          store_row<T, V, K>(p, dst + page * r.dst_stride[0] + (slot - page * p.page_size) * r.dst_stride[1], lane, x);
        }
      } else {
        const i64 b = token / p.tokens;
        store_row<T, V, K>(p, dst + b * r.dst_stride[0] + (token - b * p.tokens) * r.dst_stride[1], lane, x);
      }
    }
    job = next;
    raw = ahead;
  }
}

// Gradients of y = a R (w * x * r), r = 1 / sqrt(mean(x^2) + eps), xh = x * r:
//     g = a R^T dy;   dx = r * (w g - xh * mean(w g xh));   dw = sum over rows of g * xh
// One pass over x and dy.  The blocks are as many as fit the GPU and walk the
// tokens, so that each sums its rows' dw in registers and leaves one partial sum;
// the partial sums are added in a fixed order by the kernel below (no atomics:
// the same call gives the same bits).
template <typename T, int V, int K, int R>
__device__ __forceinline__ void backward_tensor(const Params &p, i64 token0, int tokens, const float2 *tab,
                                                const float *w, float (&sum)[K][2 * V]) {
  const Rows &r = p.rows[R];
  const int jobs = tokens * r.heads;
  const int groups = blockDim.x / p.lanes;
  const int lane = threadIdx.x & (p.lanes - 1);
  const int group = threadIdx.x / p.lanes;
  for (int first = 0; first < jobs; first += groups) {
    const bool valid = first + group < jobs;
    const int j = valid ? first + group : 0;
    const int t = j / r.heads, h = j - t * r.heads;
    const i64 token = token0 + t, b = token / p.tokens, at = token - b * p.tokens;
    Raw<T, V, K> rx, rg;
    load_row<T, V, K>(p, static_cast<const T *>(r.src) + b * r.src_stride[0] + at * r.src_stride[1] +
                             h * r.src_stride[2], lane, rx);
    load_row<T, V, K>(p, static_cast<const T *>(r.grad) + b * r.grad_stride[0] + at * r.grad_stride[1] +
                             h * r.grad_stride[2], lane, rg);
    float x[K][2 * V], g[K][2 * V];
    unpack<T, V, K>(rx, x);
    unpack<T, V, K>(rg, g);
    if (r.flags & TILA_ROWS_ROTATE) turn<V, K>(p, tab + t * p.half, lane, g);
    const float rms = rsqrtf(row_sum<V, K>(p, x, x) * p.inv_dim + p.eps);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) {
        x[k][i] *= rms;                                         // xh
        if (valid) sum[k][i] = fmaf(g[k][i], x[k][i], sum[k][i]);
      }
    times_weight<V, K>(p, w, 1.f, lane, g);                     // w g
    const float mean = row_sum<V, K>(p, g, x) * p.inv_dim;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) x[k][i] = rms * (g[k][i] - x[k][i] * mean);
    if (valid)
      store_row<T, V, K>(p, static_cast<T *>(r.dst) + b * r.dst_stride[0] + at * r.dst_stride[1] +
                                h * r.dst_stride[2], lane, x);
  }
}

// Adds the groups' sums of a block and writes them as partial sum (block, R).
template <int V, int K>
__device__ __forceinline__ void block_sum(const Params &p, float *scratch, const float (&sum)[K][2 * V], int tensor) {
  const int groups = blockDim.x / p.lanes;
  const int lane = threadIdx.x & (p.lanes - 1);
  const int group = threadIdx.x / p.lanes;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int u = lane + k * p.lanes;
    if (u < p.units) {
      int first, second;
      unit_at<V>(p, u, first, second);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        scratch[group * p.dim + first + i] = sum[k][i];
        if (second < p.dim) scratch[group * p.dim + second + i] = sum[k][V + i];
      }
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < p.dim; j += blockDim.x) {
    float s = 0.f;
    for (int g = 0; g < groups; ++g) s += scratch[g * p.dim + j];
    p.partial[(static_cast<i64>(blockIdx.x) * 2 + tensor) * p.dim + j] = s;
  }
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(256) rotary_norm_backward_kernel(const __grid_constant__ Params p) {
  extern __shared__ float2 tab[];
  float *weights = reinterpret_cast<float *>(tab + p.tokens_per_block * p.half);
  float *scratch = weights + 2 * p.dim;
  float sum0[K][2 * V], sum1[K][2 * V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) sum0[k][i] = sum1[k][i] = 0.f;
  fill_weights<T>(p, weights, p.num_rows);
  for (i64 token0 = static_cast<i64>(blockIdx.x) * p.tokens_per_block; token0 < p.tokens_all;
       token0 += static_cast<i64>(gridDim.x) * p.tokens_per_block) {
    const int tokens = static_cast<int>(min(static_cast<i64>(p.tokens_per_block), p.tokens_all - token0));
    __syncthreads();
    fill_tables<T>(p, token0, tokens, tab);
    __syncthreads();
    backward_tensor<T, V, K, 0>(p, token0, tokens, tab, weights, sum0);
    if (p.num_rows > 1) backward_tensor<T, V, K, 1>(p, token0, tokens, tab, weights + p.dim, sum1);
  }
  block_sum<V, K>(p, scratch, sum0, 0);
  if (p.num_rows > 1) block_sum<V, K>(p, scratch, sum1, 1);
}

// weight_grad[tensor][j] = sum over blocks of partial[block][tensor][j]: 32
// columns a block, 8 threads a column, each over every eighth block.
__global__ void __launch_bounds__(256) weight_grad_kernel(const float *partial, int blocks, int dim, float *g0,
                                                          float *g1) {
  __shared__ float s[8][33];
  const int c = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + c, tensor = blockIdx.y;
  float a = 0.f;
  if (j < dim)
    for (int b = part; b < blocks; b += 8) a += partial[(static_cast<i64>(b) * 2 + tensor) * dim + j];
  s[part][c] = a;
  __syncthreads();
  if (part == 0 && j < dim) {
    for (int i = 1; i < 8; ++i) a += s[i][c];
    (tensor == 0 ? g0 : g1)[j] = a;
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

constexpr int kBackwardThreads = 256;

bool aligned(u64 address, const int64_t *stride, int v, int size) {
  return address % (static_cast<u64>(v) * size) == 0 && stride[0] % v == 0 && stride[1] % v == 0 && stride[2] % v == 0;
}

// The widest vector that sizes, strides and addresses of the call allow.
int vector_width(const tila_rotary_args &a, bool backward) {
  const int size = a.dtype == TILA_F32 ? 4 : 2;
  for (int v = 16 / size; v > 1; v >>= 1) {
    bool ok = (a.rotary / 2) % v == 0 && a.dim % v == 0;
    for (int i = 0; ok && i < a.num_rows; ++i) {
      const tila_op_rows &r = a.rows[i];
      ok = aligned(r.src, r.src_stride, v, size) && aligned(r.dst, r.dst_stride, v, size) &&
           (!backward || aligned(r.grad, r.grad_stride, v, size));
    }
    if (ok) return v;
  }
  return 1;
}

int check(const tila_rotary_args *a, bool backward, char *log, size_t cap) {
  const char *who = backward ? "tila_rotary_norm_backward" : "tila_rotary_rows";
  if (a == nullptr || a->size != sizeof(tila_rotary_args) || a->reserved != 0)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: args.size is not that of this library's structure", who);
  if (a->dtype < TILA_F32 || a->dtype > TILA_BF16) return fail(TILA_ERR_ARGUMENT, log, cap, "%s: unknown dtype", who);
  if (a->batch < 0 || a->tokens < 0 || a->dim < 1 || a->dim > 512 || a->rotary < 0 || a->rotary > a->dim ||
      a->rotary % 2 != 0)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: dim must be 1 to 512 and rotary an even number up to dim", who);
  if (a->num_rows < 1 || a->num_rows > (backward ? 2 : 3))
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: num_rows out of range", who);
  bool rotates = false, paged = false;
  for (int i = 0; i < a->num_rows; ++i) {
    const tila_op_rows &r = a->rows[i];
    if (r.heads < 0 || r.heads > (1 << 20)) return fail(TILA_ERR_ARGUMENT, log, cap, "%s: heads out of range", who);
    const u64 size = a->dtype == TILA_F32 ? 4 : 2;
    if (a->batch > 0 && a->tokens > 0 && r.heads > 0 &&
        (r.src == 0 || r.dst == 0 || r.src % size != 0 || r.dst % size != 0 || r.grad % size != 0 ||
         (backward && r.grad == 0) || ((r.flags & TILA_ROWS_NORM) && r.weight == 0)))
      return fail(TILA_ERR_ARGUMENT, log, cap, "%s: an address is missing or not aligned to its elements", who);
    if (backward && (!(r.flags & TILA_ROWS_NORM) || (r.flags & TILA_ROWS_PAGED) || a->weight_grad[i] == 0))
      return fail(TILA_ERR_ARGUMENT, log, cap, "%s: rows must be normed and have a weight gradient", who);
    rotates = rotates || (r.flags & TILA_ROWS_ROTATE);
    paged = paged || (r.flags & TILA_ROWS_PAGED);
  }
  const bool any = a->batch > 0 && a->tokens > 0;
  if (any && rotates && a->rotary > 0 && (a->positions == 0 || a->inv_freq == 0))
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: positions and inv_freq are needed to rotate", who);
  if (paged && ((any && a->slots == 0) || a->page_size < 1 || a->num_slots < 0 || a->batch != 1))
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: slots, page_size and batch 1 are needed for paged rows", who);
  return TILA_OK;
}

Params make_params(const tila_rotary_args &a, bool backward, int v) {
  Params p{};
  bool rotates = false;
  for (int i = 0; i < a.num_rows; ++i) {
    const tila_op_rows &r = a.rows[i];
    Rows &o = p.rows[i];
    o.src = reinterpret_cast<const void *>(r.src);
    o.dst = reinterpret_cast<void *>(r.dst);
    o.weight = reinterpret_cast<const void *>(r.weight);
    o.grad = reinterpret_cast<const void *>(r.grad);
    for (int k = 0; k < 3; ++k) {
      o.src_stride[k] = r.src_stride[k];
      o.dst_stride[k] = r.dst_stride[k];
      o.grad_stride[k] = r.grad_stride[k];
    }
    o.heads = r.heads;
    o.flags = r.flags;
    p.heads += r.heads;
    p.any_norm |= (r.flags & TILA_ROWS_NORM) != 0;
    p.any_paged |= (r.flags & TILA_ROWS_PAGED) != 0;
    rotates = rotates || (r.flags & TILA_ROWS_ROTATE);
  }
  p.num_rows = a.num_rows;
  p.tokens_all = a.batch * a.tokens;
  p.tokens = a.tokens;
  p.dim = a.dim;
  p.half = rotates ? a.rotary / 2 : 0;
  p.interleaved = a.interleaved != 0;
  p.sign = (a.inverse != 0) != backward ? -1.f : 1.f;
  p.amplitude = a.amplitude;
  p.eps = a.eps;
  p.inv_dim = 1.f / a.dim;
  p.positions = reinterpret_cast<const void *>(a.positions);
  p.position_stride[0] = a.position_stride[0];
  p.position_stride[1] = a.position_stride[1];
  p.inv_freq = reinterpret_cast<const double *>(a.inv_freq);
  p.slots = reinterpret_cast<const void *>(a.slots);
  p.slot_stride = a.slot_stride;
  p.num_slots = a.num_slots;
  p.page_size = a.page_size;
  p.index64 = a.index64;
  p.err = reinterpret_cast<u32 *>(a.err);
  p.units = p.half / v + (a.dim - 2 * p.half + 2 * v - 1) / (2 * v);
  p.lanes = 1;
  while (p.lanes < p.units && p.lanes < 32) p.lanes <<= 1;
  return p;
}

// Tokens of a block: enough rows for about 256 threads.
int tokens_per_block(const Params &p) {
  const int threads = std::max(1, p.heads) * p.lanes;
  return std::max(1, std::min({32, 256 / threads, 4096 / std::max(1, p.half)}));
}

int backward_blocks(const Params &p) {
  // 4 blocks of 256 threads an SM: two rows of 64 bytes in flight per thread
  const i64 most = (p.tokens_all + p.tokens_per_block - 1) / p.tokens_per_block;
  return static_cast<int>(std::min<i64>(most, 4 * kSms));
}

template <typename T, int V, int K>
int launch_forward(const Params &p, cudaStream_t stream, char *log, size_t cap) {
  const i64 blocks = (p.tokens_all + p.tokens_per_block - 1) / p.tokens_per_block;
  if (blocks > 0x7fffffff) return fail(TILA_ERR_ARGUMENT, log, cap, "tila_rotary_rows: too many tokens for one launch");
  const i64 lanes = static_cast<i64>(p.tokens_per_block) * p.heads * p.lanes;
  const int threads = static_cast<int>(std::min<i64>(512, std::max<i64>(32, (lanes + 31) / 32 * 32)));
  const size_t smem = sizeof(float2) * p.tokens_per_block * p.half + (p.any_norm ? 3 * sizeof(float) * p.dim : 0);
  rotary_rows_kernel<T, V, K><<<static_cast<unsigned>(blocks), threads, smem, stream>>>(p);
  return launch_status(cudaGetLastError(), "tila_rotary_rows", log, cap);
}

template <typename T, int V, int K>
int launch_backward(const Params &p, const tila_rotary_args &a, cudaStream_t stream, char *log, size_t cap) {
  const int blocks = backward_blocks(p);
  const int groups = kBackwardThreads / p.lanes;
  const size_t smem = sizeof(float2) * p.tokens_per_block * p.half + sizeof(float) * p.dim * (2 + groups);
  cudaError_t e = cudaSuccess;
  if (smem > 48 * 1024)
    e = cudaFuncSetAttribute(rotary_norm_backward_kernel<T, V, K>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem));
  if (e != cudaSuccess) return launch_status(e, "tila_rotary_norm_backward", log, cap);
  rotary_norm_backward_kernel<T, V, K><<<blocks, kBackwardThreads, smem, stream>>>(p);
  e = cudaGetLastError();
  if (e == cudaSuccess) {
    weight_grad_kernel<<<dim3((p.dim + 31) / 32, p.num_rows), 256, 0, stream>>>(
        p.partial, blocks, p.dim, reinterpret_cast<float *>(a.weight_grad[0]),
        reinterpret_cast<float *>(a.weight_grad[1]));
    e = cudaGetLastError();
  }
  return launch_status(e, "tila_rotary_norm_backward", log, cap);
}

template <typename T>
int dispatch(const Params &p, const tila_rotary_args &a, int v, bool backward, char *log, size_t cap) {
  const cudaStream_t stream = reinterpret_cast<cudaStream_t>(a.stream);
  const int per_lane = (p.units + p.lanes - 1) / p.lanes;
#define TILA_ROTARY(V, K) \
  return backward ? launch_backward<T, V, K>(p, a, stream, log, cap) : launch_forward<T, V, K>(p, stream, log, cap)
  if constexpr (sizeof(T) == 2) {
    if (v == 8) TILA_ROTARY(8, 1);
  } else {
    if (v == 4 && per_lane == 1) TILA_ROTARY(4, 1);
  }
  if (v == 4) TILA_ROTARY(4, 2);
  if (v == 2) TILA_ROTARY(2, 4);
  TILA_ROTARY(1, 8);
#undef TILA_ROTARY
}

int run(const tila_rotary_args *a, bool backward, char *log, size_t cap) {
  int st = check(a, backward, log, cap);
  if (st != TILA_OK) return st;
  const int v = vector_width(*a, backward);
  Params p = make_params(*a, backward, v);
  const cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
  if (p.tokens_all == 0 || p.heads == 0) {
    // no row: nothing to write, but the weights' gradients are zero
    for (int i = 0; backward && i < a->num_rows; ++i)
      if (cudaMemsetAsync(reinterpret_cast<void *>(a->weight_grad[i]), 0, sizeof(float) * a->dim, stream) != cudaSuccess)
        return fail(TILA_ERR_DRIVER, log, cap, "tila_rotary_norm_backward: clearing a weight gradient failed");
    return TILA_OK;
  }
  p.tokens_per_block = tokens_per_block(p);
  if (backward) {
    if (a->workspace == 0 || a->workspace % 16 != 0 || a->workspace_bytes < tila_rotary_workspace(a))
      return fail(TILA_ERR_ARGUMENT, log, cap, "tila_rotary_norm_backward: workspace is too small or not 16-byte aligned");
    p.partial = reinterpret_cast<float *>(a->workspace);
  }
  if (a->dtype == TILA_F32) return dispatch<float>(p, *a, v, backward, log, cap);
  if (a->dtype == TILA_F16) return dispatch<__half>(p, *a, v, backward, log, cap);
  return dispatch<__nv_bfloat16>(p, *a, v, backward, log, cap);
}

}  // namespace

extern "C" int tila_rotary_rows(const tila_rotary_args *args, char *log, size_t log_cap) {
  return run(args, false, log, log_cap);
}

extern "C" int tila_rotary_norm_backward(const tila_rotary_args *args, char *log, size_t log_cap) {
  return run(args, true, log, log_cap);
}

extern "C" uint64_t tila_rotary_workspace(const tila_rotary_args *a) {
  if (check(a, true, nullptr, 0) != TILA_OK) return 0;
  Params p = make_params(*a, true, vector_width(*a, true));
  if (p.tokens_all == 0 || p.heads == 0) return 0;
  p.tokens_per_block = tokens_per_block(p);
  return static_cast<uint64_t>(backward_blocks(p)) * 2 * a->dim * sizeof(float);
}
