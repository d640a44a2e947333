// Rotary positions over rows of heads, alone, after a norm of each row, and on
// the way into a paged cache; and the gradients of the normed form.
//
// A row x (one head of one token, `dim` elements) becomes
//     y = a * R(p) * n,    n = x  or  n_j = w_j * x_j / sqrt(mean(x^2) + eps)
// where R turns each pair (n_i, n_p) by the angle p * inv_freq_i and leaves the
// elements behind `rotary` as they are.  The angle is reduced to a part of one
// turn in 64 bits (positions in the millions keep 1e-10 of a turn there, where
// 32 bits would lose the angle), and only that part goes through sincospi in 32
// bits, corrected to first order by what its own rounding to 32 bits left (up to 1e-7
// of a sine, which could be that small itself; once for each token and pair, not for
// each head).  All products and sums are 32-bit; a result is rounded once, when it is
// stored.
//
// Bound by memory: a row is read once and written once (with norms, at 16 bits, the
// instructions come close).  A block takes a few tokens with all their heads, of every
// tensor of the call, so that the sines of a token are computed once and shared
// through shared memory, and so few or many that all blocks are whole waves of the
// GPU.  A row is spread over as many lanes as it has units; a unit is the two V-element
// vectors that hold both halves of V pairs, so that neither layout moves data between
// lanes, and V elements are one 16-byte access where sizes, strides and
// addresses allow it.  Where only the rotated part stands in the way (half of it is no
// multiple of V), units are plain pieces of the row and pairs meet in shared memory
// (16384 tokens of 32 heads, f16, 84 MB each way: 20 of 80 elements rotated, 176 us
// with 4-byte accesses, 66 us so, 60 us interleaved; 40 of 80, 95 us with 8-byte
// accesses, 68 and 62 us so).  Rows are taken tensor by tensor, so that pointers, flags and
// weights stay where they are from row to row; a row is loaded one ahead, and no load
// is conditional, so that all of a row's are in flight together.  Arithmetic and
// conversions are on pairs of floats.
//
// Measured (B200): rotate gradient of 4 x 2048 tokens x 32 heads x 128, 32 bits: 46 us,
// 5.8 TB/s; norm_rotate of 8192 tokens x 40 heads x 128, bf16: 33 us, 5.1 TB/s, its
// gradient 57 us; append of 16384 tokens with 32 query and 8 key heads 72 us, 5.6 TB/s.
// Tried and not kept: a warp for each token with sines and weights in registers (norms
// 57 us where this form took 40), and the same with rows through a ring in shared
// memory (norms 41 us, but 107 us for the append and 7 us for 64 tokens).

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
  // of tokens and heads, which fit 32 bits: a row's place is two multiplications
  u32 src_token, src_head, dst_token, dst_head, grad_token, grad_head;
  int heads;
  u32 flags;
};

struct Params {
  Rows rows[3];
  int heads;             // of all tensors
  int num_rows;
  int batch;
  i64 tokens;            // of one batch entry
  i64 blocks_per_batch;
  int dim, half, interleaved;
  int lanes;             // lanes of a row, a power of two
  int units;
  int full;              // every lane has whole units
  int tokens_per_block;
  int across;            // V where pairs meet in shared memory (kAcross), else 0
  int table_units;       // of those, the units that have a part in the table
  int token_table;       // floats of the table for one token
  int row_floats;        // of a row in shared memory
  int table_mask, weight_mask;   // of `mixed`
  int weight_floats;     // of one weight, whole groups of four pieces
  int any_norm, any_paged;
  int apart;             // a block for each tensor: few tokens, where latency counts
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

__device__ __forceinline__ u64 row_at(int t, u32 token, int h, u32 head) {
  return static_cast<u64>(static_cast<u32>(t)) * token + static_cast<u64>(static_cast<u32>(h)) * head;
}

__device__ __forceinline__ i64 index_at(const void *p, i64 i, int wide) {
  return wide ? static_cast<const i64 *>(p)[i] : static_cast<i64>(static_cast<const i32 *>(p)[i]);
}

// A lane's units: where their two vectors lie in a row, and which there are.  A lane
// without a unit, or a unit without a second vector, has another one's place.
template <int V, int K> struct Units {
  int first[K], second[K];
  bool there[K], both[K], turns[K];
  __device__ __forceinline__ Units(const Params &p, int lane) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int u = lane + k * p.lanes, pairs = p.across ? 0 : p.half / V;   // units that rotate by themselves
      there[k] = u < p.units;
      turns[k] = u < pairs;
      const int at = there[k] ? u : 0;
      if (at < pairs && !p.interleaved) {
        first[k] = at * V;
        second[k] = p.half + at * V;
      } else {
        first[k] = 2 * V * at;                                // also the tail: it starts at 2 * V * pairs
        second[k] = first[k] + V;
      }
      both[k] = there[k] && second[k] < p.dim;
      if (second[k] >= p.dim) second[k] = first[k];
    }
  }
};

template <typename T, int V, int K>
struct Raw { Vec<T, V> a[K], b[K]; };

template <typename T, int V, int K>
__device__ __forceinline__ void load_row(const Units<V, K> &u, const T *row, Raw<T, V, K> &r) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    r.a[k] = *reinterpret_cast<const Vec<T, V> *>(row + u.first[k]);
    r.b[k] = *reinterpret_cast<const Vec<T, V> *>(row + u.second[k]);
  }
}

// Asks for a row that will be loaded later: into L2, no registers wait for it.  The
// gradient's two rows of 16 warps a multiprocessor are too few bytes in flight (59.5 ->
// 57.4 us); the forward kernel's 32 warps have enough and would lose (append 74 -> 87 us).
template <typename T, int V, int K>
__device__ __forceinline__ void fetch_row(const Units<V, K> &u, const T *row) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    asm volatile("prefetch.global.L2 [%0];" ::"l"(row + u.first[k]));
    asm volatile("prefetch.global.L2 [%0];" ::"l"(row + u.second[k]));
  }
}

// A lane's elements of a row as pairs of floats (two 32-bit operations an
// instruction): element 2 i and 2 i + 1 of the unit's 2 V in pair i.
template <int V, int K> using Lane = u64[K][V];

template <typename T, int V, int K>
__device__ __forceinline__ void unpack(const Params &p, const Units<V, K> &u, const Raw<T, V, K> &r, Lane<V, K> &x) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = 2 * i;
      if constexpr (sizeof(T) == 2 && V > 1) {
        const u32 *words = reinterpret_cast<const u32 *>(e < V ? r.a[k].e : r.b[k].e);
        const float2 f = unpack_pair<T>(words[e % V / 2]);
        x[k][i] = tila::pk2(f.x, f.y);
      } else {
        x[k][i] = tila::pk2(Elem<T>::get(e < V ? r.a[k].e[e % V] : r.b[k].e[e % V]),
                            Elem<T>::get(e + 1 < V ? r.a[k].e[(e + 1) % V] : r.b[k].e[(e + 1) % V]));
      }
    }
  if (p.full) return;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < 2 * V; ++e)
      if (!(e < V ? u.there[k] : u.both[k]))
        x[k][e >> 1] = e & 1 ? tila::pk2(tila::lo2(x[k][e >> 1]), 0.f) : tila::pk2(0.f, tila::hi2(x[k][e >> 1]));
}

template <typename T, int V, int K>
__device__ __forceinline__ void store_row(const Units<V, K> &u, T *row, const Lane<V, K> &x) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    Vec<T, V> a, b;
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) {
      if constexpr (sizeof(T) == 2 && V > 1) {
        if (e & 1) continue;
        u32 *words = reinterpret_cast<u32 *>(e < V ? a.e : b.e);
        words[e % V / 2] = pack_pair<T>(tila::lo2(x[k][e >> 1]), tila::hi2(x[k][e >> 1]));
      } else {
        const float f = e & 1 ? tila::hi2(x[k][e >> 1]) : tila::lo2(x[k][e >> 1]);
        (e < V ? a.e[e % V] : b.e[e % V]) = Elem<T>::put(f);
      }
    }
    if (u.there[k]) *reinterpret_cast<Vec<T, V> *>(row + u.first[k]) = a;
    if (u.both[k]) *reinterpret_cast<Vec<T, V> *>(row + u.second[k]) = b;
  }
}

// Where element e of a table or of weights lies: pieces of 16 bytes change places
// (`mask` of 4: with a neighbour; 12: within four), so that lanes that read every
// second or fourth piece meet different banks.
__host__ __device__ __forceinline__ int mixed(int e, int mask) { return e ^ (e >> 3 & mask); }

// 8 elements a lane are two pieces of the table (fewer are read without a gap); units of
// 4 and 8 are two or four of the weights.  norm_rotate of 8192 tokens 34.5 -> 33.1 us.
__host__ __device__ constexpr int table_mask(int v) { return v == 8 ? 4 : 0; }
__host__ __device__ constexpr int weight_mask(int v) { return v >= 4 ? 12 : 0; }

// V consecutive floats of shared memory (V of them aligned) from element e on.
template <int V, int kMask>
__device__ __forceinline__ void floats_at(const float *p, int e, float (&x)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 f = *reinterpret_cast<const float4 *>(p + mixed(e + i, kMask));
      x[i] = f.x, x[i + 1] = f.y, x[i + 2] = f.z, x[i + 3] = f.w;
    }
  } else if constexpr (V == 2) {
    const float2 f = *reinterpret_cast<const float2 *>(p + mixed(e, kMask));
    x[0] = f.x, x[1] = f.y;
  } else {
    x[0] = p[mixed(e, kMask)];
  }
}

// Turns the pairs of a row; `tab` holds the cosines, then the sines, of the row's
// token, the amplitude in both.
template <int V, int K>
__device__ __forceinline__ void turn(const Params &p, const Units<V, K> &u, const float *tab, int lane, Lane<V, K> &x) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!u.turns[k]) continue;                                // (elements behind `rotary` stay bit for bit)
    float c[V], s[V];
    floats_at<V, table_mask(V)>(tab, (lane + k * p.lanes) * V, c);
    floats_at<V, table_mask(V)>(tab + p.half, (lane + k * p.lanes) * V, s);
    if (V == 1 || p.interleaved) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float a = tila::lo2(x[k][i]), b = tila::hi2(x[k][i]);
        x[k][i] = tila::pk2(a * c[i] - b * s[i], b * c[i] + a * s[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const u64 a = x[k][i], b = x[k][V / 2 + i];
        const u64 cc = tila::pk2(c[2 * i], c[2 * i + 1]), ss = tila::pk2(s[2 * i], s[2 * i + 1]);
        const u64 bs = tila::mul2(b, ss);
        x[k][i] = tila::fma2(a, cc, bs ^ 0x8000000080000000ull);
        x[k][V / 2 + i] = tila::fma2(a, ss, tila::mul2(b, cc));
      }
    }
  }
}

// The same for units that are plain pieces of the row.  Each element meets its
// partner in `row` (a group's own shared memory) or, interleaved, in its own
// register; the table holds two cosines and two signed sines for each two elements.
// Both lie by place in the unit first, then by unit: neighbouring lanes read
// neighbouring words.
template <int V, int K> struct Partners {
  u32 at[K][V];                                               // places in `row`: two of 16 bits
  __device__ __forceinline__ Partners(const Params &p, const Units<V, K> &u) {
    auto place = [&](int e) {
      const int partner = e < p.half ? e + p.half : e < 2 * p.half ? e - p.half : 0;
      return static_cast<u32>(partner % (2 * V) * p.units + partner / (2 * V));
    };
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) at[k][i] = place(u.first[k] + 2 * i) | place(u.first[k] + 2 * i + 1) << 16;
  }
};

template <int V, int K>
__device__ __forceinline__ void turn_across(const Params &p, const Units<V, K> &u, const Partners<V, K> &partners,
                                            const float *tab, float *row, int lane, Lane<V, K> &x) {
  if (!p.interleaved) {
    __syncwarp();                                             // (the row before has been read)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (u.there[k]) {                                     // (all of the unit: it has its places)
          row[2 * i * p.units + lane + k * p.lanes] = tila::lo2(x[k][i]);
          row[(2 * i + 1) * p.units + lane + k * p.lanes] = tila::hi2(x[k][i]);
        }
    __syncwarp();
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (u.there[k] && u.first[k] + 2 * i < 2 * p.half) {
        const ulonglong2 t = *reinterpret_cast<const ulonglong2 *>(tab + 4 * (i * p.table_units + lane + k * p.lanes));
        const u64 other = p.interleaved ? tila::pk2(tila::hi2(x[k][i]), tila::lo2(x[k][i]))
                                        : tila::pk2(row[partners.at[k][i] & 0xffff], row[partners.at[k][i] >> 16]);
        x[k][i] = tila::fma2(x[k][i], t.x, tila::mul2(other, t.y));
      }
}

// Floats of the table: what follows it is 16-byte aligned.
__host__ __device__ __forceinline__ int table_size(const Params &p) {
  return (p.token_table * p.tokens_per_block + 3) & ~3;
}

__device__ __forceinline__ void fill_table(const Params &p, int b, i64 token0, int tokens, float *tab) {
  for (int i = threadIdx.x; i < tokens * p.half; i += blockDim.x) {
    const int t = i / p.half, j = i - t * p.half;
    const i64 pos = index_at(p.positions, b * p.position_stride[0] + (token0 + t) * p.position_stride[1], p.index64 & 1);
    double turns = static_cast<double>(pos) * p.inv_freq[j] * 0.15915494309189535;
    turns -= rint(turns);
    const float angle = static_cast<float>(2.0 * turns);              // of half turns
    const float left = static_cast<float>(2.0 * turns - static_cast<double>(angle)) * 3.14159265f;
    float sine, cosine;
    sincospif(angle, &sine, &cosine);
    const float c = fmaf(-left, sine, cosine) * p.amplitude;
    const float s = fmaf(left, cosine, sine) * p.amplitude * p.sign;
    if (p.across) {
      const int low = p.interleaved ? 2 * j : j, high = p.interleaved ? 2 * j + 1 : j + p.half;
      auto at = [&](int e) {
        return tab + t * p.token_table + 4 * ((e >> 1) % p.across * p.table_units + (e >> 1) / p.across) + (e & 1);
      };
      at(low)[0] = at(high)[0] = c;
      at(low)[2] = -s;
      at(high)[2] = s;
    } else {
      tab[2 * t * p.half + mixed(j, p.table_mask)] = c;
      tab[(2 * t + 1) * p.half + mixed(j, p.table_mask)] = s;
    }
  }
}

template <typename T>
__device__ __forceinline__ void fill_weights(const Params &p, float *weights, int count) {
  for (int i = threadIdx.x; i < count * p.dim; i += blockDim.x) {
    const int r = i / p.dim, j = i - r * p.dim;
    const Rows &rows = p.rows[r];
    if (rows.flags & TILA_ROWS_NORM)
      weights[r * p.weight_floats + mixed(j, p.weight_mask)] = (rows.flags & TILA_ROWS_WEIGHT_F32)
                                                                 ? static_cast<const float *>(rows.weight)[j]
                                                                 : Elem<T>::get(static_cast<const T *>(rows.weight)[j]);
  }
}

// Sum over the row of x * y.
template <int V, int K>
__device__ __forceinline__ float row_sum(const Params &p, const Lane<V, K> &x, const Lane<V, K> &y) {
  u64 pair = 0;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) pair = tila::fma2(x[k][i], y[k][i], pair);
  float s = tila::lo2(pair) + tila::hi2(pair);
#pragma unroll
  for (int m = 16; m > 0; m >>= 1)
    if (m < p.lanes) s += __shfl_xor_sync(0xffffffffu, s, m);
  return s;
}

// Those of x x and x y, whose exchanges run side by side.
template <int V, int K>
__device__ __forceinline__ float2 row_sums(const Params &p, const Lane<V, K> &x, const Lane<V, K> &y) {
  u64 xx = 0, xy = 0;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      xx = tila::fma2(x[k][i], x[k][i], xx);
      xy = tila::fma2(x[k][i], y[k][i], xy);
    }
  float2 s = make_float2(tila::lo2(xx) + tila::hi2(xx), tila::lo2(xy) + tila::hi2(xy));
#pragma unroll
  for (int m = 16; m > 0; m >>= 1)
    if (m < p.lanes) {
      s.x += __shfl_xor_sync(0xffffffffu, s.x, m);
      s.y += __shfl_xor_sync(0xffffffffu, s.y, m);
    }
  return s;
}

// x * w of the elements that a lane holds.
template <int V, int K>
__device__ __forceinline__ void times_weight(const Units<V, K> &u, const float *w, Lane<V, K> &x) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float e[2 * V], f[V];
    floats_at<V, weight_mask(V)>(w, u.first[k], f);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = f[i];
    floats_at<V, weight_mask(V)>(w, u.second[k], f);
#pragma unroll
    for (int i = 0; i < V; ++i) e[V + i] = f[i];
#pragma unroll
    for (int i = 0; i < V; ++i) x[k][i] = tila::mul2(x[k][i], tila::pk2(e[2 * i], e[2 * i + 1]));
  }
}

template <int V, int K> __device__ __forceinline__ void times(float f, Lane<V, K> &x) {
  const u64 ff = tila::pk2(f, f);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) x[k][i] = tila::mul2(x[k][i], ff);
}

// Blocks of 256 threads that run at once on a multiprocessor.
template <typename T, int V> struct Resident {
  static constexpr int kForward = sizeof(T) * V == 16 ? 4 : 2;
  static constexpr int kBackward = 2;
};

template <typename T, int V, int K, bool kAcross>
__global__ void __launch_bounds__(256, Resident<T, V>::kForward)
rotary_rows_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) float tab[];
  i64 *places = reinterpret_cast<i64 *>(tab + table_size(p));       // offsets of each token's slot in the paged tensors
  float *weights = reinterpret_cast<float *>(places + (p.any_paged ? 3 * p.tokens_per_block + 1 : 0) / 2 * 2);
  const u32 block = p.apart ? blockIdx.x / p.num_rows : blockIdx.x;
  const int first_r = p.apart ? blockIdx.x - block * p.num_rows : 0, last_r = p.apart ? first_r + 1 : p.num_rows;
  const u32 b = p.batch == 1 ? 0 : block / static_cast<u32>(p.blocks_per_batch);
  const i64 token0 = static_cast<i64>(block - b * static_cast<u32>(p.blocks_per_batch)) * p.tokens_per_block;
  const int tokens = static_cast<int>(min(static_cast<i64>(p.tokens_per_block), p.tokens - token0));
  const int groups = blockDim.x / p.lanes;
  const int lane = threadIdx.x & (p.lanes - 1), group = threadIdx.x / p.lanes;
  const Units<V, K> units(p, lane);
  const Partners<V, K> partners(p, units);

  // Rows are taken tensor by tensor: its heads of one token, then of the next, one
  // to a group; each group's next row is `groups` on.  A group that has none left
  // reads its last one again.
  int job = 0, t = 0, h = 0, jobs = 0;                       // of the row that is loaded
  const T *base = nullptr;
  Raw<T, V, K> raw;
  auto begin = [&](int r) {                                  // the first row of the first tensor from r on that has any
    for (; r < last_r && p.rows[r].heads == 0; ++r) {}
    if (r < last_r) {
      const Rows &rows = p.rows[r];
      jobs = tokens * rows.heads;
      job = group;
      t = min(job, jobs - 1) / rows.heads;
      h = min(job, jobs - 1) - t * rows.heads;
      base = static_cast<const T *>(rows.src) + b * rows.src_stride[0] + token0 * rows.src_stride[1];
      load_row<T, V, K>(units, base + row_at(t, rows.src_token, h, rows.src_head), raw);
    }
    return r;
  };
  int r = begin(first_r);
  if (!p.apart || (p.rows[first_r].flags & TILA_ROWS_ROTATE)) fill_table(p, b, token0, tokens, tab);
  if (p.any_norm) fill_weights<T>(p, weights, p.num_rows);
  if (p.any_paged)
    for (int i = threadIdx.x; i < tokens; i += blockDim.x) {
      const i64 slot = index_at(p.slots, (token0 + i) * p.slot_stride, p.index64 & 2);
      if (slot >= p.num_slots) tila::report_error(p.err, kErrIndex, static_cast<u32>(token0 + i));
      const bool in = slot >= 0 && slot < p.num_slots;
      const u64 place = in ? slot : 0;
      const u64 page = place >> 32 ? place / p.page_size : static_cast<u32>(place) / static_cast<u32>(p.page_size);
      const i64 row = static_cast<i64>(place - page * p.page_size);
      for (int k = 0; k < p.num_rows; ++k)
        places[3 * i + k] = in ? static_cast<i64>(page) * p.rows[k].dst_stride[0] + row * p.rows[k].dst_stride[1] : -1;
    }
  __syncthreads();

  while (r < last_r) {
    const Rows &rows = p.rows[r];
    const u32 flags = rows.flags;
    const u32 src_token = rows.src_token, src_head = rows.src_head, dst_token = rows.dst_token, dst_head = rows.dst_head;
    const int heads = rows.heads, all = jobs, this_r = r;
    const int dt = groups / heads, dh = groups - dt * heads;
    const float *w = weights + r * p.weight_floats;
    T *dst = static_cast<T *>(rows.dst) + (flags & TILA_ROWS_PAGED ? 0 : b * rows.dst_stride[0] + token0 * rows.dst_stride[1]);
    // every warp runs the same number of times: the norm's sum is over its lanes
    for (int first = 0; first < all; first += groups) {
      const bool valid = job < all;
      const int at = t, head = h;
      Lane<V, K> x;
      unpack<T, V, K>(p, units, raw, x);
      if (first + groups < all) {
        job += groups;
        if (job < all) {
          t += dt;
          h += dh;
          if (h >= heads) {
            h -= heads;
            ++t;
          }
        }
        load_row<T, V, K>(units, base + row_at(t, src_token, h, src_head), raw);
      } else {
        r = begin(this_r + 1);
      }
      if (flags & TILA_ROWS_NORM) {
        times<V, K>(rsqrtf(row_sum<V, K>(p, x, x) * p.inv_dim + p.eps), x);
        times_weight<V, K>(units, w, x);
      }
      if (flags & TILA_ROWS_ROTATE) {
        if constexpr (kAcross)
          turn_across<V, K>(p, units, partners, tab + at * p.token_table,
                            weights + (p.any_norm ? p.num_rows * p.weight_floats : 0) + group * p.row_floats, lane, x);
        else
          turn<V, K>(p, units, tab + 2 * at * p.half, lane, x);
      }
      bool put = valid;
      i64 to;
      if (flags & TILA_ROWS_PAGED) {
        const i64 place = places[3 * at + this_r];
        put = put && place >= 0;
        to = place + static_cast<i64>(row_at(0, 0, head, dst_head));
      } else {
        to = static_cast<i64>(row_at(at, dst_token, head, dst_head));
      }
      if (put) store_row<T, V, K>(units, dst + to, x);
    }
  }
}

// Gradients of y = a R (w * x * r), r = 1 / sqrt(mean(x^2) + eps), xh = x * r:
//     g = a R^T dy;   dx = r * (w g - xh * mean(w g xh));   dw = sum over rows of g * xh
// One pass over x and dy.  The blocks are as many as run at once, each with an
// equal share of the tokens, so that each sums its rows' dw in registers (first of the
// queries, then of the keys) and leaves one partial sum; the partial sums are added in a
// fixed order by the kernel below (no atomics: the same call gives the same bits).
template <typename T, int V, int K, bool kAcross>
__global__ void __launch_bounds__(256, Resident<T, V>::kBackward)
rotary_norm_backward_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) float tab[];
  float *weights = reinterpret_cast<float *>(tab + table_size(p));
  float *scratch = weights + 2 * p.weight_floats;
  const int groups = blockDim.x / p.lanes;
  const int lane = threadIdx.x & (p.lanes - 1), group = threadIdx.x / p.lanes;
  const Units<V, K> units(p, lane);
  const Partners<V, K> partners(p, units);
  tila::grid_dep_release();
  fill_weights<T>(p, weights, p.num_rows);
  const i64 all = p.batch * p.tokens;
  const i64 begin = all * blockIdx.x / gridDim.x, end = all * (blockIdx.x + 1) / gridDim.x;
  for (int tensor = 0; tensor < p.num_rows; ++tensor) {
    const Rows &r = p.rows[tensor];
    Lane<V, K> sum;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) sum[k][i] = 0;
    // pieces of the share that lie in one batch entry and fit the table
    for (i64 from = begin; from < end;) {
      const int b = static_cast<int>(from / p.tokens);
      const i64 token0 = from - b * p.tokens;
      const int tokens = static_cast<int>(min(min(static_cast<i64>(p.tokens_per_block), end - from), p.tokens - token0));
      const int jobs = tokens * r.heads;
      if (jobs == 0) break;
      int job = group, t = min(job, jobs - 1) / r.heads, h = min(job, jobs - 1) - t * r.heads;
      const int dt = groups / r.heads, dh = groups - dt * r.heads;
      const T *src = static_cast<const T *>(r.src) + b * r.src_stride[0] + token0 * r.src_stride[1];
      const T *grad = static_cast<const T *>(r.grad) + b * r.grad_stride[0] + token0 * r.grad_stride[1];
      T *dst = static_cast<T *>(r.dst) + b * r.dst_stride[0] + token0 * r.dst_stride[1];
      Raw<T, V, K> rx, rg;
      auto load = [&] {
        load_row<T, V, K>(units, src + row_at(t, r.src_token, h, r.src_head), rx);
        load_row<T, V, K>(units, grad + row_at(t, r.grad_token, h, r.grad_head), rg);
      };
      load();
      __syncthreads();
      fill_table(p, b, token0, tokens, tab);
      __syncthreads();
      for (int first = 0; first < jobs; first += groups) {
        const bool valid = job < jobs;
        const int at = t, head = h;
        Lane<V, K> x, g;
        unpack<T, V, K>(p, units, rx, x);
        unpack<T, V, K>(p, units, rg, g);
        job += groups;
        if (job < jobs) {                      // (else the same row again, unused)
          t += dt;
          h += dh;
          if (h >= r.heads) {
            h -= r.heads;
            ++t;
          }
        }
        if (first + groups < jobs) load();
        if (job + groups < jobs) {
          const int over = h + dh >= r.heads, at_t = t + dt + over, at_h = h + dh - (over ? r.heads : 0);
          fetch_row<T, V, K>(units, src + row_at(at_t, r.src_token, at_h, r.src_head));
          fetch_row<T, V, K>(units, grad + row_at(at_t, r.grad_token, at_h, r.grad_head));
        }
        if (r.flags & TILA_ROWS_ROTATE) {
          if constexpr (kAcross) turn_across<V, K>(p, units, partners, tab + at * p.token_table, scratch + group * p.row_floats, lane, g);
          else turn<V, K>(p, units, tab + 2 * at * p.half, lane, g);
        }
        Lane<V, K> wg;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) wg[k][i] = g[k][i];
        times_weight<V, K>(units, weights + tensor * p.weight_floats, wg);
        const float2 sums = row_sums<V, K>(p, x, wg);                // of x^2 and w g x, at once
        const float rms = rsqrtf(sums.x * p.inv_dim + p.eps);
        times<V, K>(rms, x);                                        // xh
        if (valid)
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) sum[k][i] = tila::fma2(g[k][i], x[k][i], sum[k][i]);
        const float mean = rms * sums.y * p.inv_dim;
        const u64 minus = tila::pk2(-mean, -mean);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) x[k][i] = tila::fma2(x[k][i], minus, wg[k][i]);
        times<V, K>(rms, x);
        if (valid)
          store_row<T, V, K>(units, dst + row_at(at, r.dst_token, head, r.dst_head), x);
      }
      from += tokens;
    }
    // the groups' sums, then this block's partial sum
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < 2 * V; ++e)
        if (e < V ? units.there[k] : units.both[k])
          scratch[group * p.dim + (e < V ? units.first[k] : units.second[k]) + e % V] =
              e & 1 ? tila::hi2(sum[k][e >> 1]) : tila::lo2(sum[k][e >> 1]);
    __syncthreads();
    for (int j = threadIdx.x; j < p.dim; j += blockDim.x) {
      float s = 0.f;
      for (int g = 0; g < groups; ++g) s += scratch[g * p.dim + j];
      p.partial[(static_cast<i64>(blockIdx.x) * 2 + tensor) * p.dim + j] = s;
    }
  }
}

// weight_grad[tensor][j] = sum over blocks of partial[block][tensor][j]: 32
// columns a block, 32 threads a column, each over every 32nd block.
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float *partial, int blocks, int dim, float *g0,
                                                           float *g1) {
  __shared__ float s[32][33];
  const int c = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int tensor = blockIdx.x & 1, j = (blockIdx.x >> 1) * 32 + c;
  tila::grid_dep_wait();
  float a = 0.f;
  if (j < dim)
#pragma unroll 4
    for (int b = part; b < blocks; b += 32) a += partial[(static_cast<i64>(b) * 2 + tensor) * dim + j];
  s[part][c] = a;
  __syncthreads();
  // column `part` by one warp, its 32 sums pairwise
  a = s[c][part];
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) a += __shfl_xor_sync(0xffffffffu, a, x);
  const int column = (blockIdx.x >> 1) * 32 + part;
  if (c == 0 && column < dim && (tensor == 0 ? g0 : g1) != nullptr) (tensor == 0 ? g0 : g1)[column] = a;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

constexpr int kBackwardThreads = 256;

bool aligned(u64 address, const int64_t *stride, int v, int size) {
  return address % (static_cast<u64>(v) * size) == 0 && stride[0] % v == 0 && stride[1] % v == 0 && stride[2] % v == 0;
}

// The widest vector that sizes, strides and addresses of the call allow; `across`
// where half of the rotated part is no multiple of it.
int vector_width(const tila_rotary_args &a, bool backward, bool &across) {
  const int size = a.dtype == TILA_F32 ? 4 : 2;
  across = false;
  for (int v = 16 / size; v > 1; v >>= 1) {
    bool ok = a.dim % v == 0;
    for (int i = 0; ok && i < a.num_rows; ++i) {
      const tila_op_rows &r = a.rows[i];
      ok = aligned(r.src, r.src_stride, v, size) && aligned(r.dst, r.dst_stride, v, size) &&
           (!backward || aligned(r.grad, r.grad_stride, v, size));
    }
    if (!ok) continue;
    across = (a.rotary / 2) % v != 0 && v == 16 / size;
    if (across || (a.rotary / 2) % v == 0) return v;
  }
  return 1;
}

int check(const tila_rotary_args *a, bool backward, char *log, size_t cap) {
  const char *who = backward ? "tila_rotary_norm_backward" : "tila_rotary_rows";
  if (a == nullptr || a->size != sizeof(tila_rotary_args) || a->reserved != 0)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: args.size is not that of this library's structure", who);
  if (a->dtype < TILA_F32 || a->dtype > TILA_BF16) return fail(TILA_ERR_ARGUMENT, log, cap, "%s: unknown dtype", who);
  if (a->batch < 0 || a->tokens < 0 || a->batch > 0x7fffffff || a->dim < 1 || a->dim > 512 || a->rotary < 0 || a->rotary > a->dim ||
      a->rotary % 2 != 0)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: dim must be 1 to 512 and rotary an even number up to dim", who);
  if (a->batch > 0 && a->tokens > (1ll << 46) / a->batch)     // (times blocks and threads that is still below 2^63)
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: more than 2^46 tokens", who);
  if (a->num_rows < 1 || a->num_rows > (backward ? 2 : 3))
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: num_rows out of range", who);
  bool rotates = false, paged = false;
  for (int i = 0; i < a->num_rows; ++i) {
    const tila_op_rows &r = a->rows[i];
    if (r.heads < 0 || r.heads > (1 << 20)) return fail(TILA_ERR_ARGUMENT, log, cap, "%s: heads out of range", who);
    const u64 size = a->dtype == TILA_F32 ? 4 : 2;
    if (a->batch > 0 && a->tokens > 0 && r.heads > 0 &&
        (r.src == 0 || r.dst == 0 || r.src % size != 0 || r.dst % size != 0 || r.grad % size != 0 ||
         (backward && r.grad == 0) ||
         ((r.flags & TILA_ROWS_NORM) &&
          (r.weight == 0 || r.weight % ((r.flags & TILA_ROWS_WEIGHT_F32) ? 4 : size) != 0))))
      return fail(TILA_ERR_ARGUMENT, log, cap, "%s: an address is missing or not aligned to its elements", who);
    const int64_t *strides[3] = {r.src_stride, r.dst_stride, r.grad_stride};
    for (int k = 0; k < (backward ? 3 : 2); ++k)
      for (int d = 1; d < 3; ++d)
        if (strides[k][d] < 0 || strides[k][d] > 0xffffffffll)
          return fail(TILA_ERR_ARGUMENT, log, cap, "%s: strides of tokens and heads must be below 2^32 elements", who);
    if (backward && (!(r.flags & TILA_ROWS_NORM) || (r.flags & TILA_ROWS_PAGED) || a->weight_grad[i] == 0 ||
                     a->weight_grad[i] % 4 != 0))
      return fail(TILA_ERR_ARGUMENT, log, cap, "%s: rows must be normed and have a weight gradient", who);
    rotates = rotates || (r.flags & TILA_ROWS_ROTATE);
    paged = paged || (r.flags & TILA_ROWS_PAGED);
  }
  const bool any = a->batch > 0 && a->tokens > 0;
  if (a->err % 8 != 0 ||
      (any && ((rotates && (a->positions % ((a->index64 & 1) ? 8 : 4) != 0 || a->inv_freq % 8 != 0)) ||
               (paged && a->slots % ((a->index64 & 2) ? 8 : 4) != 0))))
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: positions, inv_freq, slots or err are not aligned to their elements", who);
  if (any && rotates && a->rotary > 0 && (a->positions == 0 || a->inv_freq == 0))
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: positions and inv_freq are needed to rotate", who);
  if (paged && ((any && a->slots == 0) || a->page_size < 1 || a->num_slots < 0 || a->batch != 1))
    return fail(TILA_ERR_ARGUMENT, log, cap, "%s: slots, page_size and batch 1 are needed for paged rows", who);
  return TILA_OK;
}

Params make_params(const tila_rotary_args &a, bool backward, int v, bool across) {
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
    o.src_token = static_cast<u32>(r.src_stride[1]), o.src_head = static_cast<u32>(r.src_stride[2]);
    o.dst_token = static_cast<u32>(r.dst_stride[1]), o.dst_head = static_cast<u32>(r.dst_stride[2]);
    o.grad_token = static_cast<u32>(r.grad_stride[1]), o.grad_head = static_cast<u32>(r.grad_stride[2]);
    o.heads = r.heads;
    // a tensor without heads has no addresses to be read, its weight's among them
    o.flags = r.heads > 0 ? r.flags : r.flags & ~TILA_ROWS_NORM;
    p.heads += r.heads;
    p.any_norm |= (o.flags & TILA_ROWS_NORM) != 0;
    p.any_paged |= (r.flags & TILA_ROWS_PAGED) != 0;
    rotates = rotates || (r.flags & TILA_ROWS_ROTATE);
  }
  p.num_rows = a.num_rows;
  p.batch = static_cast<int>(a.batch);
  p.tokens = a.tokens;
  // batch entries that lie behind one another are one long entry
  bool flat = a.batch > 1 && (a.positions == 0 || a.position_stride[0] == a.tokens * a.position_stride[1]);
  for (int i = 0; flat && i < a.num_rows; ++i) {
    const tila_op_rows &r = a.rows[i];
    flat = r.src_stride[0] == a.tokens * r.src_stride[1] && r.dst_stride[0] == a.tokens * r.dst_stride[1] &&
           (!backward || r.grad_stride[0] == a.tokens * r.grad_stride[1]);
  }
  if (flat) {
    p.tokens *= p.batch;
    p.batch = 1;
  }
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
  p.across = across ? v : 0;
  p.units = across ? (a.dim + 2 * v - 1) / (2 * v) : p.half / v + (a.dim - 2 * p.half + 2 * v - 1) / (2 * v);
  p.table_units = (p.half + v - 1) / v;
  p.table_mask = table_mask(v);
  p.weight_mask = weight_mask(v);
  p.weight_floats = (a.dim + 15) & ~15;
  p.token_table = across ? 4 * v * p.table_units : 2 * p.half;
  p.lanes = 1;
  while (p.lanes < p.units && p.lanes < 32) p.lanes <<= 1;
  // an odd number of times the lanes: the groups of a warp lie in different banks
  p.row_floats = across ? ((2 * v * p.units + p.lanes - 1) / p.lanes | 1) * p.lanes : 0;
  return p;
}

// Tokens of a block: rows for 256 threads at least; where there are more than
// `resident` blocks a multiprocessor could take, as many as fill whole waves.
int tokens_per_block(const Params &p, int resident) {
  const i64 most = std::min(32, (p.across ? 1024 : 2048) / std::max(1, p.half));
  const i64 rows = 256 / std::max(1, p.heads * p.lanes);
  const i64 wave = static_cast<i64>(resident) * kSms, all = p.batch * p.tokens;
  const i64 waves = (all + wave * most - 1) / (wave * most);
  return static_cast<int>(std::max<i64>(1, std::min<i64>(most, std::max(rows, (all + wave * waves - 1) / (wave * waves)))));
}

int backward_blocks(const Params &p) {
  return static_cast<int>(std::min<i64>(p.batch * p.tokens, 2 * kSms));   // as many as run at once (Resident)
}

template <typename T, int V, int K, bool kAcross>
int launch_forward(Params p, cudaStream_t stream, char *log, size_t cap) {
  p.full = p.dim % (2 * V) == 0 && p.units == p.lanes * K;
  p.tokens_per_block = tokens_per_block(p, Resident<T, V>::kForward);
  p.blocks_per_batch = (p.tokens + p.tokens_per_block - 1) / p.tokens_per_block;
  i64 blocks = p.blocks_per_batch * p.batch;
  p.apart = p.num_rows > 1 && blocks * p.num_rows <= 4 * kSms;
  if (p.apart) blocks *= p.num_rows;
  if (blocks > 0x7fffffff) return fail(TILA_ERR_ARGUMENT, log, cap, "tila_rotary_rows: too many tokens for one launch");
  const i64 lanes = static_cast<i64>(p.tokens_per_block) * p.heads * p.lanes;
  const int threads = static_cast<int>(std::min<i64>(256, (lanes + 31) / 32 * 32));
  const size_t smem = sizeof(float) * table_size(p) +
                      (p.any_paged ? sizeof(i64) * ((3 * p.tokens_per_block + 1) / 2 * 2) : 0) +
                      (p.any_norm ? sizeof(float) * p.num_rows * p.weight_floats : 0) +
                      (kAcross ? sizeof(float) * p.row_floats * (threads / p.lanes) : 0);
  rotary_rows_kernel<T, V, K, kAcross><<<static_cast<unsigned>(blocks), threads, smem, stream>>>(p);
  return launch_status(cudaGetLastError(), "tila_rotary_rows", log, cap);
}

template <typename T, int V, int K, bool kAcross>
int launch_backward(Params p, const tila_rotary_args &a, cudaStream_t stream, char *log, size_t cap) {
  p.full = p.dim % (2 * V) == 0 && p.units == p.lanes * K;
  p.tokens_per_block = std::min(32, (p.across ? 1024 : 2048) / std::max(1, p.half));
  const int blocks = backward_blocks(p);
  const int groups = kBackwardThreads / p.lanes;
  // (at most 44144 bytes whatever the sizes: no more than any kernel may have)
  const size_t smem = sizeof(float) * table_size(p) + sizeof(float) * (2 * p.weight_floats + std::max(p.dim, p.row_floats) * groups) + 16;
  rotary_norm_backward_kernel<T, V, K, kAcross><<<blocks, kBackwardThreads, smem, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess)
    e = launch_kernel(weight_grad_kernel, (p.dim + 31) / 32 * 2, 1024, 0, stream, true,
                      static_cast<const float *>(p.partial), blocks, p.dim, reinterpret_cast<float *>(a.weight_grad[0]),
                      p.num_rows > 1 ? reinterpret_cast<float *>(a.weight_grad[1]) : static_cast<float *>(nullptr));
  return launch_status(e, "tila_rotary_norm_backward", log, cap);
}

template <typename T>
int dispatch(const Params &p, const tila_rotary_args &a, int v, bool backward, char *log, size_t cap) {
  const cudaStream_t stream = reinterpret_cast<cudaStream_t>(a.stream);
  const int per_lane = (p.units + p.lanes - 1) / p.lanes;
#define TILA_ROTARY(V, K, X)                                                     \
  return backward ? launch_backward<T, V, K, X>(p, a, stream, log, cap)           \
                  : launch_forward<T, V, K, X>(p, stream, log, cap)
  if constexpr (sizeof(T) == 2) {
    if (v == 8 && p.across) TILA_ROTARY(8, 1, true);
    if (v == 8) TILA_ROTARY(8, 1, false);
  } else {
    // (one unit a lane where that is enough: 20 of 80 elements, 84 MB each way 70 -> 45 us)
    if (v == 4 && p.across && per_lane == 1) TILA_ROTARY(4, 1, true);
    if (v == 4 && p.across) TILA_ROTARY(4, 2, true);
    if (v == 4 && per_lane == 1) TILA_ROTARY(4, 1, false);
  }
  if (v == 4) TILA_ROTARY(4, 2, false);
  if (v == 2) TILA_ROTARY(2, 4, false);
  TILA_ROTARY(1, 8, false);
#undef TILA_ROTARY
}

int run(const tila_rotary_args *a, bool backward, char *log, size_t cap) {
  int st = check(a, backward, log, cap);
  if (st != TILA_OK) return st;
  bool across;
  const int v = vector_width(*a, backward, across);
  Params p = make_params(*a, backward, v, across);
  const cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
  if (p.batch * p.tokens == 0 || p.heads == 0) {
    // no row: nothing to write, but the weights' gradients are zero
    for (int i = 0; backward && i < a->num_rows; ++i)
      if (cudaMemsetAsync(reinterpret_cast<void *>(a->weight_grad[i]), 0, sizeof(float) * a->dim, stream) != cudaSuccess)
        return fail(TILA_ERR_DRIVER, log, cap, "tila_rotary_norm_backward: clearing a weight gradient failed");
    return TILA_OK;
  }
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
  bool across;
  const int v = vector_width(*a, true, across);
  Params p = make_params(*a, true, v, across);
  if (p.batch * p.tokens == 0 || p.heads == 0) return 0;
  return static_cast<uint64_t>(backward_blocks(p)) * 2 * a->dim * sizeof(float);
}
