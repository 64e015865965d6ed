// Norm of each query and key head with the rotation by position in the same pass: forward and backward for training, and the form
// that serves, which also puts keys and values into the pages of a cache.
//
//   y = R(pos) (w o x inv),  inv = 1 / sqrt(mean(x^2) + eps)
//   g = R(pos)^T dy,  dw = sum g o xhat,  dx = inv (g o w - xhat mean(g o w o xhat)),  xhat = x inv
//
// Bound by memory: each element is read once and written once, and the backward recomputes inv instead of reading it.  A head's
// row of D elements belongs to a group of D / (2 VEC) lanes (rounded up to a power of two): lane i holds the 16-byte piece i of
// the lower half and piece i of the upper one, so both kinds of pairs -- neighbours, and halves -- lie within a lane, and a row's
// sum is one shuffle reduction.  A group takes up to HEADS heads of one token: their loads are in flight together, and the
// token's cosines and sines are read once for them.
#include <algorithm>

#include "paged_common.cuh"

namespace {

using paged::Batch;

constexpr int THREADS = 256;
// Heads of one token that a group takes at once, forward and backward, and the CTAs per SM that registers are left for.  fp32 rows are four
// elements a piece and gain from more warps (8 x 1024 x 24 heads of 64, forward and backward: 48.1 us with four and two heads and three CTAs,
// 45.6 so); bf16 ones are eight, are bound by the instructions of a piece and spill in fewer registers (2 x 4095 x 40 heads of 128: 91 us,
// with three CTAs 160, with pieces of four 112).
template <typename T> constexpr int HEADS = sizeof(T) == 4 ? 2 : 4;
template <typename T> constexpr int HEADS_BWD = sizeof(T) == 4 ? 1 : 2;
template <typename T> constexpr int CTAS = sizeof(T) == 4 ? 4 : 2;
constexpr int BWD_CTAS = 148 * 4;

template <typename T> struct Piece;   // 16 bytes of a row
template <> struct Piece<float> {
  static constexpr int VEC = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float* x) {
    x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <> struct Piece<__nv_bfloat16> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* x) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// The elements a lane holds of a row: its piece of the lower half, then that of the upper.
template <int VEC> struct Part { float v[2 * VEC]; };

template <typename T>
__device__ __forceinline__ void store_part(T* row, int gl, int half, const Part<Piece<T>::VEC>& x) {
  constexpr int VEC = Piece<T>::VEC;
  reinterpret_cast<uint4*>(row)[gl] = Piece<T>::pack(x.v);
  reinterpret_cast<uint4*>(row + half)[gl] = Piece<T>::pack(x.v + VEC);
}
// fp32 activations into a bf16 page: a lane's four elements of each half are 8 bytes.
__device__ __forceinline__ void store_part(__nv_bfloat16* row, int gl, int half, const Part<4>& x) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.v[4 * h], x.v[4 * h + 1]), b = __floats2bfloat162_rn(x.v[4 * h + 2], x.v[4 * h + 3]);
    reinterpret_cast<uint2*>(row + h * half)[gl] = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
}

// Two elements an instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&d);
}
template <int VEC> __device__ __forceinline__ float2 two(const Part<VEC>& x, int i) { return make_float2(x.v[2 * i], x.v[2 * i + 1]); }
template <int VEC> __device__ __forceinline__ void put(Part<VEC>& x, int i, float2 t) { x.v[2 * i] = t.x; x.v[2 * i + 1] = t.y; }
template <int VEC> __device__ __forceinline__ float dot(const Part<VEC>& a, const Part<VEC>& b) {
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < VEC; ++i) s = fma2(two(a, i), two(b, i), s);
  return s.x + s.y;
}
template <int VEC> __device__ __forceinline__ void times(Part<VEC>& a, const Part<VEC>& b) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) put(a, i, mul2(two(a, i), two(b, i)));
}
template <int VEC> __device__ __forceinline__ void times(Part<VEC>& a, float f) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) put(a, i, mul2(two(a, i), make_float2(f, f)));
}

// Floats of a (D)-vector (a weight) at the places of a lane's part.
template <int VEC>
__device__ __forceinline__ void load_weight(const float* w, int gl, int half, Part<VEC>& x) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 t = mca_ld_f4(w + h * half + gl * VEC + i);
      x.v[h * VEC + i] = t.x; x.v[h * VEC + i + 1] = t.y; x.v[h * VEC + i + 2] = t.z; x.v[h * VEC + i + 3] = t.w;
    }
}

// Cosines (or sines) of a lane's VEC pairs.  HALVES: pair i is (v[i], v[VEC + i]); else (v[2i], v[2i + 1]).
template <int VEC, bool HALVES>
__device__ __forceinline__ void load_angles(const float* row, int gl, int half, float (&c)[VEC]) {
  if constexpr (HALVES) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 t = mca_ld_f4(row + gl * VEC + i);
      c[i] = t.x; c[i + 1] = t.y; c[i + 2] = t.z; c[i + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < VEC / 2; i += 2) {
        const float2 t = mca_ld_f2(row + h * (half / 2) + gl * (VEC / 2) + i);
        c[h * (VEC / 2) + i] = t.x; c[h * (VEC / 2) + i + 1] = t.y;
      }
  }
}
// By the angles (c, s), or back with s negated.
template <int VEC, bool HALVES>
__device__ __forceinline__ void rotate(Part<VEC>& x, const float (&c)[VEC], const float (&s)[VEC]) {
  if constexpr (HALVES) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float2 a = two(x, i), b = two(x, VEC / 2 + i), ci = make_float2(c[2 * i], c[2 * i + 1]), si = make_float2(s[2 * i], s[2 * i + 1]);
      put(x, i, fma2(b, make_float2(-si.x, -si.y), mul2(a, ci)));
      put(x, VEC / 2 + i, fma2(a, si, mul2(b, ci)));
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float x0 = x.v[2 * i], x1 = x.v[2 * i + 1];
      x.v[2 * i] = x0 * c[i] - x1 * s[i];
      x.v[2 * i + 1] = x0 * s[i] + x1 * c[i];
    }
  }
}

template <int G> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct View {
  const char* data;
  int64_t sb, st, sh;   // bytes
};
inline View view(const McaHeads* h, int size) {
  if (!h) return View{nullptr, 0, 0, 0};
  return View{static_cast<const char*>(h->data), h->stride_b * size, h->stride_t * size, h->stride_h * size};
}
__device__ __forceinline__ const char* at(const View& v, int b, int t, int h) { return v.data + b * v.sb + t * v.st + h * v.sh; }

struct RotArgs {
  const float* weight[2];   // of queries and keys, or null
  const float *cos_table, *sin_table;
  int table_len, D, norm;
  float eps;
};

// Quotients by a divisor of the launch, of numerators below 2^31, from its reciprocal scaled to 33 bits (T. Granlund and P. Montgomery,
// "Division by invariant integers using multiplication", PLDI 1994): an integer division is some twenty instructions.
struct Divisor {
  uint32_t mul, shift;
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};
inline Divisor divisor(int d) {
  Divisor r{0, 0};
  while ((1ll << r.shift) < d) ++r.shift;
  r.mul = (uint32_t)(((1ull << 32) * ((1ull << r.shift) - (uint64_t)d)) / (uint64_t)d + 1);
  return r;
}

struct NormArgs {
  RotArgs r;
  View x[2], out[2];        // queries, keys.  Backward: x and dx
  View g[2];                // backward: gradients of the outputs
  const int* positions;
  int* status;
  int B, T, heads[2], ctas_q;
  Divisor by_chunks[2], by_t;
  float* partial;           // backward: (CTAs, D), or null
};

// A position's row of the tables; null: no rotation, or a position that has none (*bad).
__device__ __forceinline__ int64_t angle_row(const RotArgs& r, int pos, bool* bad) {
  *bad = r.cos_table != nullptr && (pos < 0 || pos >= r.table_len);
  return (int64_t)pos * (r.D / 2);
}

template <typename T, int G, bool HALVES>
__global__ void __launch_bounds__(THREADS, CTAS<T>) qk_norm_rope_kernel(const NormArgs p) {
  constexpr int VEC = Piece<T>::VEC;
  constexpr int GROUPS = THREADS / G;
  mca_pdl_launch_dependents();
  mca_pdl_wait();
  const int kind = (int)blockIdx.x >= p.ctas_q;
  const int cta = kind ? blockIdx.x - p.ctas_q : blockIdx.x, ctas = kind ? gridDim.x - p.ctas_q : p.ctas_q;
  const int gl = threadIdx.x % G, grp = threadIdx.x / G;
  const int half = p.r.D / 2;
  const bool in = gl * VEC < half;
  const int heads = p.heads[kind], chunks = mca_ceil_div(heads, HEADS<T>);
  const int64_t units = (int64_t)p.B * p.T * chunks;
  Part<VEC> w;
#pragma unroll
  for (int i = 0; i < 2 * VEC; ++i) w.v[i] = 1.f;
  if (in && p.r.weight[kind] != nullptr) load_weight<VEC>(p.r.weight[kind], gl, half, w);
  const float inv_d = 1.0f / (float)p.r.D;
  for (int64_t u0 = (int64_t)cta * GROUPS; u0 < units; u0 += (int64_t)ctas * GROUPS) {
    const int64_t unit = u0 + grp;
    const bool live = unit < units;
    const uint32_t un = live ? (uint32_t)unit : 0u;
    const uint32_t token = p.by_chunks[kind](un);
    const int h0 = (int)(un - token * chunks) * HEADS<T>;
    const int b = (int)p.by_t(token), t = (int)token - b * p.T;
    const bool mine = live && in;
    const int pos = p.positions != nullptr ? p.positions[token] : t;
    bool bad;   // a position that has no angles: zeros all the way
    const int64_t ar = angle_row(p.r, pos, &bad);
    uint4 raw[HEADS<T>][2];
#pragma unroll
    for (int i = 0; i < HEADS<T>; ++i) {
      raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
      if (mine && !bad && h0 + i < heads) {
        const char* row = at(p.x[kind], b, t, h0 + i);
        raw[i][0] = reinterpret_cast<const uint4*>(row)[gl];
        raw[i][1] = reinterpret_cast<const uint4*>(row + half * sizeof(T))[gl];
      }
    }
    float c[VEC], s[VEC];
    if (p.r.cos_table != nullptr && mine && !bad) {
      load_angles<VEC, HALVES>(p.r.cos_table + ar, gl, half, c);
      load_angles<VEC, HALVES>(p.r.sin_table + ar, gl, half, s);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) { c[i] = 1.f; s[i] = 0.f; }
      if (bad && live && gl == 0 && h0 == 0 && kind == 0) paged::refuse(p.status, paged::REFUSED_POSITION, (int)token, pos);
    }
#pragma unroll
    for (int i = 0; i < HEADS<T>; ++i) {
      Part<VEC> x;
      Piece<T>::unpack(raw[i][0], x.v);
      Piece<T>::unpack(raw[i][1], x.v + VEC);
      if (p.r.norm) {
        const float inv = rsqrtf(group_sum<G>(dot(x, x)) * inv_d + p.r.eps);
        times(x, bad ? 0.f : inv);
        times(x, w);
      }
      if (p.r.cos_table != nullptr) rotate<VEC, HALVES>(x, c, s);
      if (mine && h0 + i < heads) store_part<T>(reinterpret_cast<T*>(const_cast<char*>(at(p.out[kind], b, t, h0 + i))), gl, half, x);
    }
  }
}

template <typename T, int G, bool HALVES>
__global__ void __launch_bounds__(THREADS, CTAS<T>) qk_norm_rope_bwd_kernel(const NormArgs p) {
  constexpr int VEC = Piece<T>::VEC;
  constexpr int GROUPS = THREADS / G;
  __shared__ float s_dw[GROUPS * G * 2 * VEC];
  mca_pdl_launch_dependents();
  mca_pdl_wait();
  const int kind = (int)blockIdx.x >= p.ctas_q;
  const int cta = kind ? blockIdx.x - p.ctas_q : blockIdx.x, ctas = kind ? gridDim.x - p.ctas_q : p.ctas_q;
  const int gl = threadIdx.x % G, grp = threadIdx.x / G;
  const int half = p.r.D / 2;
  const bool in = gl * VEC < half;
  const int heads = p.heads[kind], chunks = mca_ceil_div(heads, HEADS_BWD<T>);
  const int64_t units = (int64_t)p.B * p.T * chunks;
  Part<VEC> w, dw;
#pragma unroll
  for (int i = 0; i < 2 * VEC; ++i) { w.v[i] = 1.f; dw.v[i] = 0.f; }
  if (in && p.r.weight[kind] != nullptr) load_weight<VEC>(p.r.weight[kind], gl, half, w);
  const float inv_d = 1.0f / (float)p.r.D;
  for (int64_t u0 = (int64_t)cta * GROUPS; u0 < units; u0 += (int64_t)ctas * GROUPS) {
    const int64_t unit = u0 + grp;
    const bool live = unit < units;
    const uint32_t un = live ? (uint32_t)unit : 0u;
    const uint32_t token = p.by_chunks[kind](un);
    const int h0 = (int)(un - token * chunks) * HEADS_BWD<T>;
    const int b = (int)p.by_t(token), t = (int)token - b * p.T;
    const bool mine = live && in;
    const int pos = p.positions != nullptr ? p.positions[token] : t;
    bool bad;   // a position that has no angles: the forward's row is a constant zero
    const int64_t ar = angle_row(p.r, pos, &bad);
    uint4 rg[HEADS_BWD<T>][2], rx[HEADS_BWD<T>][2];
#pragma unroll
    for (int i = 0; i < HEADS_BWD<T>; ++i) {
      rx[i][0] = rx[i][1] = rg[i][0] = rg[i][1] = make_uint4(0, 0, 0, 0);
      if (mine && !bad && h0 + i < heads) {
        const char* row = at(p.g[kind], b, t, h0 + i);
        rg[i][0] = reinterpret_cast<const uint4*>(row)[gl];
        rg[i][1] = reinterpret_cast<const uint4*>(row + half * sizeof(T))[gl];
        if (p.r.norm) {
          row = at(p.x[kind], b, t, h0 + i);
          rx[i][0] = reinterpret_cast<const uint4*>(row)[gl];
          rx[i][1] = reinterpret_cast<const uint4*>(row + half * sizeof(T))[gl];
        }
      }
    }
    float c[VEC], s[VEC];
    if (p.r.cos_table != nullptr && mine && !bad) {
      load_angles<VEC, HALVES>(p.r.cos_table + ar, gl, half, c);
      load_angles<VEC, HALVES>(p.r.sin_table + ar, gl, half, s);
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[i] = -s[i];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) { c[i] = 1.f; s[i] = 0.f; }
      if (bad && live && gl == 0 && h0 == 0 && kind == 0) paged::refuse(p.status, paged::REFUSED_POSITION, (int)token, pos);
    }
#pragma unroll
    for (int i = 0; i < HEADS_BWD<T>; ++i) {
      Part<VEC> g;
      Piece<T>::unpack(rg[i][0], g.v);
      Piece<T>::unpack(rg[i][1], g.v + VEC);
      if (p.r.cos_table != nullptr) rotate<VEC, HALVES>(g, c, s);
      if (p.r.norm) {
        Part<VEC> x;
        Piece<T>::unpack(rx[i][0], x.v);
        Piece<T>::unpack(rx[i][1], x.v + VEC);
        float inv = rsqrtf(group_sum<G>(dot(x, x)) * inv_d + p.r.eps);
        if (bad) inv = 0.f;
        times(x, inv);
        // rows that are not there have a zero g (and a finite x, but for eps 0): they add nothing
        if (mine && h0 + i < heads)
#pragma unroll
          for (int j = 0; j < VEC; ++j) put(dw, j, fma2(two(g, j), two(x, j), two(dw, j)));
        times(g, w);
        const float m = -group_sum<G>(dot(g, x)) * inv_d;
#pragma unroll
        for (int j = 0; j < VEC; ++j) put(g, j, fma2(two(x, j), make_float2(m, m), two(g, j)));
        times(g, inv);
      }
      if (mine && h0 + i < heads) store_part<T>(reinterpret_cast<T*>(const_cast<char*>(at(p.out[kind], b, t, h0 + i))), gl, half, g);
    }
  }
  if (p.partial != nullptr) {   // this CTA's part of dw, its groups added in their order
    const int D = p.r.D;
    if (in)
#pragma unroll
      for (int j = 0; j < 2 * VEC; ++j) s_dw[grp * D + (j < VEC ? gl * VEC + j : half + gl * VEC + j - VEC)] = dw.v[j];
    __syncthreads();
    for (int e = threadIdx.x; e < D; e += THREADS) {
      float sum = 0.f;
      for (int k = 0; k < GROUPS; ++k) sum += s_dw[k * D + e];
      p.partial[(int64_t)blockIdx.x * D + e] = sum;
    }
  }
}

// dw of queries (block x 0) and keys (1): the CTAs' parts, 32 columns of a block, in a fixed order.
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const float* partial, int ctas, int ctas_q, int D, float* dwq, float* dwk) {
  __shared__ float s[32][33];
  mca_pdl_launch_dependents();
  mca_pdl_wait();
  float* dw = blockIdx.x ? dwk : dwq;
  if (dw == nullptr) return;
  const int lo = blockIdx.x ? ctas_q : 0, hi = blockIdx.x ? ctas : ctas_q;
  const int col = blockIdx.y * 32 + threadIdx.x;
  float sum = 0.f;
  if (col < D)
#pragma unroll 8
    for (int i = lo + threadIdx.y; i < hi; i += 32) sum += __ldcg(partial + (int64_t)i * D + col);
  s[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && col < D) {
    float t = 0.f;
    for (int i = 0; i < 32; ++i) t += s[i][threadIdx.x];
    dw[col] = t;
  }
}

struct AppendArgs {
  RotArgs r;
  View in[3];               // queries, keys, values: (token, head) rows
  View q_out;
  Batch batch;
  char *k_pages, *v_pages;
  int64_t page_bytes, row_bytes, head_bytes;
  int heads[3], first_cta[4];   // queries, keys and values have CTAs of their own
  Divisor by_chunks[3];
};

template <typename T, typename CT, int G, bool HALVES>
__global__ void __launch_bounds__(THREADS, CTAS<T>) paged_append_kernel(const AppendArgs p) {
  constexpr int VEC = Piece<T>::VEC;
  constexpr int GROUPS = THREADS / G;
  mca_pdl_launch_dependents();
  mca_pdl_wait();
  if ((int)blockIdx.x == p.first_cta[3]) {   // one more CTA looks the sequences over
    for (int b = threadIdx.x; b < p.batch.n_seqs; b += THREADS) {
      const paged::Sequence s = paged::sequence(p.batch, b);
      if (!s.good) paged::refuse(p.batch.status, paged::REFUSED_LENGTHS, b, s.length);
    }
    return;
  }
  const int kind = ((int)blockIdx.x >= p.first_cta[1]) + ((int)blockIdx.x >= p.first_cta[2]);
  const int cta = blockIdx.x - p.first_cta[kind], ctas = p.first_cta[kind + 1] - p.first_cta[kind];
  const int gl = threadIdx.x % G, grp = threadIdx.x / G;
  const int half = p.r.D / 2;
  const bool in = gl * VEC < half;
  const int heads = p.heads[kind], chunks = mca_ceil_div(heads, HEADS<T>);
  const int64_t units = (int64_t)p.batch.n_tokens * chunks;
  Part<VEC> w;
#pragma unroll
  for (int i = 0; i < 2 * VEC; ++i) w.v[i] = 1.f;
  if (in && kind < 2 && p.r.weight[kind] != nullptr) load_weight<VEC>(p.r.weight[kind], gl, half, w);
  const float inv_d = 1.0f / (float)p.r.D;
  const bool norm = p.r.norm && kind < 2, turn = kind < 2 && p.r.cos_table != nullptr;
  for (int64_t u0 = (int64_t)cta * GROUPS; u0 < units; u0 += (int64_t)ctas * GROUPS) {
    const int64_t unit = u0 + grp;
    const bool live = unit < units;
    const uint32_t un = live ? (uint32_t)unit : 0u;
    const int token = (int)p.by_chunks[kind](un);
    const int h0 = (int)(un - (uint32_t)token * chunks) * HEADS<T>;
    const int b = live ? paged::sequence_of(p.batch, token) : -1;
    const bool reporter = gl == 0 && h0 == 0;
    bool mine = b >= 0 && in, zero = false;
    int pos = 0;
    if (b >= 0) {
      const paged::Sequence s = paged::sequence(p.batch, b);
      pos = s.length - s.count + (token - s.start);
      zero = !s.good;
    }
    uint4 raw[HEADS<T>][2];
#pragma unroll
    for (int i = 0; i < HEADS<T>; ++i) {
      raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
      if (mine && !zero && h0 + i < heads) {
        const char* row = at(p.in[kind], 0, token, h0 + i);
        raw[i][0] = reinterpret_cast<const uint4*>(row)[gl];
        raw[i][1] = reinterpret_cast<const uint4*>(row + half * sizeof(T))[gl];
      }
    }
    float c[VEC], s[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) { c[i] = 1.f; s[i] = 0.f; }
    if (turn && mine && !zero) {
      bool bad;
      const int64_t ar = angle_row(p.r, pos, &bad);
      if (!bad) {
        load_angles<VEC, HALVES>(p.r.cos_table + ar, gl, half, c);
        load_angles<VEC, HALVES>(p.r.sin_table + ar, gl, half, s);
      } else {
        zero = true;
        if (reporter && kind == 0) paged::refuse(p.batch.status, paged::REFUSED_POSITION, token, pos);
      }
    }
    char* dst = nullptr;     // the page row of a key or value
    if (kind > 0 && mine && !zero) {
      const int page = p.batch.table[(int64_t)b * p.batch.table_stride + (pos >> p.batch.page_shift)];
      if (p.r.cos_table != nullptr && pos >= p.r.table_len) mine = false;   // its key is refused: neither is stored
      else if (page < 0 || page >= p.batch.n_pages) {
        mine = false;
        if (reporter && kind == 1) paged::refuse(p.batch.status, paged::REFUSED_PAGE, b, page);
      } else {
        dst = (kind == 1 ? p.k_pages : p.v_pages) + page * p.page_bytes + (int64_t)(pos & ((1 << p.batch.page_shift) - 1)) * p.row_bytes;
      }
    }
#pragma unroll
    for (int i = 0; i < HEADS<T>; ++i) {
      Part<VEC> x;
      Piece<T>::unpack(raw[i][0], x.v);
      Piece<T>::unpack(raw[i][1], x.v + VEC);
      if (norm) {
        const float inv = rsqrtf(group_sum<G>(dot(x, x)) * inv_d + p.r.eps);
        times(x, inv);
        times(x, w);
      }
      if (turn) rotate<VEC, HALVES>(x, c, s);   // never of values: 0 x infinity is none of theirs
      if (zero)
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) x.v[j] = 0.f;
      if (mine && h0 + i < heads) {
        if (kind == 0) store_part<T>(reinterpret_cast<T*>(const_cast<char*>(at(p.q_out, 0, token, h0 + i))), gl, half, x);
        else if (dst != nullptr) store_part(reinterpret_cast<CT*>(dst + (h0 + i) * p.head_bytes), gl, half, x);
      }
    }
  }
}

// CTAs of a kind: one for each GROUPS units, up to a share of the machine.
int ctas_for(int64_t units, int groups, int most) { return (int)std::max<int64_t>(1, std::min<int64_t>((units + groups - 1) / groups, most)); }

template <typename T> int group_of(int D) {   // lanes that share a row
  int g = 1;
  while (g * 2 * Piece<T>::VEC < D) g *= 2;
  return g;
}

int check_rotation(const McaQkRotation* r, int D, RotArgs* out) {
  if (!r) return ERROR_PARAM_NULL;
  if ((r->cos_table == nullptr) != (r->sin_table == nullptr)) return ERROR_PARAM_NULL;
  if (r->cos_table && r->table_len <= 0) return ERROR_PARAM_OUT_OF_RANGE;
  if (r->flags & ~(MCA_QK_NORM | MCA_ROPE_HALVES)) return ERROR_PARAM_OUT_OF_RANGE;
  if ((r->flags & MCA_QK_NORM) && !(r->eps >= 0.f)) return ERROR_PARAM_OUT_OF_RANGE;
  if (!(r->flags & MCA_QK_NORM) && (r->q_weight || r->k_weight)) return ERROR_PARAM_OUT_OF_RANGE;
  if (((uintptr_t)r->q_weight | (uintptr_t)r->k_weight | (uintptr_t)r->cos_table | (uintptr_t)r->sin_table) & 15) return ERROR_PARAM_OUT_OF_RANGE;
  out->weight[0] = r->q_weight; out->weight[1] = r->k_weight;
  out->cos_table = r->cos_table; out->sin_table = r->sin_table;
  out->table_len = r->table_len; out->D = D; out->norm = (r->flags & MCA_QK_NORM) != 0; out->eps = r->eps;
  return 0;
}

int check_norm(const McaQkRotation* rotation, const McaHeads* const (&views)[6], int n_views, const int* positions, int dtype, int B, int T,
               int n_heads, int n_kv_heads, int D, NormArgs* a) {
  if (dtype != MCA_DTYPE_F32 && dtype != MCA_DTYPE_BF16) return ERROR_ATTN_UNSUPPORTED_SHAPE;
  if (D < 16 || D > 256 || D % 16) return ERROR_ATTN_UNSUPPORTED_SHAPE;
  int e = check_rotation(rotation, D, &a->r);
  if (e) return e;
  if (B <= 0 || T <= 0 || n_heads <= 0 || n_kv_heads < 0) return ERROR_PARAM_OUT_OF_RANGE;
  if ((int64_t)B * T >= (1ll << 31) || (int64_t)B * T * std::max(n_heads, n_kv_heads) >= (1ll << 31)) return ERROR_PARAM_OUT_OF_RANGE;
  if (rotation->cos_table && !positions && T > rotation->table_len) return ERROR_PARAM_OUT_OF_RANGE;
  if ((uintptr_t)positions & 3) return ERROR_PARAM_OUT_OF_RANGE;
  for (int i = 0; i < n_views; ++i) {
    if (i % 2 == 1 && n_kv_heads == 0) continue;
    if ((e = paged::check_heads(views[i], dtype, true))) return e;
  }
  const int size = dtype == MCA_DTYPE_BF16 ? 2 : 4;
  for (int i = 0; i < 2; ++i) {
    const bool none = i == 1 && n_kv_heads == 0;
    a->x[i] = view(none ? nullptr : views[i], size);
    a->out[i] = view(none ? nullptr : views[n_views - 2 + i], size);
    a->g[i] = n_views == 6 ? view(none ? nullptr : views[2 + i], size) : View{nullptr, 0, 0, 0};
  }
  a->positions = positions; a->B = B; a->T = T; a->heads[0] = n_heads; a->heads[1] = n_kv_heads; a->partial = nullptr;
  a->by_t = divisor(T);
  a->status = nullptr;
  return 0;
}

template <typename T, int G>
int launch_forward(NormArgs& a, bool halves, cudaStream_t st) {
  constexpr int GROUPS = THREADS / G, MOST = 148 * 16;
  const int64_t tokens = (int64_t)a.B * a.T;
  for (int i = 0; i < 2; ++i) a.by_chunks[i] = divisor(std::max(1, mca_ceil_div(a.heads[i], HEADS<T>)));
  a.ctas_q = ctas_for(tokens * mca_ceil_div(a.heads[0], HEADS<T>), GROUPS, MOST);
  const int ctas_k = a.heads[1] ? ctas_for(tokens * mca_ceil_div(a.heads[1], HEADS<T>), GROUPS, MOST) : 0;
  return mca_launch_pdl(halves ? qk_norm_rope_kernel<T, G, true> : qk_norm_rope_kernel<T, G, false>, dim3(a.ctas_q + ctas_k), dim3(THREADS), 0, st, a);
}
template <typename T, int G>
int launch_backward(NormArgs& a, bool halves, float* dwq, float* dwk, cudaStream_t st) {
  constexpr int GROUPS = THREADS / G;
  const int64_t tokens = (int64_t)a.B * a.T;
  const int all = a.heads[0] + a.heads[1];
  // the CTAs are shared between queries and keys by their heads
  const int most_q = a.heads[1] ? std::max(1, std::min(BWD_CTAS - 1, (int)((int64_t)BWD_CTAS * a.heads[0] / all))) : BWD_CTAS;
  for (int i = 0; i < 2; ++i) a.by_chunks[i] = divisor(std::max(1, mca_ceil_div(a.heads[i], HEADS_BWD<T>)));
  a.ctas_q = ctas_for(tokens * mca_ceil_div(a.heads[0], HEADS_BWD<T>), GROUPS, most_q);
  const int ctas_k = a.heads[1] ? ctas_for(tokens * mca_ceil_div(a.heads[1], HEADS_BWD<T>), GROUPS, BWD_CTAS - most_q) : 0;
  int e = mca_launch_pdl(halves ? qk_norm_rope_bwd_kernel<T, G, true> : qk_norm_rope_bwd_kernel<T, G, false>, dim3(a.ctas_q + ctas_k), dim3(THREADS), 0, st, a);
  if (e || a.partial == nullptr) return e;
  return mca_launch_pdl(qk_norm_dw_kernel, dim3(2, mca_ceil_div(a.r.D, 32)), dim3(32, 32), 0, st, (const float*)a.partial, a.ctas_q + ctas_k, a.ctas_q,
                        a.r.D, dwq, dwk);
}
template <typename T, typename CT, int G>
int launch_append(AppendArgs& a, bool halves, cudaStream_t st) {
  constexpr int GROUPS = THREADS / G, MOST = 148 * 16;
  a.first_cta[0] = 0;
  for (int i = 0; i < 3; ++i) a.by_chunks[i] = divisor(mca_ceil_div(a.heads[i], HEADS<T>));
  for (int i = 0; i < 3; ++i)
    a.first_cta[i + 1] = a.first_cta[i] + ctas_for((int64_t)a.batch.n_tokens * mca_ceil_div(a.heads[i], HEADS<T>), GROUPS, MOST);
  return mca_launch_pdl(halves ? paged_append_kernel<T, CT, G, true> : paged_append_kernel<T, CT, G, false>, dim3(a.first_cta[3] + 1), dim3(THREADS), 0, st, a);
}

}  // namespace

int mca_qk_norm_rope_forward(const McaQkRotation* rotation, const McaHeads* q, const McaHeads* k, const int* positions, int dtype, int B,
                             int T, int n_heads, int n_kv_heads, int D, const McaHeads* q_out, const McaHeads* k_out, void* stream) {
  NormArgs a;
  const McaHeads* const views[6] = {q, k, q_out, k_out, nullptr, nullptr};
  int e = check_norm(rotation, views, 4, positions, dtype, B, T, n_heads, n_kv_heads, D, &a);
  if (e) return e;
  if ((e = paged::find_status(&a.status))) return e;
  const bool halves = (rotation->flags & MCA_ROPE_HALVES) != 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == MCA_DTYPE_BF16) {
    switch (group_of<__nv_bfloat16>(D)) {
      case 1: return launch_forward<__nv_bfloat16, 1>(a, halves, st);
      case 2: return launch_forward<__nv_bfloat16, 2>(a, halves, st);
      case 4: return launch_forward<__nv_bfloat16, 4>(a, halves, st);
      case 8: return launch_forward<__nv_bfloat16, 8>(a, halves, st);
      default: return launch_forward<__nv_bfloat16, 16>(a, halves, st);
    }
  }
  switch (group_of<float>(D)) {
    case 2: return launch_forward<float, 2>(a, halves, st);
    case 4: return launch_forward<float, 4>(a, halves, st);
    case 8: return launch_forward<float, 8>(a, halves, st);
    case 16: return launch_forward<float, 16>(a, halves, st);
    default: return launch_forward<float, 32>(a, halves, st);
  }
}

int64_t mca_qk_norm_rope_backward_scratch_floats(int D) { return D < 16 || D > 256 || D % 16 ? -1 : (int64_t)BWD_CTAS * D; }

int mca_qk_norm_rope_backward(const McaQkRotation* rotation, const McaHeads* q, const McaHeads* k, const int* positions,
                              const McaHeads* dq_out, const McaHeads* dk_out, int dtype, int B, int T, int n_heads, int n_kv_heads, int D,
                              const McaHeads* dq, const McaHeads* dk, float* dq_weight, float* dk_weight, float* scratch,
                              int64_t scratch_floats, void* stream) {
  NormArgs a;
  const McaHeads* const views[6] = {q, k, dq_out, dk_out, dq, dk};
  int e = check_norm(rotation, views, 6, positions, dtype, B, T, n_heads, n_kv_heads, D, &a);
  if (e) return e;
  if (dq_weight || dk_weight) {
    if (!(rotation->flags & MCA_QK_NORM) || (dk_weight && n_kv_heads == 0)) return ERROR_PARAM_OUT_OF_RANGE;
    if (!scratch) return ERROR_PARAM_NULL;
    if (scratch_floats < mca_qk_norm_rope_backward_scratch_floats(D)) return ERROR_ATTN_SCRATCH_TOO_SMALL;
    if (((uintptr_t)scratch | (uintptr_t)dq_weight | (uintptr_t)dk_weight) & 3) return ERROR_PARAM_OUT_OF_RANGE;
    a.partial = scratch;
  }
  if ((e = paged::find_status(&a.status))) return e;
  const bool halves = (rotation->flags & MCA_ROPE_HALVES) != 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == MCA_DTYPE_BF16) {
    switch (group_of<__nv_bfloat16>(D)) {
      case 1: return launch_backward<__nv_bfloat16, 1>(a, halves, dq_weight, dk_weight, st);
      case 2: return launch_backward<__nv_bfloat16, 2>(a, halves, dq_weight, dk_weight, st);
      case 4: return launch_backward<__nv_bfloat16, 4>(a, halves, dq_weight, dk_weight, st);
      case 8: return launch_backward<__nv_bfloat16, 8>(a, halves, dq_weight, dk_weight, st);
      default: return launch_backward<__nv_bfloat16, 16>(a, halves, dq_weight, dk_weight, st);
    }
  }
  switch (group_of<float>(D)) {
    case 2: return launch_backward<float, 2>(a, halves, dq_weight, dk_weight, st);
    case 4: return launch_backward<float, 4>(a, halves, dq_weight, dk_weight, st);
    case 8: return launch_backward<float, 8>(a, halves, dq_weight, dk_weight, st);
    case 16: return launch_backward<float, 16>(a, halves, dq_weight, dk_weight, st);
    default: return launch_backward<float, 32>(a, halves, dq_weight, dk_weight, st);
  }
}

int mca_paged_append(const McaPagedCache* cache, const McaPagedBatch* batch, const McaQkRotation* rotation, int dtype, const McaHeads* q,
                     const McaHeads* k, const McaHeads* v, const McaHeads* q_out, void* stream) {
  AppendArgs a;
  int e = paged::check(cache, batch, &a.batch);
  if (e) return e;
  if (dtype != MCA_DTYPE_F32 && dtype != MCA_DTYPE_BF16) return ERROR_ATTN_UNSUPPORTED_SHAPE;
  if (dtype == MCA_DTYPE_BF16 && cache->dtype != MCA_DTYPE_BF16) return ERROR_ATTN_UNSUPPORTED_SHAPE;
  const int D = cache->head_size;
  if ((e = check_rotation(rotation, D, &a.r))) return e;
  if (batch->n_tokens == 0) return 0;
  if ((e = paged::check_heads(q, dtype, false)) || (e = paged::check_heads(k, dtype, false)) ||
      (e = paged::check_heads(v, dtype, false)) || (e = paged::check_heads(q_out, dtype, false)))
    return e;
  if ((int64_t)batch->n_tokens * cache->n_heads >= (1ll << 31)) return ERROR_PARAM_OUT_OF_RANGE;
  if ((e = paged::find_status(&a.batch.status))) return e;
  const int size = dtype == MCA_DTYPE_BF16 ? 2 : 4, csize = cache->dtype == MCA_DTYPE_BF16 ? 2 : 4;
  a.in[0] = view(q, size); a.in[1] = view(k, size); a.in[2] = view(v, size); a.q_out = view(q_out, size);
  a.k_pages = static_cast<char*>(cache->k_pages); a.v_pages = static_cast<char*>(cache->v_pages);
  a.page_bytes = cache->page_stride * csize; a.row_bytes = (int64_t)cache->n_kv_heads * D * csize; a.head_bytes = (int64_t)D * csize;
  a.heads[0] = cache->n_heads; a.heads[1] = a.heads[2] = cache->n_kv_heads;
  const bool halves = (rotation->flags & MCA_ROPE_HALVES) != 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == MCA_DTYPE_BF16) {
    switch (group_of<__nv_bfloat16>(D)) {
      case 2: return launch_append<__nv_bfloat16, __nv_bfloat16, 2>(a, halves, st);
      case 4: return launch_append<__nv_bfloat16, __nv_bfloat16, 4>(a, halves, st);
      default: return launch_append<__nv_bfloat16, __nv_bfloat16, 8>(a, halves, st);
    }
  }
  const int g = group_of<float>(D);
  if (cache->dtype == MCA_DTYPE_BF16) {
    if (g == 4) return launch_append<float, __nv_bfloat16, 4>(a, halves, st);
    if (g == 8) return launch_append<float, __nv_bfloat16, 8>(a, halves, st);
    return launch_append<float, __nv_bfloat16, 16>(a, halves, st);
  }
  if (g == 4) return launch_append<float, float, 4>(a, halves, st);
  if (g == 8) return launch_append<float, float, 8>(a, halves, st);
  return launch_append<float, float, 16>(a, halves, st);
}

int mca_set_fail_words_qk_norm(int* words) { return (int)cudaMemcpyToSymbol(paged::g_fail_words, &words, sizeof(words)); }
