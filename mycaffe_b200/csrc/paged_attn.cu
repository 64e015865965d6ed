// Attention of new tokens -- prompts, chunks, single tokens, any mix of them -- over a cache made of pages.
//
//   out_t = sum_j p_tj v_j / sum_j p_tj,  p_tj = exp(scale q_t . k_j - m_t),  j = 0 .. position(t)
//
// in one pass over the keys with the running maximum and sum.  The query heads that share a key/value head are rows of one
// tile (row = token x group + head), so that a page is read once for all of them.  The kernels:
//
//   paged_tc_kernel      bf16 pages: S = Q K^T and O += P V on the tensor cores (tcgen05, TMEM), pages by TMA.
//   paged_simt_kernel    fp32 activations over fp32 pages up to eight rows, four at a time, and over bf16 pages one row: exact fp32 products,
//                        a lane group per cache row.
//   paged_tile_kernel    fp32 pages, more rows: exact fp32 products on tiles in shared memory.
//   paged_join_kernel, paged_simt_join_kernel   results of one row from several CTAs, each with some of the keys, joined by their maxima and sums.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <mutex>
#include <type_traits>

#define MCA_TU_FAIL_FAMILY MCA_FAIL_PAGED
#include "paged_common.cuh"
#include "tc_common.cuh"

namespace {

using paged::Batch;
using paged::Sequence;

constexpr float LOG2E = 1.4426950408889634f;

__device__ __align__(16) int g_status[8];   // the device's own status words (paged_common.cuh)

struct AttnArgs {
  Batch batch;
  const char* q;            // (token, head) rows
  char* out;
  int64_t q_st, q_sh, out_st, out_sh;   // bytes
  const char *k_pages, *v_pages;
  int64_t page_bytes, row_bytes;
  int n_heads, n_kv, group, hs;
  int split_len, nsplit, tiles;
  float scale_log2;         // scale x log2(e): the softmax runs on powers of two
  float* part_acc;          // partial results: fp32 kernel (n_tokens, n_heads, nsplit, hs), tensor-core kernel (ctas, 2, hs / 4, rows_max, 4)
  float* part_ml;           // (n_tokens, n_heads, nsplit, 2) and (ctas, 2, rows_max, 2): reference point (log2), sum
  // tensor-core kernel
  int tile_shift, parts, items;    // log2 of the tokens of a tile; tiles that share a token's group of heads; parts x key/value heads
  int ctas, least_units, warps, rows_max;
  int row_shift;            // the join's: log2 of the rows' threads
  int span, inner;          // CTAs that share the work of `inner` heads: all of both, or ctas / items and one
  int4* meta;               // (ctas, 2): the item that ends in a CTA and began in another: {that CTA or -1, token row, head, rows}, {heads}
};

// Tile -> sequence and its first row; every lane of the warp takes part.  Tiles of a sequence: its rows (new tokens x group) in
// steps of R; a sequence that is refused has none.
__device__ __forceinline__ bool find_tile(const Batch& t, int group, int R, int tile, int* seq, int* row0, Sequence* out) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int s0 = 0; s0 < t.n_seqs; s0 += 32) {
    const int b = s0 + lane;
    Sequence s{0, 0, 0, false};
    if (b < t.n_seqs) s = paged::sequence(t, b);
    const int n = s.good ? (s.count * group + R - 1) / R : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + incl > tile);
    if (past != 0) {
      const int src = __ffs(past) - 1;
      *seq = s0 + src;
      *row0 = (tile - before - __shfl_sync(0xffffffffu, incl - n, src)) * R;
      out->start = __shfl_sync(0xffffffffu, s.start, src);
      out->count = __shfl_sync(0xffffffffu, s.count, src);
      out->length = __shfl_sync(0xffffffffu, s.length, src);
      out->good = true;
      return true;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

// What one CTA more than the work needs does: reports the sequences that are refused and writes zeros over their rows.
template <typename T> __device__ void look_over(const AttnArgs& p) {
  for (int b0 = 0; b0 < p.batch.n_seqs; b0 += blockDim.x) {
    const int mine = b0 + threadIdx.x;
    const bool bad = mine < p.batch.n_seqs && !paged::sequence(p.batch, mine).good;
    if (bad) paged::refuse(p.batch.status, paged::REFUSED_LENGTHS, mine, p.batch.lengths[mine]);
    if (!__syncthreads_or(bad)) continue;
    for (int b = b0; b < min(b0 + (int)blockDim.x, p.batch.n_seqs); ++b) {
      if (paged::sequence(p.batch, b).good) continue;
      const int lo = max(p.batch.starts[b], 0), hi = min(p.batch.starts[b + 1], p.batch.n_tokens);
      const int64_t n = (int64_t)max(hi - lo, 0) * p.n_heads * p.hs;
      for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
        const int e = (int)(i % p.hs), h = (int)(i / p.hs % p.n_heads), t = lo + (int)(i / p.hs / p.n_heads);
        reinterpret_cast<T*>(p.out + t * p.out_st + h * p.out_sh)[e] = T(0.f);
      }
    }
  }
}

// Page of a position, or -1 where it is not held (or no page of the pool: `tell` says who reports that).
__device__ __forceinline__ int page_of(const Batch& t, int seq, int pos, bool tell) {
  const int id = t.table[(int64_t)seq * t.table_stride + (pos >> t.page_shift)];
  if (id >= 0 && id < t.n_pages) return id;
  if (tell && id != -1) paged::refuse(t.status, paged::REFUSED_PAGE, seq, id);
  return -1;
}

// ---------------------------------------------------------------------------------------------------------------------
// fp32 activations: exact fp32 products
// ---------------------------------------------------------------------------------------------------------------------
constexpr int SIMT_THREADS = 256, SIMT_WARPS = SIMT_THREADS / 32;

// Elements of a row one lane holds: a group of HS / EPL lanes (a power of two) covers a row with 16-byte pieces.  (Half as many, so that
// two CTAs of four query rows fit an SM, take twice the shuffles: 16 tokens over 2000 fp32 keys, 32 / 8 heads of 128, 68 us for 61.)
template <typename CT, int HS> struct Lanes {
  static constexpr int VEC = 16 / (int)sizeof(CT);
  static constexpr int EPL = HS % 48 == 0 ? (VEC == 4 ? 12 : 24) : 16;
  static constexpr int G = HS / EPL;
  static constexpr int NV = EPL / VEC;
  static constexpr int STAGES = NV <= 2 ? 6 : (NV == 3 ? 4 : 3);   // row steps in flight: 96 KB a CTA
  static constexpr size_t RING = (size_t)SIMT_WARPS * STAGES * 2 * NV * 32 * 16;
};
template <typename CT> __device__ __forceinline__ void unpack16(const uint4& t, float* x) {
  const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(CT) == 4) {
      x[i] = __uint_as_float(w[i]);
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

template <typename CT, int HS, int R>
__global__ void __launch_bounds__(SIMT_THREADS, R <= 2 ? 2 : 1) paged_simt_kernel(const AttnArgs p) {
  using L = Lanes<CT, HS>;
  constexpr int G = L::G, EPL = L::EPL, NV = L::NV, VEC = L::VEC, STAGES = L::STAGES, RPW = 32 / G;
  __shared__ float s_acc[SIMT_WARPS][R][HS];
  __shared__ float s_ml[SIMT_WARPS][R][2];
  extern __shared__ __align__(16) uint4 ring[];
  mca_pdl_launch_dependents();
  mca_pdl_wait();
  if ((int)blockIdx.x == p.tiles) {
    if (blockIdx.y == 0 && blockIdx.z == 0) look_over<float>(p);
    return;
  }
  int seq, row0;
  Sequence sq;
  if (!find_tile(p.batch, p.group, R, blockIdx.x, &seq, &row0, &sq)) return;
  const int kvh = blockIdx.y, split = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = lane % G, g = lane / G;
  const int rows = min(R, sq.count * p.group - row0);
  const int pos0 = sq.length - sq.count;               // position of the sequence's first new token
  const int r_begin = split * p.split_len;
  const int last = pos0 + (row0 + rows - 1) / p.group;  // the last key any row sees
  if (r_begin > last) return;
  const int r_end = min(last + 1, r_begin + p.split_len);

  float q[R][EPL], m[R], l[R], acc[R][EPL];
  int lim[R];
#pragma unroll
  for (int x = 0; x < R; ++x) {
    const int row = row0 + min(x, rows - 1), t = row / p.group, h = kvh * p.group + row - t * p.group;
    lim[x] = x < rows ? pos0 + t : -1;
    const float* src = reinterpret_cast<const float*>(p.q + (int64_t)(sq.start + t) * p.q_st + h * p.q_sh);
    m[x] = -INFINITY; l[x] = 0.f;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 v = mca_ld_f4(src + (c * G + gl) * VEC + i);
        q[x][c * VEC + i] = v.x * p.scale_log2; q[x][c * VEC + i + 1] = v.y * p.scale_log2;
        q[x][c * VEC + i + 2] = v.z * p.scale_log2; q[x][c * VEC + i + 3] = v.w * p.scale_log2;
      }
#pragma unroll
    for (int i = 0; i < EPL; ++i) acc[x][i] = 0.f;
  }

  // Each lane copies exactly the 16-byte pieces that it consumes itself, so its own wait_group is all the synchronisation.
  uint4* my = ring + (size_t)warp * STAGES * 2 * NV * 32 + lane;
  const uint32_t my_s = (uint32_t)__cvta_generic_to_shared(my);
  const int first = r_begin + warp * RPW + g;
  constexpr int STRIDE = SIMT_WARPS * RPW;
  const int n_steps = (r_end - r_begin - warp * RPW + STRIDE - 1) / STRIDE;   // of the warp; not positive: none
  const int64_t head_off = (int64_t)kvh * HS * sizeof(CT);
  const int in_page = (1 << p.batch.page_shift) - 1;
  unsigned held = 0;   // of the steps in flight, whether this lane's row is there (a shift register, the newest at bit 0)
  auto issue = [&](int t) {
    const int row = first + t * STRIDE;
    int page = -1;
    if (t < n_steps && row < r_end) page = page_of(p.batch, seq, row, gl == 0 && kvh == 0);
    held = held << 1 | (page >= 0 ? 1u : 0u);
    if (page >= 0) {
      const uint32_t dst = my_s + (uint32_t)((t % STAGES) * 2 * NV * 32 * 16);
      const int64_t off = page * p.page_bytes + (int64_t)(row & in_page) * p.row_bytes + head_off + gl * 16;
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        mca_cp_async16(dst + (uint32_t)(c * 32 * 16), p.k_pages + off + c * G * 16);
        mca_cp_async16(dst + (uint32_t)((NV + c) * 32 * 16), p.v_pages + off + c * G * 16);
      }
    }
    mca_cp_async_commit();
  };
#pragma unroll
  for (int t = 0; t < STAGES - 1; ++t) issue(t);
  for (int t = 0; t < n_steps; ++t) {
    issue(t + STAGES - 1);
    mca_cp_async_wait<STAGES - 1>();
    const int row = first + t * STRIDE;
    const bool valid = (held >> (STAGES - 1)) & 1u;
    float kx[EPL], vx[EPL];
    if (valid) {
      const uint4* src = my + (size_t)(t % STAGES) * 2 * NV * 32;
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        unpack16<CT>(src[c * 32], kx + VEC * c);
        unpack16<CT>(src[(NV + c) * 32], vx + VEC * c);
      }
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) kx[i] = vx[i] = 0.f;
    }
#pragma unroll
    for (int x = 0; x < R; ++x) {
      float2 s2 = make_float2(0.f, 0.f);   // two products an instruction
#pragma unroll
      for (int i = 0; i < EPL; i += 2) s2 = tc::ffma2(make_float2(q[x][i], q[x][i + 1]), make_float2(kx[i], kx[i + 1]), s2);
      float s = s2.x + s2.y;
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (valid && row <= lim[x] && s != -INFINITY) {   // a logit of minus infinity weighs nothing, also before the first of another kind
        if (s > m[x]) {   // the running maximum moves (rare once it has settled): rescale what was accumulated
          const float f = tc::fast_exp2(m[x] - s);
          l[x] *= f;
#pragma unroll
          for (int i = 0; i < EPL; ++i) acc[x][i] *= f;
          m[x] = s;
        }
        const float w = tc::fast_exp2(s - m[x]);
        l[x] += w;
#pragma unroll
        for (int i = 0; i < EPL; i += 2) {
          const float2 a = tc::ffma2(make_float2(w, w), make_float2(vx[i], vx[i + 1]), make_float2(acc[x][i], acc[x][i + 1]));
          acc[x][i] = a.x; acc[x][i + 1] = a.y;
        }
      }
    }
  }
  mca_cp_async_wait<0>();

  // join the lane groups of a warp, then the warps of the CTA
#pragma unroll
  for (int x = 0; x < R; ++x) {
    float mx = m[x];
#pragma unroll
    for (int o = G; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float f = m[x] == -INFINITY ? (l[x] == 0.f ? 0.f : 1.f) : tc::fast_exp2(m[x] - mx);
    float sum = l[x] * f;
#pragma unroll
    for (int o = G; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      float a = f == 0.f ? 0.f : acc[x][i] * f;
#pragma unroll
      for (int o = G; o < 32; o <<= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
      if (g == 0) s_acc[warp][x][((i / VEC) * G + gl) * VEC + i % VEC] = a;
    }
    if (lane == 0) { s_ml[warp][x][0] = mx; s_ml[warp][x][1] = sum; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * HS; i += SIMT_THREADS) {
    const int x = i / HS, e = i % HS;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < SIMT_WARPS; ++w) M = fmaxf(M, s_ml[w][x][0]);
    float sum = 0.f, a = 0.f;
#pragma unroll
    for (int w = 0; w < SIMT_WARPS; ++w) {
      const float mw = s_ml[w][x][0];
      const float f = mw == -INFINITY ? (s_ml[w][x][1] == 0.f ? 0.f : 1.f) : tc::fast_exp2(mw - M);
      sum += f == 0.f ? 0.f : s_ml[w][x][1] * f;
      a += f == 0.f ? 0.f : s_acc[w][x][e] * f;
    }
    const int row = row0 + x, t = row / p.group, h = kvh * p.group + row - t * p.group;
    if (p.nsplit == 1) {
      reinterpret_cast<float*>(p.out + (int64_t)(sq.start + t) * p.out_st + h * p.out_sh)[e] = sum == 0.f ? 0.f : a / sum;
    } else {
      const int64_t slot = ((int64_t)(sq.start + t) * p.n_heads + h) * p.nsplit + split;
      p.part_acc[slot * HS + e] = a;
      if (e == 0) { p.part_ml[slot * 2] = M; p.part_ml[slot * 2 + 1] = sum; }
    }
  }
}

// More rows than a lane group's registers hold: tiles of 32 rows x 64 keys in shared memory.  A thread forms 4 x 4 logits, then 4 rows
// x HS / 16 columns of the output; 16 threads share their rows, so the softmax's maxima and sums are shuffles and the output's
// factors are at hand.  Bound by the fp32 pipes (two FMAs an instruction); the keys of the next tile arrive under this one's
// softmax and second product, its values under the next first product, and other CTAs of the SM fill the waits.
// Four prompts of up to 200 tokens over 512 keys, 6 heads of 48: 79 us with four rows a CTA, a lane group a key.
constexpr int TILE_ROWS = 32, TILE_KEYS = 64, TILE_THREADS = 128;
template <int HS> struct TilePlan {
  static constexpr int QP = HS + 4, PP = TILE_ROWS + 4;   // row pitches: 16-byte reads of neighbouring rows fall in different banks
  static constexpr int OFF_K = TILE_ROWS * QP, OFF_V = OFF_K + TILE_KEYS * QP, OFF_P = OFF_V + TILE_KEYS * HS, FLOATS = OFF_P + TILE_KEYS * PP;
  static constexpr size_t BYTES = FLOATS * sizeof(float);
  static constexpr int COLS = HS / 16, VW = COLS % 4 == 0 ? 4 : (COLS % 2 == 0 ? 2 : 1);   // columns of a thread, in pieces of VW, 16 VW apart
};
template <int HS>
__global__ void __launch_bounds__(TILE_THREADS) paged_tile_kernel(const AttnArgs p) {
  using T = TilePlan<HS>;
  extern __shared__ __align__(16) float sm[];
  __shared__ int64_t s_off[2][TILE_KEYS];   // byte offset of each key's row of the head; -1: not there
  float *sq_ = sm, *sk = sm + T::OFF_K, *sv = sm + T::OFF_V, *sp = sm + T::OFF_P;
  mca_pdl_launch_dependents();
  mca_pdl_wait();
  if ((int)blockIdx.x == p.tiles) {
    if (blockIdx.y == 0 && blockIdx.z == 0) look_over<float>(p);
    return;
  }
  int seq, row0;
  Sequence sq;
  if (!find_tile(p.batch, p.group, TILE_ROWS, p.tiles - 1 - (int)blockIdx.x, &seq, &row0, &sq)) return;   // those of a chunk's end see the most keys
  const int kvh = blockIdx.y, split = blockIdx.z, tid = threadIdx.x;
  const int rg = tid >> 4, kg = tid & 15;
  const int rows = min(TILE_ROWS, sq.count * p.group - row0);
  const int pos0 = sq.length - sq.count;
  const int first = pos0 + row0 / p.group, last = pos0 + (row0 + rows - 1) / p.group;   // the last key the first row sees, and any row
  const int r_begin = split * p.split_len;
  if (r_begin > last) return;
  const int r_end = min(last + 1, r_begin + p.split_len);
  const int n = (r_end - r_begin + TILE_KEYS - 1) / TILE_KEYS;
  const int in_page = (1 << p.batch.page_shift) - 1;

  auto look_up = [&](int j) {   // rows of key tile j
    if (tid >= TILE_KEYS || j >= n) return;
    const int key = r_begin + j * TILE_KEYS + tid;
    int64_t off = -1;
    if (key < r_end) {
      const int page = page_of(p.batch, seq, key, kvh == 0);
      if (page >= 0) off = page * p.page_bytes + (int64_t)(key & in_page) * p.row_bytes + (int64_t)kvh * HS * 4;
    }
    s_off[j & 1][tid] = off;
  };
  auto fetch = [&](const char* pages, float* dst, int pitch, int j) {
    if (j < n)
      for (int i = tid; i < TILE_KEYS * (HS / 4); i += TILE_THREADS) {
        const int r = i / (HS / 4), c = i % (HS / 4);
        const int64_t off = s_off[j & 1][r];
        float* at = dst + r * pitch + c * 4;
        if (off >= 0) mca_cp_async16((uint32_t)__cvta_generic_to_shared(at), pages + off + c * 16);
        else *reinterpret_cast<float4*>(at) = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    mca_cp_async_commit();
  };

  look_up(0);
  for (int i = tid; i < TILE_ROWS * (HS / 4); i += TILE_THREADS) {
    const int r = i / (HS / 4), c = i % (HS / 4);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rows) {
      const int row = row0 + r, t = row / p.group, h = kvh * p.group + row - t * p.group;
      v = mca_ld_f4(reinterpret_cast<const float*>(p.q + (int64_t)(sq.start + t) * p.q_st + h * p.q_sh) + c * 4);
      v.x *= p.scale_log2; v.y *= p.scale_log2; v.z *= p.scale_log2; v.w *= p.scale_log2;
    }
    *reinterpret_cast<float4*>(sq_ + r * T::QP + c * 4) = v;
  }
  __syncthreads();
  fetch(p.k_pages, sk, T::QP, 0);
  fetch(p.v_pages, sv, HS, 0);

  int lim[4];
  float m[4], l[4];
  float acc[4][T::COLS];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = rg * 4 + i;
    lim[i] = r < rows ? pos0 + (row0 + r) / p.group : -1;
    m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < T::COLS; ++c) acc[i][c] = 0.f;
  }
  for (int j = 0; j < n; ++j) {
    const int key0 = r_begin + j * TILE_KEYS;
    look_up(j + 1);
    mca_cp_async_wait<1>();      // K(j)
    __syncthreads();
    float2 s2[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) s2[i][k] = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int d = 0; d < HS; d += 4) {
      float4 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(sq_ + (rg * 4 + i) * T::QP + d);
#pragma unroll
      for (int k = 0; k < 4; ++k) b[k] = *reinterpret_cast<const float4*>(sk + (kg + 16 * k) * T::QP + d);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          s2[i][k] = tc::ffma2(make_float2(a[i].x, a[i].y), make_float2(b[k].x, b[k].y), s2[i][k]);
          s2[i][k] = tc::ffma2(make_float2(a[i].z, a[i].w), make_float2(b[k].z, b[k].w), s2[i][k]);
        }
    }
    bool there[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) there[k] = s_off[j & 1][kg + 16 * k] >= 0;
    __syncthreads();
    fetch(p.k_pages, sk, T::QP, j + 1);
    float f[4], pr[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float v = s2[i][k].x + s2[i][k].y;
        pr[i][k] = there[k] && key0 + kg + 16 * k <= lim[i] ? v : -INFINITY;
        mx = fmaxf(mx, pr[i][k]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float m_new = fmaxf(m[i], mx);
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      f[i] = m[i] == -INFINITY ? 0.f : tc::fast_exp2(m[i] - ref);
      m[i] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        pr[i][k] = tc::fast_exp2(pr[i][k] - ref);
        sum += pr[i][k];
      }
      l[i] = fmaf(l[i], f[i], sum);   // this thread's part of the row's sum
#pragma unroll
      for (int c = 0; c < T::COLS; ++c) acc[i][c] *= f[i];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      *reinterpret_cast<float4*>(sp + (kg + 16 * k) * T::PP + rg * 4) = make_float4(pr[0][k], pr[1][k], pr[2][k], pr[3][k]);
    mca_cp_async_wait<1>();      // V(j)
    __syncthreads();
    auto second = [&](auto hidden) {   // hidden: some rows do not see all keys, and 0 x infinity is not 0
#pragma unroll 4
      for (int key = 0; key < TILE_KEYS; ++key) {
        const float4 w = *reinterpret_cast<const float4*>(sp + key * T::PP + rg * 4);
        const float wi[4] = {w.x, w.y, w.z, w.w};
        float v[T::COLS];
#pragma unroll
        for (int c = 0; c < T::COLS / T::VW; ++c) {
          const float* at = sv + key * HS + c * 16 * T::VW + kg * T::VW;
          if constexpr (T::VW == 4) {
            const float4 t = *reinterpret_cast<const float4*>(at);
            v[4 * c] = t.x; v[4 * c + 1] = t.y; v[4 * c + 2] = t.z; v[4 * c + 3] = t.w;
          } else if constexpr (T::VW == 2) {
            const float2 t = *reinterpret_cast<const float2*>(at);
            v[2 * c] = t.x; v[2 * c + 1] = t.y;
          } else {
            v[c] = *at;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (decltype(hidden)::value && key0 + key > lim[i]) continue;
          if constexpr (T::COLS % 2 == 0) {
#pragma unroll
            for (int c = 0; c < T::COLS; c += 2) {
              const float2 t = tc::ffma2(make_float2(wi[i], wi[i]), make_float2(v[c], v[c + 1]), make_float2(acc[i][c], acc[i][c + 1]));
              acc[i][c] = t.x; acc[i][c + 1] = t.y;
            }
          } else {
#pragma unroll
            for (int c = 0; c < T::COLS; ++c) acc[i][c] = fmaf(wi[i], v[c], acc[i][c]);
          }
        }
      }
    };
    if (key0 + TILE_KEYS - 1 > first) second(std::true_type{});
    else second(std::false_type{});
    __syncthreads();
    fetch(p.v_pages, sv, HS, j + 1);
  }
  mca_cp_async_wait<0>();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float sum = l[i];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int r = rg * 4 + i;
    if (r >= rows) continue;
    const int row = row0 + r, t = row / p.group, h = kvh * p.group + row - t * p.group;
    const int64_t slot = ((int64_t)(sq.start + t) * p.n_heads + h) * p.nsplit + split;
    const float inv = p.nsplit > 1 ? 1.f : (sum == 0.f ? 0.f : 1.f / sum);
    float* dst = p.nsplit > 1 ? p.part_acc + slot * HS : reinterpret_cast<float*>(p.out + (int64_t)(sq.start + t) * p.out_st + h * p.out_sh);
#pragma unroll
    for (int c = 0; c < T::COLS; ++c) dst[c / T::VW * 16 * T::VW + kg * T::VW + c % T::VW] = acc[i][c] * inv;
    if (p.nsplit > 1 && kg == 0) {
      p.part_ml[slot * 2] = m[i];
      p.part_ml[slot * 2 + 1] = sum;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Join of the splits: out = sum_s 2^(m_s - M) acc_s / sum_s 2^(m_s - M) l_s.  A warp per (token, head), a lane four elements.
// ---------------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(128) paged_simt_join_kernel(const AttnArgs p) {
  mca_pdl_launch_dependents();
  mca_pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(item / p.n_heads), h = (int)(item - (int64_t)t * p.n_heads);
  if (t >= p.batch.n_tokens) return;
  const int b = paged::sequence_of(p.batch, t);
  if (b < 0) return;
  const Sequence s = paged::sequence(p.batch, b);
  if (!s.good) return;
  const int pos = s.length - s.count + t - s.start;
  const int n = pos / p.split_len + 1;   // splits that have keys of this row
  const int64_t slot = item * p.nsplit;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + slot;
  float M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, ml[i].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float sum = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* acc = reinterpret_cast<const float4*>(p.part_acc + slot * p.hs) + lane;
  const int step = p.hs / 4;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float2 v = ml[i];
    const float f = v.y == 0.f ? 0.f : (v.x == -INFINITY ? 1.f : tc::fast_exp2(v.x - M));
    if (f == 0.f) continue;   // a split with nothing of this row: its sums need not be there
    sum = fmaf(v.y, f, sum);
    if (lane < step) {
      const float4 w = acc[(int64_t)i * step];
      a.x = fmaf(w.x, f, a.x); a.y = fmaf(w.y, f, a.y); a.z = fmaf(w.z, f, a.z); a.w = fmaf(w.w, f, a.w);
    }
  }
  if (lane < step) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    reinterpret_cast<float4*>(p.out + t * p.out_st + h * p.out_sh)[lane] = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// bf16 pages: the tensor-core kernel
// ---------------------------------------------------------------------------------------------------------------------
// Work is counted in units: an item is a tile of query rows of one (sequence, key/value head), its units are the tiles of 128 keys
// that the rows see (and ITEM_UNITS more, for its set-up and end).  The launch's CTAs, as many as the machine holds at once, take
// equal contiguous shares of all units, whatever the lengths are: a CTA ends the item its neighbour began, works whole ones, and
// begins one more.  Where the heads divide the CTAs well, each has as many of them, which walk through the sequences side by side
// with the other heads', whose keys lie in the same rows of a page (64 sequences of up to 4096 keys 119.6 -> 116.1 us, eight prompts of up to
// 1000 tokens 64.5 -> 58.5); else all CTAs share all heads.  An item within one CTA is written out; the parts of the others go to the workspace (at most two a CTA) and
// are joined by paged_join_kernel in the order of the CTAs.
//   warps 0-7   write the query tile, then softmax: a warp reads 16 rows x 128 keys of S in the 16-lane quad layout.  Where no
//               sequence has that many rows the warps behind the last take no part in the key loop.
//   warp 8      walks through the work and puts its parts into a ring for the others; TMA producer: lane i fetches the i-th page of a key tile.  Columns behind the head size, and pages that are not
//               held, lie outside the tensor map and arrive as zeros.
//   warp 9      MMA issuer (an elected lane), owner of the TMEM allocation.
// FEW: no sequence has more rows than a tile, so pages are read once: bound by memory.  One CTA per SM with all its shared
//   memory in K and V stages (192 KB on their way), two S tiles, so that the next product runs under this one's softmax.  64 sequences of
//   up to 4096 keys, 32 / 8 heads of 128: 112 us for 700 MB, 6.2 TB/s (two CTAs of one stage each: 145).
// else: tiles share their keys through L2, and the products bound: two CTAs per SM, one's softmax under the other's products.  2048 tokens
//   over 16384, 32 / 8 heads of 128: 605 us call after call, 0.97 PFLOP/s at 1485 MHz; the tensor pipe is 62 % active, between a tile's S and
//   its P V it waits for the softmax.
// fp32 activations (ACT32) over bf16 pages: a query row q is two bf16 rows of the tile, hi = bf16(q) and lo = bf16(q - hi), 16
// lanes apart, so that one product S = [hi; lo] K^T forms both and the softmax warp adds them (the pages are bf16 as they are: q
// to 2^-16 is all that is rounded); the probabilities go back the same way, [p_hi; p_lo], and the two halves of O are added at the
// end.  64 query rows fill a tile then.
using namespace tc;

constexpr int KEYS = 128;   // of a key tile
// Queries in, sums out: 4500 cycles where a key tile takes 3200.  Eight prompts of 400 to 1000 tokens, with 1, 2, 3 and 4: 16 heads of 64 46.1, 45.0, 45.3,
// 45.7 us, 32 / 8 of 128 112, 98.6, 93.3, 92.5; 32 prompts of 33 to 160, 16 of 64: 26.2, 24.7, 26.1, 25.7; steps of single tokens the same within 3 %.
constexpr int ITEM_UNITS = 2;

template <int HDP, bool FEW> struct TcPlan {   // HDP: 64 or 128, the head size padded
  static constexpr int SUB = HDP / 64;
  static constexpr uint32_t SUB_BYTES = KEYS * 128, TILE_BYTES = SUB * SUB_BYTES;
  static constexpr int STG = FEW ? (HDP == 64 ? 6 : 3) : (HDP == 64 ? 2 : 1);
  static constexpr uint32_t OFF_Q = 0, OFF_K = TILE_BYTES, OFF_V = OFF_K + STG * TILE_BYTES, OFF_BAR = OFF_V + STG * TILE_BYTES;
  static constexpr uint32_t OFF_SEG = OFF_BAR + 384, OFF_RED = OFF_SEG + 256;
  static constexpr uint32_t BYTES = OFF_RED + 2 * 128 * 4 + 1024;   // + alignment slack
  static constexpr int CTAS = FEW ? 1 : 2;                          // per SM
  static constexpr uint32_t TMEM = FEW ? 512 : 256;                 // S tiles, then O
  static constexpr uint32_t O_COL = FEW ? 256 : 128;
  static_assert(FEW ? BYTES + 64 <= 227 * 1024 : 2 * (BYTES + 1024) <= 227 * 1024, "shared memory of an SM");
};
constexpr int SEGMENTS = 4;   // parts of items that the producer is ahead of the others
constexpr int TC_THREADS = 320, TC_WARP_TMA = 8, TC_WARP_MMA = 9;
constexpr float TC_RESCALE = 8.0f;   // the softmax's reference point moves when a row's maximum outgrows it by 2^8

enum TcBar : int {
  TB_Q = 0,      // query tile written
  TB_S = 1,      // [2] S written by the MMA (FEW: two tiles in turn)
  TB_P1 = 3,     // [2] first 64 keys of P written by the softmax warps, then 32, then 32 (FEW: in turn, as the softmax may be one
  TB_P2 = 5,     //     key tile ahead of the products)
  TB_P3 = 7,
  TB_O = 9,      // FEW: P V of a key tile finished
  TB_DONE = 10,  // the item's last product finished
  TB_RED = 11,   // row sums in shared memory
  TB_DRAIN = 12,
  TB_KF = 13,    // [6] each: K, V stages full, empty
  TB_KE = 19,
  TB_VF = 25,
  TB_VE = 31,
  TB_GF = 37,    // [SEGMENTS] each: entries of the segment ring full, empty
  TB_GE = 41,
  TB_COUNT = 45
};

// Sum over the first n tiles of c = 2^shift tokens, from position `pos` on, of the key tiles that each sees: ceil((pos + (i + 1) c) / 128).
// With k = 128 / c tiles to a key tile that is floor((i + d) / k), d = floor((pos + c + 127) / c), whose sums have a closed form.
__device__ __forceinline__ int64_t key_tiles_of(int pos, int shift, int n) {
  const int k = 7 - shift;
  auto below = [&](int64_t x) {   // sum of floor(i / 2^k) over i < x
    const int64_t q = x >> k;
    return (q * (q - 1) << k) / 2 + q * (x - (q << k));
  };
  const int64_t d = ((int64_t)pos + (1 << shift) + KEYS - 1) >> shift;
  return below(d + n) - below(d);
}

// a / b for a >= 0, b > 0: in 32 bits where both fit (a 64-bit division is some hundred instructions of one dependent chain).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// The items in their order (sequences, their tiles of 2^tile_shift tokens, the heads of the CTA's span) and a CTA's share of their units;
// all lanes of the walking warp hold the same.
struct Walk {
  int64_t share, left;      // units of a CTA; of this one's, those still to come
  int64_t item_unit;        // first unit of the current item
  int from;                 // units of the current item that belong to the CTAs before
  int seq, tile, head;      // current item; head: key/value head x parts of its group
  int first_cta, head0;     // of the CTA's span
  int start, count, pos0;   // of its sequence

  __device__ __forceinline__ int tiles(const AttnArgs& p) const { return (count + (1 << p.tile_shift) - 1) >> p.tile_shift; }
  __device__ __forceinline__ int last(const AttnArgs& p) const { return pos0 + min((tile + 1) << p.tile_shift, count) - 1; }   // key any row of the item sees
  __device__ __forceinline__ int key_tiles(const AttnArgs& p) const { return last(p) / KEYS + 1; }
  // units of a sequence's first n tiles, all of them full, for one head
  static __device__ __forceinline__ int64_t units_of(const AttnArgs& p, int pos0, int n) {
    return n <= 0 ? 0 : key_tiles_of(pos0, p.tile_shift, n) + (int64_t)n * ITEM_UNITS;
  }
  static __device__ __forceinline__ int64_t units_of(const AttnArgs& p, const Sequence& s) {
    if (!s.good || s.count == 0) return 0;
    const int full = (s.count - 1) >> p.tile_shift;
    return units_of(p, s.length - s.count, full) + (s.length + KEYS - 1) / KEYS + ITEM_UNITS;
  }
  __device__ __forceinline__ void enter(const AttnArgs& p, int b) {
    const Sequence s = paged::sequence(p.batch, b);
    seq = b; start = s.start; count = s.good ? s.count : 0; pos0 = s.length - s.count;
  }

  __device__ __forceinline__ void begin(const AttnArgs& p, int cta) {
    const int lane = threadIdx.x & 31, n = p.batch.n_seqs;
    const int64_t first = lane < n ? units_of(p, paged::sequence(p.batch, lane)) : 0;
    int64_t total = first;
    for (int b = lane + 32; b < n; b += 32) total += units_of(p, paged::sequence(p.batch, b));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    total *= p.inner;
    share = max(quotient(total + p.span - 1, p.span), (int64_t)p.least_units);
    head0 = p.inner == 1 ? cta / p.span : 0;
    first_cta = head0 * p.span;
    const int64_t lo = (int64_t)(cta - first_cta) * share;
    left = min(total - lo, share);
    item_unit = 0; from = seq = tile = start = count = pos0 = 0; head = head0;
    if (left <= 0) return;
    int64_t before = 0;
    for (int s0 = 0; s0 < n; s0 += 32) {
      const int64_t mine = (s0 == 0 ? first : (s0 + lane < n ? units_of(p, paged::sequence(p.batch, s0 + lane)) : 0)) * p.inner;
      int64_t incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + incl > lo);
      if (past != 0) {
        const int src = __ffs(past) - 1;
        before += __shfl_sync(0xffffffffu, incl - mine, src);
        enter(p, s0 + src);
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    // the last tile that begins at or before the share, 32 candidates at a time
    const int64_t rel = lo - before;
    int a = 0, b = tiles(p);
    while (b - a > 1) {
      const int step = (b - a + 31) / 32, t = a + lane * step;
      const unsigned fits = __ballot_sync(0xffffffffu, t < b && units_of(p, pos0, t) * p.inner <= rel);
      a += (__popc(fits) - 1) * step;
      b = min(b, a + step);
    }
    tile = a;
    const int64_t in = rel - units_of(p, pos0, tile) * p.inner;
    const int units = key_tiles(p) + ITEM_UNITS;
    const int h = (int)quotient(in, units);
    head = head0 + h;
    from = (int)(in - (int64_t)h * units);
    item_unit = lo - from;
  }
  // Key tiles [kt0, kt1) of the current item are this CTA's (there may be none).
  __device__ __forceinline__ void take(const AttnArgs& p, int* kt0, int* kt1) {
    const int units = key_tiles(p) + ITEM_UNITS;
    const int to = (int)min((int64_t)units, from + left);
    *kt0 = max(from - ITEM_UNITS, 0);
    *kt1 = max(to - ITEM_UNITS, 0);
    left -= to - from;
  }
  __device__ __forceinline__ void advance(const AttnArgs& p) {
    item_unit += key_tiles(p) + ITEM_UNITS;
    from = 0;
    if (++head < head0 + p.inner) return;
    head = head0;
    if (++tile < tiles(p)) return;
    tile = 0;
    do {
      if (seq + 1 >= p.batch.n_seqs) { left = 0; return; }   // cannot happen: the shares end with the last item
      enter(p, seq + 1);
    } while (count == 0);
  }
};

// One part of an item.  The producer's warp walks and puts the parts into a ring in shared memory, where the other roles read them
// (the softmax has no registers to hold them: with a walk of its own in each warp a key tile took a quarter longer).
struct __align__(16) Segment {
  int n, k_begin, k_end, last;    // key tiles (0: no more work); keys [k_begin, k_end); the last key any row sees
  int token0, rows, heads, pos;   // first token row; rows; query heads of the part; position of the first token
  int head0, kvh, seq;            // first query head; key/value head; sequence
  int slot;                       // workspace slot of a part; -1: all keys of the item, written out
};
static_assert(sizeof(Segment) * SEGMENTS <= 256, "segment ring");
template <int R> __device__ __forceinline__ Segment segment(const AttnArgs& p, const Walk& w, int kt0, int kt1) {
  Segment g;
  const int part = p.parts > 1 ? w.head % p.parts : 0;
  g.kvh = p.parts > 1 ? w.head / p.parts : w.head;
  g.head0 = g.kvh * p.group + part * R;
  g.heads = min(R, p.group - part * R);
  const int t0 = w.tile << p.tile_shift;
  g.token0 = w.start + t0;
  g.rows = min(1 << p.tile_shift, w.count - t0) * g.heads;
  g.pos = w.pos0 + t0;
  g.seq = w.seq;
  g.last = w.last(p);
  g.n = kt1 - kt0;
  g.k_begin = kt0 * KEYS;
  g.k_end = min(g.last + 1, kt1 * KEYS);
  g.slot = kt0 == 0 && kt1 == w.key_tiles(p) ? -1 : 2 * (int)blockIdx.x + (kt0 == 0 ? 1 : 0);
  return g;
}

// Values of a key tile that not every row may see (rows v0 on): 0 x infinity is not 0.  Behind the last key (z0 on) they become zeros;
// those of the later tokens become zeros where they are not finite, and the rows that do see them get them in the end (add_odd).  The
// work of `threads` threads; were there any of this one's?
template <int HDP> __device__ __forceinline__ bool clear_odd(uint32_t v, int v0, int z0, int thread, int threads) {
  constexpr int CH = HDP / 8, SUB_BYTES = KEYS * 128;
  auto at = [&](int i) { return v + (uint32_t)(((i % CH) >> 3) * SUB_BYTES + i / CH * 128 + (i & 7) * 16); };
  for (int i = max(z0, v0) * CH + thread; i < KEYS * CH; i += threads)
    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at(i)), "r"(0u) : "memory");
  bool any = false;
#pragma unroll 2
  for (int i = v0 * CH + thread; i < min(z0, KEYS) * CH; i += threads) {
    uint32_t w[4];
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at(i)) : "memory");
    // an exponent of all ones carries into the sign's place
    uint32_t odd = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) odd |= (w[k] & 0x7f807f80u) + 0x00800080u;
    if (odd & 0x80008000u) {
      any = true;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t o = ((w[k] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
        if (o & 0x8000u) w[k] &= 0xffff0000u;
        if (o & 0x80000000u) w[k] &= 0xffffu;
      }
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at(i)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  return any;
}
// Adds the values that clear_odd took out, of the later tokens that the row sees (its last key), to `n` columns of what the thread
// has just written: the output (bf16 where T is) or the part's sums, whose pieces of four lie `pitch` floats apart.
template <typename T> __device__ __noinline__ void add_odd(const AttnArgs& p, const Segment& g, int last, int col, int n, T* out, int pitch) {
  for (int key = max(g.k_begin, g.pos + 1); key <= min(last, g.k_end - 1); ++key) {
    const int page = page_of(p.batch, g.seq, key, false);
    if (page < 0) continue;
    const __nv_bfloat16* v = reinterpret_cast<const __nv_bfloat16*>(p.v_pages + page * p.page_bytes + (int64_t)(key & ((1 << p.batch.page_shift) - 1)) * p.row_bytes) +
                             g.kvh * p.hs;
    for (int i = col; i < col + n; ++i) {
      const float x = __bfloat162float(v[i]);
      if (isfinite(x)) continue;
      T* at = out + (int64_t)(i >> 2) * pitch + (i & 3);
      *at = T(float(*at) + x);
    }
  }
}

// Bounded waits.  The words that one which gives up leaves are looked up where that happens: their address in the registers of the softmax
// warps is spilled for others (2048 tokens over 16384, 32 / 8 heads of 128: 661 us for 609).
__shared__ int* s_wait_words;
__device__ __noinline__ bool wait_longer(uint32_t bar, uint32_t parity, int stage, int iter) {
  return mbar_wait_limited(bar, parity, *const_cast<int* volatile*>(&s_wait_words), stage, iter, WAIT_LIMIT_NS);
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, int stage, int iter) {
  return mbar_try_wait(bar, parity) || wait_longer(bar, parity, stage, iter);
}

template <int HDP, bool ACT32, bool FEW>
__global__ void __launch_bounds__(TC_THREADS, (TcPlan<HDP, FEW>::CTAS)) paged_tc_kernel(const __grid_constant__ CUtensorMap map_k,
                                                                                       const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnArgs p) {
  using PL = TcPlan<HDP, FEW>;
  constexpr int STG = PL::STG;
  constexpr int R = ACT32 ? 64 : 128;   // query rows of a tile
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + PL::OFF_BAR + TB_COUNT * 8);
  auto bar = [&](int i) { return smem_base + PL::OFF_BAR + 8u * (uint32_t)i; };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ int s_abort;

  mca_pdl_launch_dependents();
  if ((int)blockIdx.x == p.ctas) {   // one more CTA looks the sequences over
    mca_pdl_wait();
    if constexpr (ACT32) look_over<float>(p);
    else look_over<__nv_bfloat16>(p);
    return;
  }
  if (warp == TC_WARP_MMA) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), PL::TMEM);
    tmem_relinquish();
  }
  if (warp == TC_WARP_TMA && lane == 0) {
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  if (tid == 0) {
    *reinterpret_cast<volatile int*>(smem + PL::OFF_BAR + TB_COUNT * 8 + 8) = 0;
    for (int i = 0; i < TB_COUNT; ++i) {
      const bool by_softmax = (i >= TB_P1 && i < TB_O) || i == TB_RED;
      mbar_init(bar(i), i == TB_Q ? 8u : (by_softmax ? (uint32_t)p.warps : (i >= TB_GE ? 9u : 1u)));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  mca_pdl_wait();   // from here on the results of the kernels before this one are complete and visible
  if (tid == 32) {
    s_wait_words = p.batch.status + paged::WAIT_WORDS;
    s_abort = *reinterpret_cast<volatile int*>(s_wait_words);
    if (p.meta != nullptr) p.meta[2 * blockIdx.x].x = -1;   // no item ends here that another CTA began, unless the producer finds one
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (s_abort != 0) {   // a CTA of this call or, until its words are read, an earlier one gave up (a uniform decision, before any copy or product)
    if (warp == TC_WARP_MMA) tmem_dealloc(tmem_base, PL::TMEM);
    return;
  }
  bool ok = true;
  volatile int* const s_odd = reinterpret_cast<volatile int*>(smem + PL::OFF_BAR + TB_COUNT * 8 + 8);   // the last part that values were taken out of, plus one
  int c = 0;      // key tiles so far: stages and phases go by it
  int item = 0;   // parts of items so far
  Segment* const ring = reinterpret_cast<Segment*>(smem + PL::OFF_SEG);
  auto next_segment = [&](int stage) -> const Segment* {   // for the roles but the producer; null: no more
    ok = __all_sync(0xffffffffu, wait_for(bar(TB_GF + item % SEGMENTS), (uint32_t)((item / SEGMENTS) & 1), stage, item));
    return ok && ring[item % SEGMENTS].n > 0 ? ring + item % SEGMENTS : nullptr;
  };
  auto release_segment = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(TB_GE + item % SEGMENTS));
    ++item;
  };

  if (warp == TC_WARP_TMA) {
    // ------------------------------------------------------------------ producer
    const int shift = p.batch.page_shift;
    const int box_rows = shift >= 7 ? KEYS : 1 << shift;
    const int boxes = KEYS / box_rows;
    int issued_k = 0, issued_v = 0;
    Walk w;
    w.begin(p, blockIdx.x);
    bool more = w.left > 0, first = true;
    while (ok) {
      int kt0 = 0, kt1 = 0;
      Segment g;
      g.n = 0;
      if (more) {
        w.take(p, &kt0, &kt1);
        g = segment<R>(p, w, kt0, kt1);
        if (first && p.meta != nullptr && lane == 0 && g.n > 0 && kt0 > 0 && kt1 == w.key_tiles(p)) {   // what the join needs
          p.meta[2 * blockIdx.x] = make_int4(w.first_cta + (int)quotient(w.item_unit + ITEM_UNITS, w.share), g.token0, g.head0, g.rows);
          p.meta[2 * blockIdx.x + 1] = make_int4(g.heads, 0, 0, 0);
        }
        first = false;
      }
      if (!more || g.n > 0) {
        ok = __all_sync(0xffffffffu, wait_for(bar(TB_GE + item % SEGMENTS), (uint32_t)((item / SEGMENTS) & 1) ^ 1u, 9, item));
        if (!ok) break;
        if (lane == 0) {
          ring[item % SEGMENTS] = g;
          mbar_arrive(bar(TB_GF + item % SEGMENTS));
        }
        ++item;
      }
      if (!more) break;
      auto page_at = [&](int j) {   // this lane's page of key tile j; n_pages: none, zeros arrive
        const int pos = g.k_begin + j * KEYS + lane * box_rows;
        if (lane >= boxes || pos >= g.k_end || j >= g.n) return p.batch.n_pages;
        const int id = p.batch.table[(int64_t)g.seq * p.batch.table_stride + (pos >> shift)];
        return id >= 0 && id < p.batch.n_pages ? id : p.batch.n_pages;
      };
      int page = page_at(0);
      for (int j = 0; j < g.n; ++j, ++c) {
        const int st = c % STG;
        const uint32_t ph = (uint32_t)((c / STG) & 1);
        const int next = page_at(j + 1);
        const int slot = (g.k_begin + j * KEYS + lane * box_rows) & ((1 << shift) - 1);
        ok = __all_sync(0xffffffffu, wait_for(bar(TB_KE + st), ph ^ 1u, 10, c));
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(bar(TB_KF + st), PL::TILE_BYTES);
        __syncwarp();
        if (lane < boxes)
#pragma unroll
          for (int s = 0; s < PL::SUB; ++s)
            tma_load_4d(smem_base + PL::OFF_K + st * PL::TILE_BYTES + s * PL::SUB_BYTES + lane * box_rows * 128, &map_k, bar(TB_KF + st), s * 64, g.kvh, slot, page);
        issued_k = c + 1;
        ok = __all_sync(0xffffffffu, wait_for(bar(TB_VE + st), ph ^ 1u, 11, c));
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(bar(TB_VF + st), PL::TILE_BYTES);
        __syncwarp();
        if (lane < boxes)
#pragma unroll
          for (int s = 0; s < PL::SUB; ++s)
            tma_load_4d(smem_base + PL::OFF_V + st * PL::TILE_BYTES + s * PL::SUB_BYTES + lane * box_rows * 128, &map_v, bar(TB_VF + st), s * 64, g.kvh, slot, page);
        issued_v = c + 1;
        page = next;
      }
      more = w.left > 0;
      if (more) w.advance(p);
    }
    if (!ok) {   // copies in flight get a bounded time to land before the CTA's memory is released
      for (int j = max(0, issued_k - STG); j < issued_k; ++j) wait_for(bar(TB_KF + (j % STG)), (uint32_t)((j / STG) & 1), 13, j);
      for (int j = max(0, issued_v - STG); j < issued_v; ++j) wait_for(bar(TB_VF + (j % STG)), (uint32_t)((j / STG) & 1), 14, j);
    }
  } else if (warp == TC_WARP_MMA) {
    // ------------------------------------------------------------------ MMA issuer, in lock step; one elected lane issues
    const uint32_t leader = elect_one() ? 1u : 0u;
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem_base, 0);
    constexpr uint32_t IDESC_QK = make_idesc_fmt(128, KEYS, 0, 0, 1), IDESC_PV = make_idesc_fmt(128, HDP, 0, 1, 1);
    const uint64_t dq = make_desc(smem_base + PL::OFF_Q, 16, 1024);
    const uint64_t dk0 = make_desc(smem_base + PL::OFF_K, 16, 1024), dv0 = make_desc(smem_base + PL::OFF_V, PL::SUB_BYTES, 1024);
    auto issue_qk = [&](int t) {   // of key tile t (of the CTA's)
      const uint64_t dk = dk0 + (uint64_t)(((t % STG) * PL::TILE_BYTES) >> 4);
      const uint32_t d = tm + (FEW ? (uint32_t)(t & 1) * 128u : 0u);
#pragma unroll
      for (int kk = 0; kk < HDP / 16; ++kk) {
        const uint32_t off = ((uint32_t)(kk >> 2) * PL::SUB_BYTES + (uint32_t)(kk & 3) * 32u) >> 4;
        umma_ss_if<false>(leader, d, dq + off, dk + off, IDESC_QK, kk > 0 ? 1u : 0u);
      }
      umma_commit_if(leader, bar(TB_S + (FEW ? t & 1 : 0)));   // covers every product before it
      umma_commit_if(leader, bar(TB_KE + t % STG));
    };
    auto issue_pv = [&](int t, bool first, int lo, int hi) {   // 16 keys a step
      const uint64_t dv = dv0 + (uint64_t)(((t % STG) * PL::TILE_BYTES) >> 4);
      const uint32_t a = tm + (FEW ? (uint32_t)(t & 1) * 128u : 0u);
#pragma unroll
      for (int kk = lo; kk < hi; ++kk)
        umma_ts_if<false>(leader, tm + PL::O_COL, a + (uint32_t)(kk * 8), dv + (uint64_t)((uint32_t)kk * (2048u >> 4)), IDESC_PV, (first && kk == 0) ? 0u : 1u);
    };
    auto wait = [&](int b, uint32_t ph, int stage) { return __all_sync(0xffffffffu, wait_for(bar(b), ph & 1u, stage, c)); };
    while (const Segment* g = next_segment(19)) {
      const int n = g->n;
      {
        ok = wait(TB_Q, item, 20) && wait(TB_KF + c % STG, c / STG, 21);
        if (!ok) break;
        tc_fence_after();
        issue_qk(c);
        for (int j = 0; j < n; ++j, ++c) {
          if (FEW && j + 1 < n) {
            if (!(ok = wait(TB_KF + (c + 1) % STG, (c + 1) / STG, 25))) break;
            tc_fence_after();
            issue_qk(c + 1);
          }
          if (!(ok = wait(TB_VF + c % STG, c / STG, 22))) break;
          if (!(ok = wait(TB_P1 + (FEW ? c & 1 : 0), FEW ? c >> 1 : c, 28))) break;
          tc_fence_after();
          issue_pv(c, j == 0, 0, 4);
          if (!FEW && j + 1 < n && !(ok = wait(TB_KF + (c + 1) % STG, (c + 1) / STG, 25))) break;
          if (!(ok = wait(TB_P2 + (FEW ? c & 1 : 0), FEW ? c >> 1 : c, 40))) break;
          tc_fence_after();
          issue_pv(c, j == 0, 4, 6);
          if (!(ok = wait(TB_P3 + (FEW ? c & 1 : 0), FEW ? c >> 1 : c, 23))) break;
          tc_fence_after();
          issue_pv(c, j == 0, 6, 8);
          umma_commit_if(leader, bar(TB_VE + c % STG));
          if (FEW) umma_commit_if(leader, bar(TB_O));
          if (j + 1 == n) umma_commit_if(leader, bar(TB_DONE));
          else if (!FEW) issue_qk(c + 1);
        }
      }
      if (!ok) break;
      release_segment();
    }
    umma_commit_if(leader, bar(TB_DRAIN));   // the tensor pipe is idle (bounded) before TMEM is freed
    wait_for(bar(TB_DRAIN), 0, 27, 0);
    __syncwarp();
  } else {
    constexpr int CH = HDP / 8;   // 16-byte pieces of a row
    const int rank = ACT32 ? warp : (warp & 3) * 2 + (warp >> 2);   // the 16 rows of the tile that are this warp's
    const int lane_base = ACT32 ? warp * 32 : rank * 16;
    const int quad = lane & 3;
    const int r0 = rank * 16 + (lane >> 2);
    float* red_l = reinterpret_cast<float*>(smem + PL::OFF_RED);
    float* red_m = red_l + 128;
    const float scale = p.scale_log2;
    const float2 scale2 = make_float2(scale, scale);
    constexpr int QN = R * CH / 256, QV = ACT32 ? 2 : 1;   // pieces of the query tile of a thread: eight elements, QV vectors each
    uint4 raw[QN][QV];
    auto load_query = [&](const Segment& g) {   // all loads go out together
#pragma unroll
      for (int i = 0; i < QN; ++i) {
        const int r = (i * 256 + tid) / CH, ch = tid % CH;
#pragma unroll
        for (int k = 0; k < QV; ++k) raw[i][k] = make_uint4(0, 0, 0, 0);
        if (r < g.rows && ch * 8 < p.hs) {
          const int t = r / g.heads;
          const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t)(g.token0 + t) * p.q_st + (g.head0 + r - t * g.heads) * p.q_sh);
#pragma unroll
          for (int k = 0; k < QV; ++k) raw[i][k] = src[ch * QV + k];
        }
      }
    };
    const Segment* gp = next_segment(18);
    if (FEW && gp != nullptr) load_query(*gp);
    while (gp != nullptr) {
      const Segment& g = *gp;
      const Segment* gn = nullptr;   // the part after it
      {
        // ---------------------------------------------------------------- the query tile, 16-byte pieces in the swizzled layout; rows behind the last are
        // zeros, and so are their logits and what is read as their probabilities: products of zeros take less power, and under the
        // power cap the clock is the time (64 single tokens, 4 rows of 128, call after call: 127 -> 119 us)
        if (!FEW) load_query(g);   // no registers to hold them from before the last part's end
#pragma unroll
        for (int i = 0; i < QN; ++i) {
          const int r = (i * 256 + tid) / CH, ch = tid % CH;
          const uint32_t sub = PL::OFF_Q + (uint32_t)(ch >> 3) * PL::SUB_BYTES;
          if constexpr (ACT32) {
            const uint32_t* x = reinterpret_cast<const uint32_t*>(raw[i]);
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float a = __uint_as_float(x[2 * k]), b = __uint_as_float(x[2 * k + 1]);
              hi[k] = pack_bf16(a, b);
              lo[k] = pack_bf16(a - __uint_as_float(hi[k] << 16), b - __uint_as_float(hi[k] & 0xffff0000u));
            }
            const int r_hi = (r >> 4) * 32 + (r & 15);
            const uint32_t at = sub + (uint32_t)(r_hi * 128 + (((ch & 7) ^ (r_hi & 7)) << 4));
            *reinterpret_cast<uint4*>(smem + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(smem + at + 16 * 128) = make_uint4(lo[0], lo[1], lo[2], lo[3]);   // 16 rows on: the same swizzle
          } else {
            *reinterpret_cast<uint4*>(smem + sub + (uint32_t)(r * 128 + (((ch & 7) ^ (r & 7)) << 4))) = raw[i][0];
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(TB_Q));

        // ---------------------------------------------------------------- softmax
        if (rank < p.warps) {
          bool hole = false;   // does the part meet a page that is not held?
          for (int i = (g.k_begin >> p.batch.page_shift) + lane; i <= (g.k_end - 1) >> p.batch.page_shift; i += 32) {
            const int id = p.batch.table[(int64_t)g.seq * p.batch.table_stride + i];
            if (id < 0 || id >= p.batch.n_pages) {
              hole = true;
              if (id != -1 && rank == 0 && g.head0 == 0) paged::refuse(p.batch.status, paged::REFUSED_PAGE, g.seq, id);
            }
          }
          const bool holes = __any_sync(0xffffffffu, hole);
          constexpr uint32_t LO = 16u << 16;   // ACT32: the low halves' lanes
          const uint32_t t_row = tmem_base + ((uint32_t)lane_base << 16), t_o = t_row + PL::O_COL;
          int lim[2];   // the last key that rows r0 and r0 + 8 see
#pragma unroll
          for (int h = 0; h < 2; ++h) lim[h] = r0 + 8 * h < g.rows ? g.pos + (r0 + 8 * h) / g.heads : -1;
          float m_used[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
          for (int j = 0; j < g.n; ++j, ++c) {
            const uint32_t t_s = t_row + (FEW ? (uint32_t)(c & 1) * 128u : 0u);
            ok = __all_sync(0xffffffffu, wait_for(bar(TB_S + (FEW ? c & 1 : 0)), (uint32_t)((FEW ? c >> 1 : c) & 1), 30, c));
            if (!ok) break;
            const int key0 = g.k_begin + j * KEYS;
            // g.pos: the last key the tile's first row sees.  Here, while there are registers for it, and not before S is there: with one stage,
            // S says that the values before these have arrived and been used, so that the parity waited for is these values' own
            if (key0 + KEYS - 1 > g.pos) {
              ok = __all_sync(0xffffffffu, wait_for(bar(TB_VF + c % STG), (uint32_t)((c / STG) & 1), 31, c));
              if (!ok) break;
              if (clear_odd<HDP>(smem_base + PL::OFF_V + (c % STG) * PL::TILE_BYTES, max(g.pos + 1 - key0, 0), g.last + 1 - key0, rank * 32 + lane, p.warps * 32)) *s_odd = item + 1;
            }
            tc_fence_after();
            // s[4g + 2h + e] = logit of row r0 + 8h, key 8g + 2 quad + e
            uint32_t s[64];
            if constexpr (ACT32) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint32_t lo[16];
                tmem_ldq256_x2(t_s + 32 * k, s + 16 * k);
                tmem_ldq256_x2(t_s + 32 * k + 16, s + 16 * k + 8);
                tmem_ldq256_x2(t_s + LO + 32 * k, lo);
                tmem_ldq256_x2(t_s + LO + 32 * k + 16, lo + 8);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) s[16 * k + i] = __float_as_uint(__uint_as_float(s[16 * k + i]) + __uint_as_float(lo[i]));
              }
            } else {
              tmem_ldq256_x8(t_s, s);
              tmem_ldq256_x8(t_s + 64, s + 32);
              tmem_wait_ld();
            }
            if (key0 + KEYS - 1 > g.pos) {
#pragma unroll
              for (int i = 0; i < 64; ++i)
                if (key0 + 8 * (i >> 2) + 2 * quad + (i & 1) > lim[(i >> 1) & 1]) s[i] = 0xff800000u;
            }
            if (holes) {
#pragma unroll 1
              for (int k = 0; k < 8; ++k) {   // 16 keys: within one page
                const int pos = key0 + 16 * k;
                if (pos >= g.k_end || page_of(p.batch, g.seq, pos, false) >= 0) continue;
#pragma unroll
                for (int i = 0; i < 64; ++i)
                  if ((i >> 3) == k) s[i] = 0xff800000u;
              }
            }
            float mx[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float ma = -INFINITY, mb = -INFINITY;
#pragma unroll
              for (int k = 0; k < 16; k += 2) {
                ma = max3(ma, __uint_as_float(s[4 * k + 2 * h]), __uint_as_float(s[4 * k + 2 * h + 1]));
                mb = max3(mb, __uint_as_float(s[4 * k + 4 + 2 * h]), __uint_as_float(s[4 * k + 4 + 2 * h + 1]));
              }
              mx[h] = fmaxf(ma, mb) * scale;
            }
            const bool grown = mx[0] > m_used[0] + TC_RESCALE || mx[1] > m_used[1] + TC_RESCALE;
            if (j == 0 || __any_sync(0xffffffffu, grown)) {
              float f[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                const float m_new = mx[h] > m_used[h] + TC_RESCALE ? mx[h] : m_used[h];   // minus infinity until the row sees a key
                f[h] = m_new != m_used[h] ? fast_exp2(m_used[h] - m_new) : 1.0f;
                l[h] *= f[h];
                m_used[h] = m_new;
              }
              if (j > 0) {
                if constexpr (FEW) {   // P V(c - 1) may still be running; with one S tile it finished before S(c) did
                  ok = __all_sync(0xffffffffu, wait_for(bar(TB_O), (uint32_t)((c - 1) & 1), 32, c));
                  if (!ok) break;
                  tc_fence_after();
                }
#pragma unroll
                for (int k = 0; k < (ACT32 ? 2 : 1) * (HDP / 16); ++k) {
                  const uint32_t at = t_o + (k % (HDP / 16)) * 16 + (k >= HDP / 16 ? LO : 0u);
                  uint32_t o[8];
                  tmem_ldq256_x2(at, o);
                  tmem_wait_ld();
#pragma unroll
                  for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f[(i >> 1) & 1]);
                  tmem_stq256_x2(at, o);
                }
              }
            }
            // p = 2^(s scale - m), handed over in three pieces (64, 32, 32 keys); the sum is of the unrounded ones.  They are rounded to bf16, the type of the
            // values they multiply (fp32 activations: to two halves, 2^-16): with the output's own rounding 2.3e-3 off in the 2-norm, that alone
            // 1.7e-3.  Of a row that has seen no key all s are minus infinity, and any finite m gives the zeros
            const float nm[2] = {-fmaxf(m_used[0], -FLT_MAX), -fmaxf(m_used[1], -FLT_MAX)};
            const float2 nm2[2] = {make_float2(nm[0], nm[0]), make_float2(nm[1], nm[1])};
            float2 rs[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            auto quarter = [&](const int q) {
              uint32_t pk[8], pl[ACT32 ? 8 : 1];
#pragma unroll
              for (int k = 4 * q; k < 4 * q + 4; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const float2 xx = ffma2(make_float2(__uint_as_float(s[4 * k + 2 * h]), __uint_as_float(s[4 * k + 2 * h + 1])), scale2, nm2[h]);
                  const float p0 = fast_exp2(xx.x), p1 = fast_exp2(xx.y);
                  const uint32_t pw = pack_bf16(p0, p1);
                  pk[2 * (k & 3) + h] = pw;
                  if constexpr (ACT32) pl[2 * (k & 3) + h] = pack_bf16(p0 - __uint_as_float(pw << 16), p1 - __uint_as_float(pw & 0xffff0000u));
                  rs[h] = fadd2(rs[h], make_float2(p0, p1));
                }
              tmem_stq128_x4(t_s + 16 * q, pk);
              if constexpr (ACT32) tmem_stq128_x4(t_s + LO + 16 * q, pl);
            };
            auto hand_over = [&](int b) {
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(b));
            };
            quarter(0);
            quarter(1);
            hand_over(TB_P1 + (FEW ? c & 1 : 0));
            quarter(2);
            hand_over(TB_P2 + (FEW ? c & 1 : 0));
            quarter(3);
            hand_over(TB_P3 + (FEW ? c & 1 : 0));
            l[0] += rs[0].x + rs[0].y;
            l[1] += rs[1].x + rs[1].y;
          }
          if (ok) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
              l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            }
            if (quad == 0) {
              red_l[r0] = l[0]; red_l[r0 + 8] = l[1];
              red_m[r0] = m_used[0]; red_m[r0 + 8] = m_used[1];
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(TB_RED));
          }
        } else {
          c += g.n;
        }
        // ---------------------------------------------------------------- epilogue: a lane a row, warps w and w + 4 half the columns each.  All eight wait for the
        // item's last product: it has read the query tile and left O, which the next item's overwrite
        const int at = item;
        if (ok) {   // the next part's query rows are asked for meanwhile
          ++item;
          gn = next_segment(17);
          if (FEW && gn != nullptr) load_query(*gn);
          item = at;
        }
        if (ok) ok = __all_sync(0xffffffffu, wait_for(bar(TB_DONE), (uint32_t)(item & 1), 34, c));
        if (ok) ok = __all_sync(0xffffffffu, wait_for(bar(TB_RED), (uint32_t)(item & 1), 36, c));
        const int first_row = ACT32 ? (warp & 3) * 16 : (warp & 3) * 32;
        if (ok && first_row < g.rows) {
          tc_fence_after();
          constexpr int OC = HDP / 2;
          const int col0 = (warp >> 2) * OC;
          const int r = ACT32 ? first_row + (lane & 15) : first_row + lane;
          const uint32_t t_o = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + PL::O_COL + col0;
          const bool mine = r < g.rows && (!ACT32 || lane < 16);
          const int rr = min(r, g.rows - 1), t = rr / g.heads;
          const float sum = red_l[rr];
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          char* dst = p.out + (int64_t)(g.token0 + t) * p.out_st + (g.head0 + rr - t * g.heads) * p.out_sh;
          const int64_t slot = (int64_t)g.slot * p.rows_max + rr;
          if (g.slot >= 0 && mine && col0 == 0) {
            p.part_ml[slot * 2] = red_m[rr];
            p.part_ml[slot * 2 + 1] = sum;
          }
#pragma unroll
          for (int k = 0; k < OC / 16; ++k) {
            uint32_t o[16];
            tmem_ld16(t_o + k * 16, o);
            tmem_wait_ld();
            if constexpr (ACT32)
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) + __uint_as_float(__shfl_xor_sync(0xffffffffu, o[i], 16)));
            const int col = col0 + k * 16;
            if (mine && col < p.hs) {
              if (g.slot >= 0) {   // the lanes' rows side by side
                float4* f = reinterpret_cast<float4*>(p.part_acc) + ((int64_t)g.slot * (p.hs / 4) + col / 4) * p.rows_max + rr;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  f[(int64_t)i * p.rows_max] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
              } else if constexpr (ACT32) {
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                  *reinterpret_cast<float4*>(reinterpret_cast<float*>(dst) + col + i) = make_float4(
                      __uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv, __uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
              } else {
#pragma unroll
                for (int i = 0; i < 16; i += 8)
                  *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(dst) + col + i) =
                      make_uint4(pack_bf16(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv), pack_bf16(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv),
                                 pack_bf16(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv), pack_bf16(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv));
              }
            }
          }
          if (*s_odd == item + 1 && mine) {
            const int n = min(OC, p.hs - col0);
            if (g.slot >= 0) add_odd<float>(p, g, g.pos + t, col0, n, p.part_acc + ((int64_t)g.slot * (p.hs / 4) * p.rows_max + rr) * 4, p.rows_max * 4);
            else if constexpr (ACT32) add_odd<float>(p, g, g.pos + t, col0, n, reinterpret_cast<float*>(dst), 4);
            else add_odd<__nv_bfloat16>(p, g, g.pos + t, col0, n, reinterpret_cast<__nv_bfloat16*>(dst), 4);
          }
          tc_fence_before();   // O has been read before the query tile's barrier lets the next products start
        }
      }
      if (!ok) break;
      release_segment();
      gp = gn;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == TC_WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem_base, PL::TMEM);
  }
}

// Join of the items that several CTAs worked on: out = sum_s 2^(m_s - M) acc_s / sum_s 2^(m_s - M) l_s over their parts, in the order
// of the CTAs.  Block x is the CTA where an item ended; 2^row_shift neighbouring threads take its rows, as the parts lie, and each
// JOIN_QUADS pieces of four elements.
constexpr int JOIN_QUADS = 4;
template <typename T>
__global__ void __launch_bounds__(256) paged_join_kernel(const AttnArgs p) {
  mca_pdl_launch_dependents();
  mca_pdl_wait();
  const int gave_up = __ldcg(p.batch.status + paged::WAIT_WORDS);   // then there are parts that nobody wrote
  const int4 m0 = __ldcg(p.meta + 2 * blockIdx.x);
  const int heads = __ldcg(p.meta + 2 * blockIdx.x + 1).x;
  const int r = threadIdx.x & ((1 << p.row_shift) - 1), lanes = 256 >> p.row_shift, quads = p.hs / 4;
  const int q0 = blockIdx.y * lanes * JOIN_QUADS + (threadIdx.x >> p.row_shift);
  if (gave_up != 0 || m0.x < 0 || r >= m0.w || q0 >= quads) return;
  const int first = m0.x, n = (int)blockIdx.x - first + 1;
  auto slot = [&](int k) { return 2ll * (first + k) + (k == 0 ? 1 : 0); };   // the first CTA's last part, then the others' first ones
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + r;
  const float4* acc = reinterpret_cast<const float4*>(p.part_acc) + r;
  float M = -INFINITY;
#pragma unroll 4
  for (int k = 0; k < n; ++k) {
    const float2 v = ml[slot(k) * p.rows_max];
    if (v.y != 0.f) M = fmaxf(M, v.x);
  }
  float sum = 0.f;
  float4 a[JOIN_QUADS];
#pragma unroll
  for (int i = 0; i < JOIN_QUADS; ++i) a[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
  for (int k = 0; k < n; ++k) {
    const float2 v = ml[slot(k) * p.rows_max];
    float4 x[JOIN_QUADS];
#pragma unroll
    for (int i = 0; i < JOIN_QUADS; ++i)
      if (q0 + i * lanes < quads) x[i] = acc[(slot(k) * quads + q0 + i * lanes) * p.rows_max];
    const float f = v.y == 0.f ? 0.f : fast_exp2(v.x - M);
    sum = fmaf(v.y, f, sum);
#pragma unroll
    for (int i = 0; i < JOIN_QUADS; ++i) {
      a[i].x = fmaf(x[i].x, f, a[i].x); a[i].y = fmaf(x[i].y, f, a[i].y); a[i].z = fmaf(x[i].z, f, a[i].z); a[i].w = fmaf(x[i].w, f, a[i].w);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int t = r / heads;
  char* dst = p.out + (int64_t)(m0.y + t) * p.out_st + (m0.z + r - t * heads) * p.out_sh;
#pragma unroll
  for (int i = 0; i < JOIN_QUADS; ++i) {
    const int q = q0 + i * lanes;
    if (q >= quads) continue;
    if constexpr (sizeof(T) == 4) reinterpret_cast<float4*>(dst)[q] = make_float4(a[i].x * inv, a[i].y * inv, a[i].z * inv, a[i].w * inv);
    else reinterpret_cast<uint2*>(dst)[q] = make_uint2(pack_bf16(a[i].x * inv, a[i].y * inv), pack_bf16(a[i].z * inv, a[i].w * inv));
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Takes what the status words say out of them.  A wait that gave up goes first and leaves the refusals for the next reading, as does a
// refusal whose details are still being written.
// ---------------------------------------------------------------------------------------------------------------------
__device__ int g_taken[4];
__global__ void __launch_bounds__(1) take_status_kernel(int* words) {
  volatile int* const w = words;
  int kind = 0, a = 0, b = 0, n = 0;
  if (w[paged::WAIT_WORDS] != 0) {
    __threadfence();
    kind = paged::REFUSED_WAIT; a = w[paged::WAIT_WORDS + 1]; b = w[paged::WAIT_WORDS + 2]; n = 1;
    for (int i = 3; i > 0; --i) w[paged::WAIT_WORDS + i] = 0;
    __threadfence();
    w[paged::WAIT_WORDS] = 0;
  } else if (w[0] > 0) {
    kind = w[0];
    __threadfence();
    a = w[1]; b = w[2];
    __threadfence();
    atomicExch(words, 0);
    __threadfence();
    n = max(atomicExch(words + 3, 0), 1);   // 0: counted by the reading before, which came between its count and its details
  }
  g_taken[0] = kind; g_taken[1] = a; g_taken[2] = b; g_taken[3] = n;
}

// ---------------------------------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------------------------------
struct Plan {
  bool tc, few;
  int rows;       // query rows of a tile
  int tiles, split_len, nsplit;                             // fp32 kernel
  int tile_shift, parts, ctas, span, inner, least_units, rows_max;       // tensor-core kernel
  bool join;
  int64_t bytes;  // of workspace
};

// Which kernel, and how the keys are shared out.
int make_plan(const McaPagedCache* c, const McaPagedBatch* b, int dtype, Plan* out) {
  const int group = c->n_heads / c->n_kv_heads;
  const int64_t most_rows = (int64_t)b->max_new * group;   // of one sequence and key/value head
  const bool act32 = dtype == MCA_DTYPE_F32;
  *out = Plan{};
  // bf16 pages: the tensor-core kernel, but for fp32 queries that share their keys with none (16 tokens over 2000 keys of 32 heads of
  // 128: 76 us in exact fp32 here, bound by memory either way; with 4 queries to a key 65 us there and 31 on the tensor cores)
  out->tc = !act32 || (c->dtype == MCA_DTYPE_BF16 && most_rows > 1);
  if (out->tc) {
    const int R = act32 ? 64 : 128;
    out->rows = R;
    // tokens of a tile: a power of two, for which a sequence's key tiles have a closed sum (a group of 3, 5 or 6 heads leaves a
    // quarter or a third of the tile's rows empty)
    while (group << (out->tile_shift + 1) <= R) ++out->tile_shift;
    const int tile_tokens = 1 << out->tile_shift;
    out->parts = mca_ceil_div(group, R);
    out->few = b->max_new <= tile_tokens;
    out->rows_max = std::min(tile_tokens, b->max_new) * std::min(group, R);
    out->least_units = 2;
    const int64_t tiles = out->few ? b->n_seqs : (int64_t)b->n_tokens / tile_tokens + b->n_seqs;
    const double units = (double)tiles * out->parts * c->n_kv_heads * (b->max_len / KEYS + 1 + ITEM_UNITS);
    out->ctas = (int)std::min((double)(out->few ? 148 : 296), std::max(1.0, std::ceil(units / out->least_units)));
    const int items = out->parts * c->n_kv_heads;
    out->span = out->ctas; out->inner = items;
    // each head CTAs of its own where that leaves out at most an eighth of them.  64 sequences of 1200 to 4000 keys, heads of 64, with / without: 12 heads
    // (144 of 148 CTAs) 110 / 126 us, 20 (140) 178 / 202, 32 (128: a seventh, and so without) 302 / 316, 40 (120) 398 / 391; four prompts of 400 to
    // 1000, 128-wide: 12 heads (288 of 296) 37.0 / 36.5, 20 (280) 48.1 / 49.4
    if (out->ctas / items * items * 8 >= out->ctas * 7) {
      out->span = out->ctas / items; out->inner = 1;
      out->ctas = out->span * items;
    }
    out->join = b->max_len > KEYS && out->span > 1;   // an item of one key tile is one CTA's
    out->bytes = out->join ? (int64_t)out->ctas * (2ll * out->rows_max * (c->head_size + 2) * 4 + 32) : 0;
    return 0;
  }
  // fp32 pages: more than eight rows on tiles, fewer a lane group a key, four rows a CTA, which read a sequence's keys once for each four.  16 tokens over 500 to
  // 1500 keys, rows x 4 heads of 64 over 4, tiles / lane groups: 5 rows 36.0 / 26.2 us, 8 36.0 / 34.0, 9 36.4 / 41.6, 16 37.1 / 55.7; 128-wide 5 62 / 46,
  // 8 62 / 49, 9 62 / 65, 16 63 / 83.  In steps that leave most of the machine empty the lane groups are ahead for longer (three chunks over 100 to 500 keys,
  // 8 heads of 64: 9 rows 19.5 / 10.8, 24 23.6 / 11.4): the rule is that of full ones.
  out->rows = most_rows > 8 ? TILE_ROWS : (most_rows > 2 ? 4 : (int)most_rows);
  const int64_t tiles = most_rows <= out->rows ? b->n_seqs : (int64_t)b->n_tokens * group / out->rows + b->n_seqs;
  if (tiles >= (1ll << 30)) return ERROR_PARAM_OUT_OF_RANGE;
  out->tiles = (int)tiles;
  const int64_t ctas = tiles * c->n_kv_heads;
  const int tile_bytes = (TILE_ROWS + TILE_KEYS) * (c->head_size + 4) * 4 + TILE_KEYS * (c->head_size + TILE_ROWS + 4) * 4 + 2048;
  const int slots = out->rows == TILE_ROWS ? 148 * (227 * 1024 / tile_bytes) : (out->rows == 4 ? 148 : 296);
  // time in keys of one CTA: whole waves of (set-up + the keys of a split); more than one split also writes partial results (at some 5 TB/s)
  // and joins them in some 4 us.  128 keys take a lane group's CTA about a microsecond, a tile's eight (of 48-wide heads; with 5, 14 and 24 for them the splits, and the
  // times of 19 of 20 steps of 32- to 128-wide heads, are the same: only four prompts of up to 200 over 512, 16 heads of 64, take 53 us from 14 on for 69).
  const double key_us = (out->rows == TILE_ROWS ? 8.0 : 1.0) / 128.0;
  const double part_keys = (double)b->n_tokens * c->n_heads * c->head_size * 8.0 / 5e6 / key_us, join_keys = 4.0 / key_us;
  double best = 1e300;
  int64_t len = 0;
  const int step = out->rows == TILE_ROWS ? TILE_KEYS : 16;
  for (int n = 1; n <= std::max(1, std::min(64, b->max_len / 128)); ++n) {
    const int64_t l = ((b->max_len + n - 1) / n + step - 1) / step * step;
    const double cost = (double)((ctas * n + slots - 1) / slots) * (64.0 + (double)l) + (n > 1 ? join_keys + n * part_keys : 0);
    if (cost < best) { best = cost; len = l; }
  }
  out->split_len = (int)len;
  out->nsplit = (int)((b->max_len + len - 1) / len);
  out->join = out->nsplit > 1;
  out->bytes = out->join ? (int64_t)b->n_tokens * c->n_heads * out->nsplit * (c->head_size + 2) * 4 : 0;
  return 0;
}

int page_map(CUtensorMap* map, const void* base, const McaPagedCache* c) {
  EncodeTiledFn fn = get_encode_fn();
  if (!fn) return ERROR_NOT_IMPLEMENTED;
  const cuuint64_t dims[4] = {(cuuint64_t)c->head_size, (cuuint64_t)c->n_kv_heads, (cuuint64_t)c->page_size, (cuuint64_t)c->n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)c->head_size * 2, (cuuint64_t)c->n_kv_heads * c->head_size * 2, (cuuint64_t)c->page_stride * 2};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)std::min(c->page_size, KEYS), 1}, ones[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : ERROR_PARAM_OUT_OF_RANGE;
}

template <int HDP, bool ACT32, bool FEW>
int launch_tc(const McaPagedCache* c, const AttnArgs& a, cudaStream_t st) {
  CUtensorMap mk, mv;
  int e;
  if ((e = page_map(&mk, c->k_pages, c)) || (e = page_map(&mv, c->v_pages, c))) return e;
  static std::atomic<uint64_t> done{0};
  if ((e = mca_smem_once(done, paged_tc_kernel<HDP, ACT32, FEW>, TcPlan<HDP, FEW>::BYTES))) return e;
  return mca_launch_pdl(paged_tc_kernel<HDP, ACT32, FEW>, dim3(a.ctas + 1), dim3(TC_THREADS), TcPlan<HDP, FEW>::BYTES, st, mk, mv, a);
}
template <bool ACT32, bool FEW>
int launch_tc(const McaPagedCache* c, const AttnArgs& a, cudaStream_t st) {
  return a.hs <= 64 ? launch_tc<64, ACT32, FEW>(c, a, st) : launch_tc<128, ACT32, FEW>(c, a, st);
}
template <int HS>
int launch_tile(const AttnArgs& a, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const int e = mca_smem_once(done, paged_tile_kernel<HS>, TilePlan<HS>::BYTES);
  if (e) return e;
  return mca_launch_pdl(paged_tile_kernel<HS>, dim3(a.tiles + 1, a.n_kv, a.nsplit), dim3(TILE_THREADS), TilePlan<HS>::BYTES, st, a);
}

template <typename CT, int HS, int R>
int launch_simt(const AttnArgs& a, cudaStream_t st) {
  constexpr size_t smem = Lanes<CT, HS>::RING;
  static std::atomic<uint64_t> done{0};
  const int e = mca_smem_once(done, paged_simt_kernel<CT, HS, R>, smem);
  if (e) return e;
  return mca_launch_pdl(paged_simt_kernel<CT, HS, R>, dim3(a.tiles + 1, a.n_kv, a.nsplit), dim3(SIMT_THREADS), smem, st, a);
}
template <int HS>
int launch_f32(int rows, bool bf16_pages, const AttnArgs& a, cudaStream_t st) {
  if (bf16_pages) return launch_simt<__nv_bfloat16, HS, 1>(a, st);
  switch (rows) {
    case 1: return launch_simt<float, HS, 1>(a, st);
    case 2: return launch_simt<float, HS, 2>(a, st);
    case 4: return launch_simt<float, HS, 4>(a, st);
    default: return launch_tile<HS>(a, st);
  }
}
int check_types(const McaPagedCache* c, int dtype) {
  if (dtype != MCA_DTYPE_F32 && dtype != MCA_DTYPE_BF16) return ERROR_ATTN_UNSUPPORTED_SHAPE;
  if (dtype == MCA_DTYPE_BF16 && c->dtype != MCA_DTYPE_BF16) return ERROR_ATTN_UNSUPPORTED_SHAPE;
  return c->n_kv_heads > 65535 ? ERROR_PARAM_OUT_OF_RANGE : 0;
}

}  // namespace

int64_t mca_paged_attention_workspace_bytes(const McaPagedCache* cache, const McaPagedBatch* batch, int dtype) {
  Batch view;
  Plan plan;
  if (paged::check(cache, batch, &view) || check_types(cache, dtype) || make_plan(cache, batch, dtype, &plan)) return -1;
  return plan.bytes;
}

int mca_paged_attention(const McaPagedCache* cache, const McaPagedBatch* batch, int dtype, const McaHeads* q, float scale, const McaHeads* out,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  AttnArgs a;
  int e = paged::check(cache, batch, &a.batch);
  if (e || (e = check_types(cache, dtype))) return e;
  // as a power of two's factor it has to be a normal number too: minus infinity times a zero is no mask, nor is infinity a factor
  if (scale != 0.f && !(scale * LOG2E >= FLT_MIN && scale * LOG2E <= FLT_MAX)) return ERROR_PARAM_OUT_OF_RANGE;
  if (batch->n_tokens == 0) return 0;
  if ((e = paged::check_heads(q, dtype, false)) || (e = paged::check_heads(out, dtype, false))) return e;
  Plan plan;
  if ((e = make_plan(cache, batch, dtype, &plan))) return e;
  if (plan.bytes > 0) {
    if (!workspace || workspace_bytes < plan.bytes) return ERROR_ATTN_SCRATCH_TOO_SMALL;
    if ((uintptr_t)workspace & 15) return ERROR_PARAM_OUT_OF_RANGE;
  }
  if ((e = paged::find_status(&a.batch.status))) return e;
  const int D = cache->head_size, size = dtype == MCA_DTYPE_BF16 ? 2 : 4, csize = cache->dtype == MCA_DTYPE_BF16 ? 2 : 4;
  a.q = static_cast<const char*>(q->data); a.out = static_cast<char*>(out->data);
  a.q_st = q->stride_t * size; a.q_sh = q->stride_h * size; a.out_st = out->stride_t * size; a.out_sh = out->stride_h * size;
  a.k_pages = static_cast<const char*>(cache->k_pages); a.v_pages = static_cast<const char*>(cache->v_pages);
  a.page_bytes = cache->page_stride * csize; a.row_bytes = (int64_t)cache->n_kv_heads * D * csize;
  a.n_heads = cache->n_heads; a.n_kv = cache->n_kv_heads; a.group = cache->n_heads / cache->n_kv_heads; a.hs = D;
  a.split_len = plan.split_len; a.nsplit = plan.nsplit; a.tiles = plan.tiles;
  a.scale_log2 = (scale == 0.f ? 1.0f / sqrtf((float)D) : scale) * LOG2E;
  a.tile_shift = plan.tile_shift; a.parts = plan.parts; a.items = plan.parts * cache->n_kv_heads;
  a.ctas = plan.ctas; a.span = plan.span; a.inner = plan.inner; a.least_units = plan.least_units; a.warps = (plan.rows_max + 15) / 16; a.rows_max = plan.rows_max;
  a.row_shift = 0;
  while (1 << a.row_shift < plan.rows_max) ++a.row_shift;
  const int64_t slots = plan.tc ? 2ll * plan.ctas * plan.rows_max : (int64_t)batch->n_tokens * cache->n_heads * plan.nsplit;
  a.part_acc = plan.join ? static_cast<float*>(workspace) : nullptr;
  a.part_ml = plan.join ? a.part_acc + slots * D : nullptr;
  a.meta = plan.join && plan.tc ? reinterpret_cast<int4*>(a.part_ml + slots * 2) : nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  const bool f32 = dtype == MCA_DTYPE_F32;
  if (plan.tc) {
    if (f32) e = plan.few ? launch_tc<true, true>(cache, a, st) : launch_tc<true, false>(cache, a, st);
    else e = plan.few ? launch_tc<false, true>(cache, a, st) : launch_tc<false, false>(cache, a, st);
    if (e || !plan.join) return e;
    const dim3 grid(plan.ctas, mca_ceil_div(D / 4, (256 >> a.row_shift) * JOIN_QUADS));
    return f32 ? mca_launch_pdl(paged_join_kernel<float>, grid, dim3(256), 0, st, a) : mca_launch_pdl(paged_join_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, a);
  }
  switch (D) {
#define MCA_PAGED_CASE(HS_) case HS_: e = launch_f32<HS_>(plan.rows, csize == 2, a, st); break;
    MCA_PAGED_CASE(32) MCA_PAGED_CASE(48) MCA_PAGED_CASE(64) MCA_PAGED_CASE(96) MCA_PAGED_CASE(128)
#undef MCA_PAGED_CASE
    default: return ERROR_ATTN_UNSUPPORTED_SHAPE;
  }
  if (e || !plan.join) return e;
  const int64_t rows = (int64_t)batch->n_tokens * cache->n_heads;
  return mca_launch_pdl(paged_simt_join_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, a);
}

int mca_paged_device_status(int** words) {
  static std::atomic<int*> known[MCA_FAIL_DEVICES];
  int dev = 0;
  MCA_CUDA_TRY(cudaGetDevice(&dev));
  int* at = dev < MCA_FAIL_DEVICES ? known[dev].load(std::memory_order_relaxed) : nullptr;
  if (at == nullptr) {
    MCA_CUDA_TRY(cudaGetSymbolAddress((void**)&at, g_status));
    if (dev < MCA_FAIL_DEVICES) known[dev].store(at, std::memory_order_relaxed);
  }
  *words = at;
  return 0;
}

int mca_paged_status_of(int* status, int* status4) {
  if (!status || !status4) return ERROR_PARAM_NULL;
  if ((uintptr_t)status & 15) return ERROR_PARAM_OUT_OF_RANGE;
  static std::mutex one_reader;   // of g_taken
  std::lock_guard<std::mutex> lock(one_reader);
  take_status_kernel<<<1, 1>>>(status);
  const int e = mca_launch_status();
  if (e) return e;
  return (int)cudaMemcpyFromSymbol(status4, g_taken, sizeof(int) * 4);
}
int mca_paged_status(int* status4) {
  if (!status4) return ERROR_PARAM_NULL;
  int* words = nullptr;
  const int e = mca_paged_device_status(&words);
  return e ? e : mca_paged_status_of(words, status4);
}

int mca_set_fail_words_paged(int* words) {
  MCA_CUDA_TRY(cudaMemcpyToSymbol(paged::g_fail_words, &words, sizeof(words)));
  return (int)cudaMemcpyToSymbol(tc::g_fail_words, &words, sizeof(words));
}
