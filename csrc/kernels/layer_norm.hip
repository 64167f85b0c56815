// Layer norm over the last dimension, forward and backward.
//
//   mu = mean x, r = (mean (x - mu)^2 + eps)^-1/2, xh = (x - mu) r, y = gamma xh + beta
//   g = gamma dy, dx = r (g - mean g - xh mean(g xh)), dgamma = sum_rows dy xh, dbeta = sum_rows dy
//
// Bound by memory: each row is read once into the registers of one group of threads -- 8, 16, 32 or 64 lanes of a
// wave, or a block of 2 to 16 waves -- where its mean and then its centred square sum are formed in f32 (no
// difference of large squares), and written once.  A group walks over many rows, so gamma and beta stay in its
// registers, and it has the next row's loads in flight while it reduces the present one.  The group is the one whose
// vectors the row fills best: instructions on empty lanes cost as much as on full ones.
// The weights' gradients are summed by column in the group's registers over all its rows; the groups of a block join,
// then the blocks through `part`, in one order each (no atomics: equal inputs give equal gradients).
#include "row_vec.h"
#include "tfx_kernels.h"

namespace tfx {

namespace {

// The group of a row: L lanes of a wave (several groups a wave, 256 threads a block), or for L = 0 the whole block.
template <int L>
__device__ __forceinline__ int group_threads() {
  return L ? L : (int)blockDim.x;
}

// vector v of thread t holds the row's elements (v * tpr + t) * N ..., once fix_row has put 0 past the end
template <typename T, int NV, bool SHORT>
__device__ __forceinline__ void load_row(const T* row, int t, int tpr, int C, u32x4_t* raw) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int v = 0; v < NV; ++v) raw[v] = vec_ld_near<T, SHORT>(row, (v * tpr + t) * N, C, 0u);
}
template <typename T, int NV, bool SHORT>
__device__ __forceinline__ void fix_row(u32x4_t* raw, int t, int tpr, int C) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int v = 0; v < NV; ++v)
    if ((v + 1) * tpr * N > C) raw[v] = vec_fix<T, SHORT>(raw[v], (v * tpr + t) * N, C, 0u);  // uniform
}

// the thread's columns of gamma or beta (`none` if there is none); 0 past the end
template <typename T, int NV, bool SHORT>
__device__ __forceinline__ void load_cols(const float* p, int t, int tpr, int C, float none, float* f) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int e = (v * tpr + t) * N;
    if (!p) {
#pragma unroll
      for (int j = 0; j < N; ++j) f[v * N + j] = e + j < C ? none : 0.f;
    } else if ((v + 1) * tpr * N <= C) {
#pragma unroll
      for (int h = 0; h < N; h += 4) vec_unpack<float>(vec_ld(p + h, (uint32_t)e), f + v * N + h);
    } else {
#pragma unroll
      for (int h = 0; h < N; h += 4) vec_unpack<float>(vec_ld_tail<float, SHORT>(p, e + h, C, 0u), f + v * N + h);
    }
  }
}

// the waves' sums in red, four at a time; those of waves that the block does not have are 0
template <int MAXT>
__device__ __forceinline__ float waves_sum(const float* red) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < MAXT / 64; i += 4)
    if (i * 64 < (int)blockDim.x) {  // uniform
      const float4 r = *reinterpret_cast<const float4*>(red + i);
      s += (r.x + r.y) + (r.z + r.w);
    }
  return s;
}

// sum over the group, in every thread; red: this reduction's own 16 floats (L = 0)
template <int L, int MAXT>
__device__ __forceinline__ float group_sum(float v, float* red) {
  if (L) return lanes_sum<L ? L : 64>(v);
  v = wave64_sum(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return waves_sum<MAXT>(red);
}

// the first row of the thread's group, and the groups of the grid
template <int L>
__device__ __forceinline__ int64_t first_row(int& t, int64_t& step) {
  if (!L) {
    t = threadIdx.x;
    step = gridDim.x;
    return blockIdx.x;
  }
  constexpr int G = L ? 256 / (L ? L : 1) : 1;
  t = threadIdx.x % (L ? L : 1);
  step = (int64_t)gridDim.x * G;
  const int g = threadIdx.x / (L ? L : 1);
  return (int64_t)blockIdx.x * G + (L == 64 ? __builtin_amdgcn_readfirstlane(g) : g);
}

}  // namespace

// MAXT: 256 for L > 0, else the most threads of the block
template <typename T, int L, int NV, int MAXT, bool SHORT>
__global__ void __launch_bounds__(MAXT) ln_fwd_kernel(const LayerNormArgs a) {
  constexpr int N = Vec<T>::N;
  // two reductions a row, each behind its own barrier: a slot is written again only after the other's barrier
  __shared__ __attribute__((aligned(16))) float red[2][16];
  int lane;
  int64_t step, row = first_row<L>(lane, step);
  if (row >= a.rows) return;  // a whole group
  if (!L) {
    if (threadIdx.x < 32) red[threadIdx.x >> 4][threadIdx.x & 15] = 0.f;
    __syncthreads();
  }
  const int tpr = group_threads<L>(), C = a.C;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  const float inv_c = 1.f / (float)C;
  u32x4_t next[NV];
  load_row<T, NV, SHORT>(x + row * a.stride, lane, tpr, C, next);
  float gam[NV * N], bet[NV * N];
  load_cols<T, NV, SHORT>(a.gamma, lane, tpr, C, 1.f, gam);
  load_cols<T, NV, SHORT>(a.beta, lane, tpr, C, 0.f, bet);
  for (; row < a.rows; row += step) {
    const int t = thread_again(lane);
    u32x4_t raw[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) raw[v] = next[v];
    if (row + step < a.rows) load_row<T, NV, SHORT>(x + (row + step) * a.stride, t, tpr, C, next);
    fix_row<T, NV, SHORT>(raw, t, tpr, C);
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[N];
      vec_unpack_again<T>(raw[v], f);
#pragma unroll
      for (int j = 0; j < N; ++j) s += f[j];
    }
    const float mean = group_sum<L, MAXT>(s, red[0]) * inv_c;
    float q = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[N];
      vec_unpack_again<T>(raw[v], f);
      if ((v + 1) * tpr * N <= C) {  // uniform
#pragma unroll
        for (int j = 0; j < N; ++j) q += (f[j] - mean) * (f[j] - mean);
      } else {
        const int e = (v * tpr + t) * N;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float d = e + j < C ? f[j] - mean : 0.f;
          q += d * d;
        }
      }
    }
    const float r = __builtin_amdgcn_rsqf(group_sum<L, MAXT>(q, red[1]) * inv_c + a.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[N];
      vec_unpack_again<T>(raw[v], f);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = (f[j] - mean) * r * gam[v * N + j] + bet[v * N + j];
      if (v * tpr * N < C) vec_st_block(y + row * C + v * tpr * N, t, tpr, C - v * tpr * N, f);
    }
    if (a.stats && t == 0) reinterpret_cast<float2*>(a.stats)[row] = make_float2(mean, r);
  }
}

template <typename T, int L, int NV, int MAXT, bool SHORT>
__global__ void __launch_bounds__(MAXT) ln_bwd_kernel(const LayerNormArgs a) {
  constexpr int N = Vec<T>::N, E = NV * N;
  // by the row's parity: the other one may still be read
  __shared__ __attribute__((aligned(16))) float red[2][2][16];
  __shared__ float col[L ? 2 * (L ? L : 1) * E : 1];  // the waves' column sums, added up in their order
  // sixteen waves leave 128 registers a thread: no room for the next row's loads
  constexpr bool AHEAD = MAXT < 1024;
  int lane;
  int64_t step, row = first_row<L>(lane, step);
  if (!L) {
    if (threadIdx.x < 64) (&red[0][0][0])[threadIdx.x] = 0.f;
    __syncthreads();
  }
  const int tpr = group_threads<L>(), C = a.C;
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  T* dx = static_cast<T*>(a.dx);
  const float inv_c = 1.f / (float)C;
  float gam[E], dg[E], db[E];
#pragma unroll
  for (int i = 0; i < E; ++i) dg[i] = db[i] = 0.f;
  u32x4_t nx[NV], nd[NV];
  float2 ns = make_float2(0.f, 0.f);
  if (AHEAD && row < a.rows) {
    load_row<T, NV, SHORT>(x + row * a.stride, lane, tpr, C, nx);
    load_row<T, NV, SHORT>(dy + row * a.dy_stride, lane, tpr, C, nd);
    ns = reinterpret_cast<const float2*>(a.stats)[row];
  }
  load_cols<T, NV, SHORT>(a.gamma, lane, tpr, C, 1.f, gam);
  int par = 0;
  for (; row < a.rows; row += step, par ^= 1) {
    const int t = thread_again(lane);
    if (!AHEAD) {
      load_row<T, NV, SHORT>(x + row * a.stride, t, tpr, C, nx);
      load_row<T, NV, SHORT>(dy + row * a.dy_stride, t, tpr, C, nd);
      ns = reinterpret_cast<const float2*>(a.stats)[row];
    }
    u32x4_t rx[NV], rd[NV];
    const float mean = ns.x, r = ns.y;
#pragma unroll
    for (int v = 0; v < NV; ++v) rx[v] = nx[v], rd[v] = nd[v];
    if (AHEAD && row + step < a.rows) {
      load_row<T, NV, SHORT>(x + (row + step) * a.stride, t, tpr, C, nx);
      load_row<T, NV, SHORT>(dy + (row + step) * a.dy_stride, t, tpr, C, nd);
      ns = reinterpret_cast<const float2*>(a.stats)[row + step];
    }
    fix_row<T, NV, SHORT>(rx, t, tpr, C);
    fix_row<T, NV, SHORT>(rd, t, tpr, C);
    // past the end dy, gamma and with them every term are 0
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[N], d[N];
      vec_unpack_again<T>(rx[v], f);
      vec_unpack_again<T>(rd[v], d);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float xh = (f[j] - mean) * r, g = d[j] * gam[v * N + j];
        s1 += g;
        s2 += g * xh;
        dg[v * N + j] += d[j] * xh;
        db[v * N + j] += d[j];
      }
    }
    if (!dx) continue;  // uniform
    if (L) {
      s1 = lanes_sum<L ? L : 64>(s1);
      s2 = lanes_sum<L ? L : 64>(s2);
    } else {
      s1 = wave64_sum(s1);
      s2 = wave64_sum(s2);
      if ((threadIdx.x & 63) == 0) red[par][0][threadIdx.x >> 6] = s1, red[par][1][threadIdx.x >> 6] = s2;
      __syncthreads();
      s1 = waves_sum<MAXT>(red[par][0]);
      s2 = waves_sum<MAXT>(red[par][1]);
    }
    s1 *= inv_c;
    s2 *= inv_c;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[N], d[N];
      vec_unpack_again<T>(rx[v], f);
      vec_unpack_again<T>(rd[v], d);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float xh = (f[j] - mean) * r, g = d[j] * gam[v * N + j];
        f[j] = r * (g - s1 - xh * s2);
      }
      if (v * tpr * N < C) vec_st_block(dx + row * C + v * tpr * N, t, tpr, C - v * tpr * N, f);
    }
  }
  if (!a.part) return;
  if (L) {
    // the groups of a wave, then the waves
#pragma unroll
    for (int o = L ? L : 64; o < 64; o <<= 1)
#pragma unroll
      for (int i = 0; i < E; ++i) dg[i] += __shfl_xor(dg[i], o, 64), db[i] += __shfl_xor(db[i], o, 64);
    for (int k = 0; k < 4; ++k) {
      __syncthreads();
      if ((int)(threadIdx.x >> 6) == k && (int)(threadIdx.x & 63) < L) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          col[i * L + lane] = (k ? col[i * L + lane] : 0.f) + dg[i];
          col[(E + i) * L + lane] = (k ? col[(E + i) * L + lane] : 0.f) + db[i];
        }
      }
    }
    if ((int)threadIdx.x < 192 || (int)threadIdx.x >= 192 + L) return;  // the last wave wrote what it reads
#pragma unroll
    for (int i = 0; i < E; ++i) dg[i] = col[i * L + lane], db[i] = col[(E + i) * L + lane];
  }
  float* part = a.part + (int64_t)blockIdx.x * 2 * C;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = (v * tpr + lane) * N + j;
      if (e < C) part[e] = dg[v * N + j], part[C + e] = db[v * N + j];
    }
}

// dgamma += / dbeta += the column sums of part [P][2][C]: 64 columns a block, the blocks' rows over its waves
__global__ void __launch_bounds__(1024) ln_cols_kernel(const float* __restrict__ part, int P, int C,
                                                       float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float sum[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;  // a column of 2 C
  float s = 0.f;
  if (c < 2 * C) {
    const float* from = part + c;
    int p = w;
    for (; p + 7 * 16 < P; p += 8 * 16) {  // eight loads in flight
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = from[(int64_t)(p + 16 * i) * 2 * C];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
    for (; p < P; p += 16) s += from[(int64_t)p * 2 * C];
  }
  sum[w][lane] = s;
  __syncthreads();
  if (w || c >= 2 * C) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += sum[i][lane];
  float* to = c < C ? dgamma : dbeta;
  if (to) to[c < C ? c : c - C] += s;
}

// ---------------------------------------------------------------- rows that no group's registers hold
// The row is gone through again for each of its sums (from the caches behind the first pass).
// (red: a row of 16 floats, all of which are written: 1024 threads are 16 waves)
__device__ __forceinline__ float block1024_sum(float v, float* red) { return group_sum<0, 1024>(v, red); }

// Sums of term(i, a, b) over i = from, from + step, ... < to: in pieces of 16 terms, which are added up in 64 bits (one after
// the other in f32 their roundings grow with the number of terms: a thread of a row of 2^24 columns has 16384).  All loads
// of a piece are in flight at once: 5000 rows of 20000 in bf16, forward, 250 -> 169 us
template <typename I, typename F>
__device__ __forceinline__ void long_sums(I from, I to, I step, float& a, float& b, F term) {
  double sa = 0., sb = 0.;
  for (; from + 15 * step < to; from += 16 * step) {
    float pa = 0.f, pb = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) term(from + k * step, pa, pb);
    sa += pa;
    sb += pb;
  }
  float pa = 0.f, pb = 0.f;
  for (; from < to; from += step) term(from, pa, pb);
  sa += pa;
  sb += pb;
  a = (float)sa;
  b = (float)sb;
}

template <typename T>
__global__ void __launch_bounds__(1024) ln_fwd_wide_kernel(const LayerNormArgs a) {
  __shared__ __attribute__((aligned(16))) float red[2][16];
  const float inv_c = 1.f / (float)a.C;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    T* y = static_cast<T*>(a.y) + row * a.C;
    float s, q, unused;
    long_sums((int)threadIdx.x, a.C, 1024, s, unused, [&](int i, float& p, float&) { p += elem_f32(x[i]); });
    const float mean = block1024_sum(s, red[0]) * inv_c;
    long_sums((int)threadIdx.x, a.C, 1024, q, unused, [&](int i, float& p, float&) {
      const float d = elem_f32(x[i]) - mean;
      p += d * d;
    });
    const float r = __builtin_amdgcn_rsqf(block1024_sum(q, red[1]) * inv_c + a.eps);
    for (int i = threadIdx.x; i < a.C; i += 1024)
      elem_st(y + i, (elem_f32(x[i]) - mean) * r * (a.gamma ? a.gamma[i] : 1.f) + (a.beta ? a.beta[i] : 0.f));
    if (a.stats && threadIdx.x == 0) reinterpret_cast<float2*>(a.stats)[row] = make_float2(mean, r);
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) ln_bwd_wide_kernel(const LayerNormArgs a) {
  __shared__ __attribute__((aligned(16))) float red[2][16];
  const float inv_c = 1.f / (float)a.C;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    T* dx = static_cast<T*>(a.dx) + row * a.C;
    const float2 st = reinterpret_cast<const float2*>(a.stats)[row];
    float s1, s2;
    long_sums((int)threadIdx.x, a.C, 1024, s1, s2, [&](int i, float& p1, float& p2) {
      const float g = elem_f32(dy[i]) * (a.gamma ? a.gamma[i] : 1.f);
      p1 += g;
      p2 += g * (elem_f32(x[i]) - st.x) * st.y;
    });
    s1 = block1024_sum(s1, red[0]) * inv_c;
    s2 = block1024_sum(s2, red[1]) * inv_c;
    for (int i = threadIdx.x; i < a.C; i += 1024) {
      const float g = elem_f32(dy[i]) * (a.gamma ? a.gamma[i] : 1.f);
      elem_st(dx + i, st.y * (g - s1 - (elem_f32(x[i]) - st.x) * st.y * s2));
    }
  }
}

// part[blockIdx.y] of 256 columns: the rows blockIdx.y, + gridDim.y, ...
template <typename T>
__global__ void __launch_bounds__(256) ln_cols_wide_kernel(const LayerNormArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  float dg, db;
  long_sums((int64_t)blockIdx.y, a.rows, (int64_t)gridDim.y, dg, db, [&](int64_t row, float& pg, float& pb) {
    const float2 st = reinterpret_cast<const float2*>(a.stats)[row];
    const float d = elem_f32(dy[row * a.dy_stride + c]);
    pg += d * (elem_f32(x[row * a.stride + c]) - st.x) * st.y;
    pb += d;
  });
  float* part = a.part + (int64_t)blockIdx.y * 2 * a.C;
  part[c] = dg;
  part[a.C + c] = db;
}

// ---------------------------------------------------------------- host
namespace {

struct LnShape {
  int lanes, waves, nv;  // lanes of a wave, or 0 and the block's waves; nv = 0: no group's registers hold the row
};

// A row that one wave's registers hold has lanes of a wave: 8 to 64, of 1, 2 or (in f32) 4 vectors.  Else it has the
// block and the vectors a thread that leave the fewest empty, more vectors before more waves.  (40000 rows of 5000 in bf16, backward: 5 waves x 2 vectors
// 363 us, 4 x 4 -- as many as 8192 columns need -- 626.)
template <typename T>
LnShape ln_shape(int64_t C) {
  constexpr int N = Vec<T>::N;
  const int64_t vecs = (C + N - 1) / N;
  for (int l = 8; l <= 64; l *= 2)
    if (vecs <= l) return {l, 1, 1};
  if (vecs <= 128) return {64, 1, 2};
  LnShape best = {0, 0, 0};
  for (int nv = N == 4 ? 4 : 2; nv >= 1; nv /= 2) {
    const int64_t w = (vecs + 64 * nv - 1) / (64 * nv);
    if (w <= 16 && (!best.nv || w * nv < (int64_t)best.waves * best.nv)) best = {w == 1 ? 64 : 0, (int)w, nv};
  }
  return best;
}
LnShape ln_shape(bool bf16, int64_t C) { return bf16 ? ln_shape<uint16_t>(C) : ln_shape<float>(C); }

int64_t ln_grid(LnShape s, int64_t rows, int64_t most) {
  const int64_t g = s.lanes ? 256 / s.lanes : 1;
  return std::max<int64_t>(1, std::min(most, (rows + g - 1) / g));
}
int ln_threads(LnShape s) { return s.lanes ? 256 : 64 * s.waves; }

#define LN_SHAPES(GO)                                                        \
  do {                                                                       \
    if (a.C < Vec<T>::N) GO(8, 1, 256, true);                                \
    else if (s.lanes == 8) GO(8, 1, 256, false);                             \
    else if (s.lanes == 16) GO(16, 1, 256, false);                           \
    else if (s.lanes == 32) GO(32, 1, 256, false);                           \
    else if (s.lanes == 64 && s.nv == 1) GO(64, 1, 256, false);              \
    else if (s.lanes == 64 && s.nv == 2) GO(64, 2, 256, false);              \
    else if (s.nv == 1 && s.waves <= 8) GO(0, 1, 512, false);                \
    else if (s.nv == 1) GO(0, 1, 1024, false);                               \
    else if (s.nv == 2 && s.waves <= 8) GO(0, 2, 512, false);                \
    else if (s.nv == 2) GO(0, 2, 1024, false);                               \
    else if constexpr (Vec<T>::N == 4) {                                     \
      if (s.lanes == 64) GO(64, 4, 256, false);                              \
      else if (s.waves <= 8) GO(0, 4, 512, false);                                \
      else GO(0, 4, 1024, false);                                            \
    }                                                                        \
  } while (0)

template <typename T>
void fwd_launch(const LayerNormArgs& a, hipStream_t st) {
  const LnShape s = ln_shape<T>(a.C);
  if (!s.nv) {
    launch(ln_fwd_wide_kernel<T>, (int)std::min<int64_t>(a.rows, 4096), 1024, 0, st, a);
    return;
  }
  // as many waves as are resident at once (6400 rows of 512 in bf16: 1600 blocks 5.4 us, 256 blocks 7.6; 16384 rows of
  // 8192: 1024 blocks 89 us, 6.0 TB/s).  Of more than 8 waves one or two blocks fit a CU: two a CU, or the last ones run
  // alone (in bf16, 14648 rows of 10240: 819 blocks 171 us, 512 143; 10463 of 14336: 585 blocks 146, 512 117)
  const int grid = (int)ln_grid(s, a.rows, s.lanes ? 2048 : s.waves > 8 ? 512 : 8192 / s.waves);
#define GO(L, NV, MAXT, SH) launch(ln_fwd_kernel<T, L, NV, MAXT, SH>, grid, ln_threads(s), 0, st, a)
  LN_SHAPES(GO);
#undef GO
}

template <typename T>
void bwd_launch(const LayerNormArgs& a, hipStream_t st) {
  const LnShape s = ln_shape<T>(a.C);
  const int parts = layer_norm_parts(a.bf16, a.rows, a.C);
  if (!s.nv) {
    if (a.dx) launch(ln_bwd_wide_kernel<T>, (int)std::min<int64_t>(a.rows, 4096), 1024, 0, st, a);
    if (a.part) launch(ln_cols_wide_kernel<T>, dim3((a.C + 255) / 256, parts), 256, 0, st, a);
  } else {
#define GO(L, NV, MAXT, SH) launch(ln_bwd_kernel<T, L, NV, MAXT, SH>, parts, ln_threads(s), 0, st, a)
    LN_SHAPES(GO);
#undef GO
  }
  if (a.part) launch(ln_cols_kernel, (2 * a.C + 63) / 64, 1024, 0, st, a.part, parts, a.C, a.dgamma, a.dbeta);
}

}  // namespace

// Blocks of the backward pass, each with its partial sums of the weights' gradients: more of them hide more
// latency and write more sums (6400 rows of 512 in bf16: 512 blocks 8.4 us and 3.8 to join them, 1600 blocks
// 10.7 and 5.6; 2999 rows of 1001 in f32: 512 blocks of four rows 11.0 and 4.4, a block for each row 18.0 and 13.4).
// A whole number of blocks a CU (40000 rows of 5000 in bf16: 512 blocks 363 us, 409 436); with as many as fit at once,
// 12 waves a CU for the larger shapes, the sums cost what the loads gain (66666 rows of 3000 in bf16, 3 waves each:
// 768 blocks 235 us, 1024 305; 48828 rows of 4096, 4 waves: 512 225, 768 245; 133333 rows of 1500: 768 286, 1024 259).
int layer_norm_parts(bool bf16, int64_t rows, int64_t C) {
  const LnShape s = ln_shape(bf16, C);
  if (!s.nv) return (int)std::min<int64_t>(rows, 16);
  if (s.lanes) return (int)ln_grid(s, rows, s.lanes == 64 ? 512 : 1024);
  const bool large = rows * C * (bf16 ? 2 : 4) > (64 << 20);
  return (int)ln_grid(s, rows, 256 * std::max(1, ((large ? 2048 : 4096) / s.waves + 128) / 256));
}

void layer_norm_fwd(const LayerNormArgs& a, hipStream_t st) {
  a.bf16 ? fwd_launch<uint16_t>(a, st) : fwd_launch<float>(a, st);
}

void layer_norm_bwd(const LayerNormArgs& a, hipStream_t st) {
  a.bf16 ? bwd_launch<uint16_t>(a, st) : bwd_launch<float>(a, st);
}

}  // namespace tfx
