// Log-softmax over the rows of a [rows, vocabulary] matrix: log probabilities of given tokens,
// entropies and top alternatives (token_log_probs), and the distillation loss from a teacher's top
// logits, each with its gradient.
//
// With z = x / T, a reference R near max x, c = log2(e) / T and d_v = (x_v - R) c:
//   s = sum 2^d_v,  log p_v = (x_v - R) / T - log s,  H = log s - ln2 (sum 2^d_v d_v) / s
//   d(g log p_t + h H)/dx_v = [g (1[v = t] - p_v) - h p_v (log p_v + H)] / T
//   KL = sum_k q_k (log q_k - log p_{id_k}),  d(w T^2 KL)/dx_v = w T (p_v - sum_{k: id_k = v} q_k)
// All of it is bound by memory: a row is read once, in 16-byte loads, into registers (or, only summed and longer than
// a wave holds, streamed through them), its sums are formed there, and a gradient that may be formed in the same pass is
// written from the registers (the row is never read again).  Sums, maxima and exponents are f32.
#include "row_vec.h"
#include "tfx_kernels.h"

namespace tfx {

namespace {

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLow = -200.f;  // 2^d is 0 from here on down: stands in for -inf in 2^d d

__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ int64_t whole(const void* __restrict__ p, int is64, int64_t i) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}

// Values in the order of their unsigned keys (-0 counts as 0)
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_val(uint32_t k) {
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}
// larger value first, then lower index; 0 is "nothing there"
__device__ __forceinline__ uint64_t cand_key(float v, int idx) {
  return ((uint64_t)order_key(v) << 32) | (uint32_t)~idx;
}

// Vectors that a row fills for certain where one of NV a thread was chosen for it: those of the next smaller choice
// (1, 2, 4, 8, 10, ...)
constexpr int sure_vectors(int nv) { return nv > 8 ? nv - 2 : nv / 2; }

// Vector v of the part [p0, end) of a row: thread t holds elements p0 + (v * TPB + t) * N ..., once fix_part has put
// -inf at and behind the end.  Behind the part's last vector the row's last 16 bytes are loaded again.
// The first SURE vectors are whole in every thread.
template <typename T, int TPB, int NV, int SURE, bool ONCE = false>
__device__ __forceinline__ void load_part(const T* row, int t, int p0, int end, u32x4_t* raw) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int v = 0; v < SURE; ++v) raw[v] = vec_ld<T, ONCE>(row + p0 + v * TPB * N, (uint32_t)(t * N));
#pragma unroll
  for (int v = SURE; v < NV; ++v)
    raw[v] = vec_ld_near<T, TPB == 64 && NV == 1, ONCE>(row, p0 + (v * TPB + t) * N, end, Vec<T>::kNegInf);
}
template <typename T, int TPB, int NV, int SURE>
__device__ __forceinline__ void fix_part(u32x4_t* raw, int t, int p0, int end) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int v = SURE; v < NV; ++v) {
    if (p0 + (v + 1) * TPB * N > end)  // uniform
      raw[v] = vec_fix<T, TPB == 64 && NV == 1>(raw[v], p0 + (v * TPB + thread_again(t)) * N, end, Vec<T>::kNegInf);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// ASIDE: in a branch, here and below
template <typename T, int NV, bool ASIDE = false>
__device__ __forceinline__ float lane_max(u32x4_t* raw) {
  constexpr int N = Vec<T>::N;
  float m = -INFINITY;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float f[N];
    if (ASIDE) vec_unpack_aside<T>(raw[v], f);
    else vec_unpack_again<T>(raw[v], f);
#pragma unroll
    for (int j = 0; j < N; j += 2) m = fmaxf(m, fmaxf(f[j], f[j + 1]));
    if (ASIDE) __builtin_amdgcn_sched_barrier(0);
  }
  return m;
}

// v is formed here: where only one side of a branch needs it the compiler would form it there, out of every term
__device__ __forceinline__ void form_here(float& v) { asm volatile("" : "+v"(v)); }

// s += sum 2^d, t += sum 2^d d over the lane's elements, d = (x - R) c.
// FMA: d + (R c - k) = x c - k in one rounding, with k the whole number next to R c; the caller takes the
// fraction out again.
// MAX: vm[v] = the largest of vector v.
template <typename T, int V0, int V1, bool ENT, bool FMA, bool MAX = false, bool ASIDE = false>
__device__ __forceinline__ void lane_sums(u32x4_t* raw, float R, float k, float c, float& s, float& t,
                                          float* vm = nullptr) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int v = V0; v < V1; ++v) {
    float f[N];
    if (ASIDE) vec_unpack_aside<T>(raw[v], f);
    else vec_unpack_again<T>(raw[v], f);
    if (MAX) {
      vm[v] = f[0];
#pragma unroll
      for (int j = 1; j < N; ++j) vm[v] = fmaxf(vm[v], f[j]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d = FMA ? __builtin_fmaf(f[j], c, -k) : (f[j] - R) * c;
      const float e = exp2_fast(d);
      s += e;
      if (ENT) t = __builtin_fmaf(e, fmaxf(d, kLow), t);
    }
    // one vector's unpacked values at a time: spread over all vectors they cost twice the registers
    form_here(s);
    if (ENT) form_here(t);
    __builtin_amdgcn_sched_barrier(0);
  }
}
// (m, s, t) of a piece added to S, Tt against the finite reference M, at least m
__device__ __forceinline__ void join_piece(float m, float s, float t, float M, float c, float& S, float& Tt) {
  const float d = fmaxf((m - M) * c, kLow);
  const float h = s == 0.f ? 0.f : exp2_fast(d);
  S += s == 0.f ? 0.f : s * h;
  Tt += s == 0.f ? 0.f : h * __builtin_fmaf(s, d, t);
}

// the waves' (R, s, t) joined, in every thread; red: 3 * TPB / 64 floats
template <int TPB, bool ENT>
__device__ __forceinline__ void join_waves(float c, float* red, float& R, float& s, float& t) {
  constexpr int W = TPB / 64;
  s = wave64_sum(s);
  if (ENT) t = wave64_sum(t);
  if (W == 1) return;
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) red[w] = R, red[W + w] = s, red[2 * W + w] = t;
  __syncthreads();
  // a lane for each wave: every wave joins all of them, and one after the other that were W exponentials in each
  // (4096 rows of 131072 in bf16, distillation: 466 -> 450 us)
  constexpr int L = W < 8 ? 8 : W;
  const int l = threadIdx.x & (L - 1);
  const float lr = l < W ? red[l] : 0.f, ls = l < W ? red[W + l] : 0.f, lt = ENT && l < W ? red[2 * W + l] : 0.f;
  R = finite_max(lanes_max<L>(ls == 0.f ? -INFINITY : lr));  // that of the waves that hold anything
  s = t = 0.f;
  join_piece(lr, ls, lt, R, c, s, t);
  s = lanes_sum<L>(s);
  if (ENT) t = lanes_sum<L>(t);
}

// the finite maximum of the lanes' m, in every thread; red: TPB / 64 floats, free again behind it
template <int TPB>
__device__ __forceinline__ float block_max(float m, float* red) {
  m = wave64_max(m);
  if (TPB > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TPB / 64; ++i) m = fmaxf(m, red[i]);
    __syncthreads();
  }
  return finite_max(m);
}

// Long sums are added up in two steps: pieces of kPiece vectors a lane, 32 terms at most, and the pieces.  (In one, a
// lane's rounding grew with the row: 7e-6 in the logarithm at 131072 columns of few values, 1e-3 at 2^24.)
constexpr int kPiece = 4;

// No maximum is looked for first: a wave sums against a reference R, the largest value of its first vector, which is
// there first.  Whether R was near enough shows in the pieces' sums: one of up to n terms of about 2^0 and less is at
// most sqrt(2) n against 2^k, k the whole number next to R c, and one above 1.5 n holds a value above R.  Then the wave
// takes a new reference from what it holds.  So no value is more than 2^5.6 beside its wave's reference, 3.9 nats: what
// the f32 roundings of log s and t / s leave of that distance in log p and the entropy is some 1e-6 at most.
template <typename T>
constexpr float kPieceMost = 1.5f * kPiece * Vec<T>::N;

// may be a reference: rintf(m c) is exact (of -inf: no)
__device__ __forceinline__ bool near_zero(float m, float c) { return fabsf(m * c) <= 16777216.f; }

__device__ __forceinline__ float wave_uniform(float v) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}

// lane_sums in pieces; big: at least the largest piece's sum
template <typename T, int V0, int V1, bool ENT, bool FMA>
__device__ __forceinline__ void lane_pieces(u32x4_t* raw, float R, float k, float c, float& s, float& t, float& big) {
  if constexpr (V0 < V1) {
    constexpr int E = V0 + kPiece < V1 ? V0 + kPiece : V1;
    float ps = 0.f, pt = 0.f;
    lane_sums<T, V0, E, ENT, FMA, false, !FMA>(raw, R, k, c, ps, pt);
    s += ps;
    if (ENT) t += pt;
    big = fmaxf(big, ps);
    lane_pieces<T, E, V1, ENT, FMA>(raw, R, k, c, s, t, big);
  }
}

// A reference R, sum and weighted sum of the block's part, in every thread: s = sum 2^d, t = sum 2^d d with
// d = (x - R) c.
//
// One pass in FMA form; a wave whose reference was too low, or whose first vector had none (all masked, NaN, or far
// out), goes over its registers again, against their maximum.  NaN and +inf make s NaN.
// Instructions an element in bf16: unpack, fma, exp2 (4 slots), add; against the maximum two more for that and
// one for the difference.
// The part comes as load_part left it and is whole afterwards.
template <typename T, int TPB, int NV, bool ENT>
__device__ __forceinline__ void part_stats(u32x4_t* raw, int tid, int len, float c, float* red, float& R, float& s,
                                           float& t) {
  constexpr int Q = sure_vectors(NV);
  if (Q == 0) fix_part<T, TPB, NV, 0>(raw, tid, 0, len);
  R = wave_uniform(wave64_max(lane_max<T, 1>(raw)));
  const bool near = near_zero(R, c);
  const float k = near ? rintf(R * c) : 0.f;
  float big = near ? 0.f : INFINITY;
  s = t = 0.f;
  lane_pieces<T, 0, Q, ENT, true>(raw, 0.f, k, c, s, t, big);
  if (Q) fix_part<T, TPB, NV, Q>(raw, tid, 0, len);
  lane_pieces<T, Q, NV, ENT, true>(raw, 0.f, k, c, s, t, big);
  if (__ballot(big > kPieceMost<T>)) {
    R = wave_uniform(finite_max(wave64_max(lane_max<T, NV, true>(raw))));
    s = t = 0.f;
    lane_pieces<T, 0, NV, ENT, false>(raw, R, 0.f, c, s, t, big);
  } else {
    const float off = __builtin_fmaf(-R, c, k), f = exp2_fast(off);
    if (ENT) t = f * __builtin_fmaf(s, off, t);
    s *= f;
  }
  join_waves<TPB, ENT>(c, red, R, s, t);
}

// how many of n keys in LDS are above k (eight reads in flight)
__device__ __forceinline__ int keys_above(const uint64_t* keys, int n, uint64_t k) {
  int r = 0, j = 0;
  for (; j + 8 <= n; j += 8) {
    uint64_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = keys[j + i];
#pragma unroll
    for (int i = 0; i < 8; ++i) r += v[i] > k;
  }
  for (; j < n; ++j) r += keys[j] > k;
  return r;
}

// Of n distinct keys in LDS the K largest, in order, by counting the larger ones of each (n is a few
// more than K but for rows made to defeat the threshold); `put(rank, key)` for each.
template <int TPB, typename F>
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int n, int K, F put) {
  for (int i = threadIdx.x; i < n; i += TPB) {
    const uint64_t k = keys[i];
    const int r = keys_above(keys, n, k);
    if (r < K) put(r, k);
  }
}

// The K-th largest of the 64 W keys in LDS, its bits from `LOW` on (the others 0), in every lane of the wave: from
// the highest bit on, a bit is set where K keys reach the value with it.
template <int W>
struct LaneKeys {
  uint32_t k[W];
};
template <int W, int LOW>
__device__ __forceinline__ uint32_t kth_of(LaneKeys<W> l, int K) {
  uint32_t at = 0;
#pragma unroll
  for (int b = 31; b >= LOW; --b) {
    const uint32_t tr = at | (1u << b);
    int n = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) n += __popcll(__ballot(l.k[i] >= tr));
    if (n >= K) at = tr;
  }
  return at;
}
template <int W, int LOW>
__device__ __forceinline__ uint32_t kth_key(const uint32_t* keys, int K) {
  LaneKeys<W> l;
#pragma unroll
  for (int i = 0; i < W; ++i) l.k[i] = keys[i * 64 + (threadIdx.x & 63)];
  return kth_of<W, LOW>(l, K);
}

// The K largest finite values of a row that one wave's registers hold, as keys in buf[0, n), in no order; n, at least
// the number of values asked for that are there, is at most top_room.
//
// Threshold: the K-th largest of the maxima of disjoint groups of values is a lower bound of the K-th largest value,
// for K groups hold one of at least that each -- and a tight one where the groups are many: the 64 lanes' values for
// the smallest K, 4 or 8 groups in each lane for others (16384 rows of 2048 in f32, top 64: in lanes' groups alone
// 320 us, for most of the row passes).  Its upper 16 bits do at first (the whole of it in bf16): values from there on are the
// candidates.  Where these are too many (ties, a constant row) the whole of it, t, is found: fewer than K groups hold a
// value above t, so buf holds those; then the values equal to t are taken in the order of the row.
constexpr int kFewTop = 8;
constexpr int lane_groups(int nv) { return nv > 4 ? nv : 4; }
template <typename T, int NV>
__host__ __device__ __forceinline__ int top_room(int K) {
  return K * (K <= kFewTop ? Vec<T>::N * NV : Vec<T>::N * NV / lane_groups(NV));
}

template <typename T, int NV, int LOW>
__device__ __forceinline__ float wave_kth(u32x4_t* raw, const float* vm, int K) {
  constexpr int N = Vec<T>::N, W = lane_groups(NV), GS = N * NV / W;
  uint32_t at;
  if (K <= kFewTop) {
    float m = vm[0];
#pragma unroll
    for (int v = 1; v < NV; ++v) m = fmaxf(m, vm[v]);
    at = kth_of<1, LOW>(LaneKeys<1>{{order_key(m)}}, K);
  } else {
    LaneKeys<W> l;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[N];
      vec_unpack_aside<T>(raw[v], f);
#pragma unroll
      for (int j = 0; j < N; j += GS) {
        float m = -INFINITY;  // (of NaN too)
#pragma unroll
        for (int i = j; i < j + GS; ++i) m = fmaxf(m, f[i]);
        l.k[(v * N + j) / GS] = order_key(m);
      }
    }
    at = kth_of<W, LOW>(l, K);
  }
  const float t = order_val(at);
  return t > -INFINITY ? t : -INFINITY;  // (of bits that are cut to those of a NaN)
}

// The values that pass `ok`, as keys in buf[0, room); returns how many they are
template <typename T, int NV, typename F>
__device__ __forceinline__ int wave_collect(u32x4_t* raw, const float* vm, int tid, uint64_t* buf, int room, F ok) {
  constexpr int N = Vec<T>::N;
  int n = 0;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (!__ballot(ok(vm[v]))) continue;
    float f[N];
    vec_unpack_aside<T>(raw[v], f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint64_t m = __ballot(ok(f[j]));
      if (!m) continue;
      const int at = n + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
      if (ok(f[j]) && at < room) buf[at] = cand_key(f[j], (v * 64 + tid) * N + j);
      n += __popcll(m);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  return n;
}

template <typename T, int NV>
__device__ __forceinline__ int wave_top(u32x4_t* raw, int tid, int K, uint64_t* buf) {
  constexpr int N = Vec<T>::N;
  const int room = top_room<T, NV>(K);
  float vm[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) vm[v] = lane_max<T, 1>(raw + v);
  float t = wave_kth<T, NV, 16>(raw, vm, K);
  int n = wave_collect<T, NV>(raw, vm, tid, buf, room, [&](float f) { return t > -INFINITY ? f >= t : f > t; });
  if (n <= room) return n;
  t = wave_kth<T, NV, 0>(raw, vm, K);
  n = wave_collect<T, NV>(raw, vm, tid, buf, room, [&](float f) { return f > t; });
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (n >= K || !__ballot(vm[v] >= t)) continue;  // uniform
    float f[N];
    vec_unpack_aside<T>(raw[v], f);
    int mine = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) mine += f[j] == t;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(incl, o, 64);
      if (tid >= o) incl += u;
    }
    int at = n + incl - mine;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (f[j] == t) {
        if (at < K) buf[at] = cand_key(f[j], (v * 64 + tid) * N + j);
        ++at;
      }
    n = min(K, n + __shfl(incl, 63, 64));
    __builtin_amdgcn_sched_barrier(0);
  }
  return n;
}

// One row's outputs from its maximum and sums (one thread)
__device__ __forceinline__ void put_row(const VocabArgs& a, int row, float x_tok, float M, float s, float t,
                                        float& logs) {
  const bool empty = s == 0.f;  // every logit -inf
  logs = empty ? INFINITY : logf(s);
  const float inv = empty ? 0.f : 1.f / s;
  // H = log s - ln2 t / s.  Where one value makes up the sum both are its distance from M: a whole number of halvings is
  // taken off s and t / s alike, in front of the roundings.
  const float e = rintf(fmaxf(t * inv, 0.f));
  const float H = empty ? 0.f : e == 0.f ? logs - kLn2 * t * inv : logf(__builtin_ldexpf(s, -(int)e)) + kLn2 * (__builtin_fmaf(e, s, -t) * inv);
  if (a.logp) a.logp[row] = empty ? x_tok : __builtin_fmaf(x_tok - M, a.scale, -logs);
  if (a.ent) a.ent[row] = H;
  if (a.stats) reinterpret_cast<float4*>(a.stats)[row] = make_float4(M, inv, empty ? 0.f : logs, H);
}

// A row that is padding: nothing of it is read
__device__ __forceinline__ void put_padding(const VocabArgs& a, int row) {
  if (threadIdx.x == 0) {
    if (a.logp) a.logp[row] = 0.f;
    if (a.ent) a.ent[row] = 0.f;
    if (a.stats) reinterpret_cast<float4*>(a.stats)[row] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int k = threadIdx.x; k < a.K; k += blockDim.x) {
    a.top_logp[(int64_t)row * a.K + k] = -INFINITY;
    a.top_ids[(int64_t)row * a.K + k] = -1;
  }
}

__device__ __forceinline__ bool is_padding(const VocabArgs& a, int row, int64_t& tok) {
  tok = 0;
  if (a.tok) tok = whole(a.tok, a.tok64, row);
  return tok < 0 || (a.weight && a.weight[row] == 0.f);
}

// The token's logit; NaN for a token outside the vocabulary (its log probability is then NaN)
template <typename T>
__device__ __forceinline__ float token_logit(const VocabArgs& a, int row, int64_t tok) {
  if (!a.logp) return 0.f;
  if (tok >= a.V) return NAN;
  return elem_f32(static_cast<const T*>(a.x)[(int64_t)row * a.stride + tok]);
}

__device__ __forceinline__ void put_top(const VocabArgs& a, int row, int r, uint64_t key, float M, float logs) {
  const float x = order_val((uint32_t)(key >> 32));
  a.top_logp[(int64_t)row * a.K + r] = __builtin_fmaf(x - M, a.scale, -logs);
  a.top_ids[(int64_t)row * a.K + r] = (int64_t)(uint32_t)~(uint32_t)key;
}

// The K largest of n keys in LDS: a finished row's alternatives, or its part's list
template <int TPB>
__device__ __forceinline__ void put_list(const VocabArgs& a, int row, int item, float M, float s, const uint64_t* keys,
                                         int n) {
  if (a.nparts == 1) {
    const float logs = s == 0.f ? INFINITY : logf(s);
    rank_keys<TPB>(keys, n, a.K, [&](int r, uint64_t k) { put_top(a, row, r, k, M, logs); });
    for (int k = n + threadIdx.x; k < a.K; k += TPB) {
      a.top_logp[(int64_t)row * a.K + k] = -INFINITY;
      a.top_ids[(int64_t)row * a.K + k] = -1;
    }
  } else {
    uint64_t* to = a.ws_keys + (int64_t)item * a.K;
    rank_keys<TPB>(keys, n, a.K, [&](int r, uint64_t k) { to[r] = k; });
    for (int k = n + threadIdx.x; k < a.K; k += TPB) to[k] = 0;
  }
}

}  // namespace

// Rows that one wave's registers hold
template <typename T, int NV, bool ENT, bool TOP>
__global__ void __launch_bounds__(64) vocab_stats_kernel(const VocabArgs a) {
  extern __shared__ uint64_t buf[];
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    int64_t tok;
    if (is_padding(a, row, tok)) {
      put_padding(a, row);
      continue;
    }
    u32x4_t raw[NV];
    const int tid = thread_again(threadIdx.x);
    load_part<T, 64, NV, sure_vectors(NV)>(static_cast<const T*>(a.x) + (int64_t)row * a.stride, tid, 0, a.V, raw);
    float x_tok = 0.f;
    if (threadIdx.x == 0) x_tok = token_logit<T>(a, row, tok);
    float M, s, t, logs = 0.f;
    part_stats<T, 64, NV, ENT>(raw, tid, a.V, a.c, nullptr, M, s, t);
    if (threadIdx.x == 0) put_row(a, row, x_tok, M, s, t, logs);
    if (TOP) {
      const int n = wave_top<T, NV>(raw, tid, a.K, buf);
      __syncthreads();
      put_list<64>(a, row, row, M, s, buf, n);
    }
    __syncthreads();  // buf is the next row's
  }
}

// Longer rows are streamed, nothing of them stays: a block goes over its part in pieces of kChunk vectors a thread,
// the next piece's loads ahead of the present one's sums.  The whole row is one part unless rows are few.  (4096 rows
// of 50000 in bf16: 72 us, 5.7 TB/s; with parts held in registers 105 us and 9 to join them.)
//
// Top alternatives ride along: each vector's maximum is compared with a threshold, a lower bound of the K-th largest
// value (the K-th largest of the lanes' own maxima so far), and where it reaches that, the vector's number is noted.
// The threshold is formed behind the first piece and again behind the 4th, 16th and last, so a few times K vectors are
// noted; these are read again and their values that reach the last threshold are ranked.
constexpr int kChunk = kPiece;
constexpr int kNoted = 4096;   // vectors noted: all that fewer than K lanes can hold, 64 each
constexpr int kCands = 512;    // values ranked
constexpr int kTopVecs = 64;   // vectors of a thread in a part with top alternatives

struct TopState {
  uint32_t keys[256];
  uint32_t noted[kNoted];
  uint64_t cands[kCands];
  int n_noted, n_cands;
  float thr;
  uint64_t best[4];
};

// the K-th largest of the lanes' maxima (its upper bits), in every thread; -inf where fewer than K lanes hold a value.
// COARSE: for small K of the maxima of 64 groups of four lanes: a little lower, and found in a quarter of the compares.
template <int LOW, bool COARSE = false>
__device__ __forceinline__ float block_kth(float lmax, int K, TopState& st) {
  st.keys[threadIdx.x] = order_key(lmax);
  __syncthreads();
  if (threadIdx.x < 64) {
    uint32_t at;
    if (COARSE && K <= 24) {
      const uint32_t* k = st.keys + threadIdx.x;
      at = kth_of<1, LOW>(LaneKeys<1>{{max(max(k[0], k[64]), max(k[128], k[192]))}}, K);
    } else {
      at = kth_key<4, LOW>(st.keys, K);
    }
    if (threadIdx.x == 0) st.thr = order_val(at);
  }
  __syncthreads();
  const float t = st.thr;
  return t > -INFINITY ? t : -INFINITY;  // (of bits that are cut to those of a NaN)
}

__device__ __forceinline__ bool reaches(float v, float thr) { return thr > -INFINITY ? v >= thr : v > -INFINITY; }

// Vector `vec` of thread t's elements that pass `ok`, as candidates; counted past the end of the list, not written
template <typename T, typename F>
__device__ __forceinline__ void add_cands(const T* x, int p0, int end, int vec, int t, TopState& st, F ok) {
  constexpr int N = Vec<T>::N;
  const int e = p0 + (vec * 256 + t) * N;
  if (e >= end) return;
  float f[N];
  vec_unpack<T>(vec_ld_tail<T, false>(x, e, end, Vec<T>::kNegInf), f);
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (ok(f[j])) {
      const int at = atomicAdd(&st.n_cands, 1);
      if (at < kCands) st.cands[at] = cand_key(f[j], e + j);
    }
}

// Rows that defeat the threshold: many values equal to it, or the large ones all in few lanes.  Those above the exact
// K-th largest lane maximum, then the first ones equal to it in the order of the row; if even those above are too
// many, one pass for each rank.  Returns the number of candidates.
template <typename T>
__device__ __noinline__ int top_slowly(const T* x, int p0, int end, float lmax, int K, TopState& st) {
  constexpr int N = Vec<T>::N;
  const int vecs = (end - p0 + 256 * N - 1) / (256 * N), tid = threadIdx.x, lane = tid & 63;
  const float t = block_kth<0>(lmax, K, st);
  if (tid == 0) st.n_cands = 0;
  __syncthreads();
  for (int v = 0; v < vecs; ++v) add_cands(x, p0, end, v, tid, st, [&](float f) { return f > t; });
  __syncthreads();
  int n = st.n_cands;
  __syncthreads();
  if (n > kCands) {
    uint64_t last = ~0ull;
    for (n = 0; n < K; ++n) {
      uint64_t best = 0;
      for (int v = 0; v < vecs; ++v) {
        const int e = p0 + (v * 256 + tid) * N;
        if (e >= end) break;
        float f[N];
        vec_unpack<T>(vec_ld_tail<T, false>(x, e, end, Vec<T>::kNegInf), f);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const uint64_t k = cand_key(f[j], e + j);
          if (f[j] > -INFINITY && k < last && k > best) best = k;
        }
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        const uint64_t u = __shfl_xor(best, o, 64);
        best = u > best ? u : best;
      }
      if (lane == 0) st.best[tid >> 6] = best;
      __syncthreads();
      best = st.best[0];
      for (int i = 1; i < 4; ++i) best = st.best[i] > best ? st.best[i] : best;
      __syncthreads();
      if (!best) break;
      if (tid == 0) st.cands[n] = best;
      last = best;
    }
    __syncthreads();
    return n;
  }
  int need = t > -INFINITY ? K - n : 0;
  for (int v = 0; v < vecs && need > 0; ++v) {  // uniform
    const int e = p0 + (v * 256 + tid) * N;
    float f[N];
    vec_unpack<T>(vec_ld_tail<T, false>(x, e, end, Vec<T>::kNegInf), f);
    int mine = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) mine += f[j] == t;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(incl, o, 64);
      if (lane >= o) incl += u;
    }
    if (lane == 63) st.keys[tid >> 6] = (uint32_t)incl;
    __syncthreads();
    int before = incl - mine, total = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < (tid >> 6)) before += (int)st.keys[i];
      total += (int)st.keys[i];
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (f[j] == t) {
        if (before < need) st.cands[n + before] = cand_key(f[j], e + j);
        ++before;
      }
    const int took = min(need, total);
    n += took;
    need -= took;
    __syncthreads();
  }
  __syncthreads();
  return n;
}

// A piece of the stream.  (Read once by most: kept out of the caches, which are then not written back for it: a step of
// 4096 rows of 50000 in bf16 with its backward pass 240 -> 222 us, below 200 MB the same.)
template <typename T>
__device__ __forceinline__ void load_piece(const T* row, int t, int p0, int end, u32x4_t* raw) {
  load_part<T, 256, kChunk, 0, true>(row, thread_again(t), p0, end, raw);
}

// A wave's sums over the pieces so far, lane by lane: s = sum 2^(x c - k), t = sum 2^(x c - k) (x c - k), k the whole
// number next to R c.  In 64 bits: a lane of a row of 2^24 columns adds 2048 pieces and more.
struct Running {
  double s = 0., t = 0.;
  float R = 0.f, k = 0.f;
  bool there = false;      // there is a reference
  float far = -INFINITY;   // the largest value met without one that is too far out to be one itself
};

// The piece at `at`, whose sums ps, pt are against a reference that is too low, or none: the wave takes the piece's
// maximum, and what it has so far is brought to that without a rounding.  The piece is read again: kept for this in its
// registers it cost every piece more than this costs the few (4096 rows of 50000 in bf16, top 5: 93 us, read again 88).
// vm: its vectors' maxima, if they are known.
template <typename T, bool ENT>
__device__ __forceinline__ void refer_again(const T* x, int tid, int at, int end, const float* vm, float c, Running& w,
                                            float& ps, float& pt) {
  u32x4_t raw[kChunk];
  load_part<T, 256, kChunk, 0>(x, thread_again(tid), at, end, raw);
  fix_part<T, 256, kChunk, 0>(raw, tid, at, end);
  const float lm = vm ? fmaxf(fmaxf(vm[0], vm[1]), fmaxf(vm[2], vm[3])) : lane_max<T, kChunk>(raw);
  const float m = wave_uniform(wave64_max(lm));
  if (!near_zero(m, c)) {  // (of all masked: ps is 0, or NaN; of +inf and far out with a reference: ps is inf or NaN)
    if (!w.there) w.far = fmaxf(w.far, m);
    return;
  }
  if (w.there && m <= w.R) return;
  const float k = rintf(m * c);
  if (w.there) {
    const double f = ldexp(1., (int)fmaxf(w.k - k, -1000.f));
    if (ENT) w.t = f * (w.t + w.s * (double)(w.k - k));
    w.s *= f;
  } else if ((m - w.far) * c < 160.f) {  // what was far out may count after all
    w.s = NAN;
  }
  w.R = m;
  w.k = k;
  w.there = true;
  ps = pt = 0.f;
  lane_sums<T, 0, kChunk, ENT, true>(raw, 0.f, k, c, ps, pt);
}

// (with alternatives five blocks a CU: the compiler would take the registers of one more; 16384 rows of 9000 in bf16,
// top 20: 127 us, with four 150)
template <typename T, bool ENT, bool TOP>
__global__ void __launch_bounds__(256, TOP ? 5 : 1) vocab_stream_kernel(const VocabArgs a) {
  constexpr int N = Vec<T>::N, STEP = 256 * N * kChunk;
  __shared__ float red[12];
  __shared__ uint64_t top_lds[TOP ? sizeof(TopState) / 8 : 1];
  TopState& top = *reinterpret_cast<TopState*>(top_lds);
  const int items = a.rows * a.nparts;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int row = a.nparts == 1 ? item : item / a.nparts, p0 = (item - row * a.nparts) * a.part_len;
    int64_t tok;
    if (is_padding(a, row, tok)) {
      if (a.nparts == 1) put_padding(a, row);
      continue;
    }
    const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.stride;
    const int end = min(a.V, p0 + a.part_len), tid = thread_again(threadIdx.x);
    u32x4_t raw[kChunk], next[kChunk];
    load_piece<T>(x, tid, p0, end, raw);
    float x_tok = 0.f;
    if (a.nparts == 1 && threadIdx.x == 0) x_tok = token_logit<T>(a, row, tok);
    if (TOP && threadIdx.x == 0) top.n_noted = top.n_cands = 0;  // the first use is behind block_kth's barriers
    // as part_stats: a reference from the wave's first vector, sums of 2^(x c - k)
    Running w;
    float s, t = 0.f, logs, R = wave_uniform(wave64_max(lane_max<T, 1>(raw)));
    if (near_zero(R, a.c)) w.there = true, w.R = R, w.k = rintf(R * a.c);
    float lmax = -INFINITY, thr = -INFINITY;
    for (int piece = 0, at = p0; at < end; at += STEP, ++piece) {
      if (at + STEP < end) load_piece<T>(x, tid, at + STEP, end, next);
      if (at + STEP > end) fix_part<T, 256, kChunk, 0>(raw, tid, at, end);
      float vm[kChunk];
      vm[2] = vm[3] = -INFINITY;
      float ps = 0.f, pt = 0.f;
      lane_sums<T, 0, 2, ENT, true, TOP>(raw, 0.f, w.k, a.c, ps, pt, vm);
      if (at + STEP / 2 < end) lane_sums<T, 2, 4, ENT, true, TOP>(raw, 0.f, w.k, a.c, ps, pt, vm);  // uniform
      if (!w.there || __ballot(!(ps <= kPieceMost<T>))) refer_again<T, ENT>(x, tid, at, end, TOP ? vm : nullptr, a.c, w, ps, pt);
      w.s += ps;
      if (ENT) w.t += pt;
      if (TOP) {
#pragma unroll
        for (int v = 0; v < kChunk; ++v) lmax = fmaxf(lmax, vm[v]);
        // behind pieces 0, 3, 15, ...; the last one's is formed below
        if (piece == 0 || ((piece == 3 || piece == 15) && at + STEP < end)) thr = block_kth<16, true>(lmax, a.K, top);
#pragma unroll
        for (int v = 0; v < kChunk; ++v)
          if (reaches(vm[v], thr)) {
            const int n = atomicAdd(&top.n_noted, 1);
            if (n < kNoted) top.noted[n] = (uint32_t)((piece * kChunk + v) * 256 + tid);
          }
      }
#pragma unroll
      for (int v = 0; v < kChunk; ++v) raw[v] = next[v];
    }
    const float off = __builtin_fmaf(-w.R, a.c, w.k), f = exp2_fast(off);
    R = w.R;
    s = !w.there && w.far > -INFINITY ? NAN : (float)w.s * f;
    if (ENT) t = f * (float)(w.t + w.s * (double)off);
    join_waves<256, ENT>(a.c, red, R, s, t);
    if (!(s < INFINITY)) {  // NaN, +inf or values far out: once more against the maximum, read again
      __syncthreads();
      float m = -INFINITY;
      for (int at = p0; at < end; at += STEP) {
        load_part<T, 256, kChunk, 0>(x, tid, at, end, raw);
        fix_part<T, 256, kChunk, 0>(raw, tid, at, end);
        m = fmaxf(m, lane_max<T, kChunk>(raw));
      }
      R = block_max<256>(m, red);
      w.s = w.t = 0.;
      for (int at = p0; at < end; at += STEP) {
        load_part<T, 256, kChunk, 0>(x, tid, at, end, raw);
        fix_part<T, 256, kChunk, 0>(raw, tid, at, end);
        float ps = 0.f, pt = 0.f;
        lane_sums<T, 0, kChunk, ENT, false>(raw, R, 0.f, a.c, ps, pt);
        w.s += ps;
        if (ENT) w.t += pt;
      }
      s = (float)w.s;
      t = (float)w.t;
      join_waves<256, ENT>(a.c, red, R, s, t);
    }
    if (threadIdx.x == 0) {
      if (a.nparts == 1) put_row(a, row, x_tok, R, s, t, logs);
      else reinterpret_cast<float4*>(a.ws)[item] = make_float4(R, s, t, 0.f);
    }
    if (TOP) {
      if (end - p0 > STEP) thr = block_kth<16, true>(lmax, a.K, top);
      else __syncthreads();
      const int noted = top.n_noted;
      int n = kCands + 1;
      if (noted <= kNoted) {
        for (int i = tid; i < noted; i += 256) {
          const uint32_t w = top.noted[i];
          add_cands(x, p0, end, (int)(w >> 8), (int)(w & 255), top, [&](float f) { return reaches(f, thr); });
        }
        __syncthreads();
        n = top.n_cands;
      }
      if (n > kCands) {  // uniform
        __syncthreads();
        n = top_slowly(x, p0, end, lmax, a.K, top);
      }
      put_list<256>(a, row, item, R, s, top.cands, n);
    }
    __syncthreads();  // red and the lists are the next item's
  }
}

// The parts of each row joined: one block a row.
// Top alternatives: of the first entries of all lists (some 2 K of them, the heads) the K-th best is a threshold.  Keys
// from there on are in at most K lists, so they are at most K * K, and but for odd rows a few more than K.
__host__ __device__ __forceinline__ int heads_of(int nparts, int K) { return min((2 * K + nparts - 1) / nparts, K); }

template <typename T, bool TOP>
__global__ void __launch_bounds__(256) vocab_join_kernel(const VocabArgs a) {
  extern __shared__ uint64_t buf[];  // K * K candidates, then the heads
  __shared__ float red[12];
  __shared__ int count;
  __shared__ uint64_t least;
  const int tid = threadIdx.x;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    int64_t tok;
    if (is_padding(a, row, tok)) {
      put_padding(a, row);
      continue;
    }
    float x_tok = 0.f;
    if (tid == 0) x_tok = token_logit<T>(a, row, tok);
    const float4* ws = reinterpret_cast<const float4*>(a.ws) + (int64_t)row * a.nparts;
    const uint64_t* keys = TOP ? a.ws_keys + (int64_t)row * a.nparts * a.K : nullptr;
    uint64_t* heads = buf + a.K * a.K;
    const int all = a.nparts * a.K, H = TOP ? heads_of(a.nparts, a.K) : 0, nheads = a.nparts * H;
    constexpr int AHEAD = 8;
    uint64_t first[AHEAD];
    if (TOP) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) first[i] = tid + i * 256 < all ? keys[tid + i * 256] : 0;
      for (int i = tid; i < nheads; i += 256) heads[i] = keys[i / H * a.K + i % H];
      if (tid == 0) count = 0, least = 1;  // every key but "nothing there"
    }
    // the reference: that of the parts that hold anything (NaN holds something)
    float m = -INFINITY, s = 0.f, t = 0.f;
    for (int p = tid; p < a.nparts; p += 256) m = ws[p].y == 0.f ? m : fmaxf(m, ws[p].x);
    m = wave64_max(m);
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    m = finite_max(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    for (int p = tid; p < a.nparts; p += 256) join_piece(ws[p].x, ws[p].y, ws[p].z, m, a.c, s, t);
    s = wave64_sum(s);
    t = wave64_sum(t);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = s, red[8 + (tid >> 6)] = t;
    __syncthreads();
    s = red[4] + red[5] + red[6] + red[7];
    t = red[8] + red[9] + red[10] + red[11];
    float logs;
    if (tid == 0) put_row(a, row, x_tok, m, s, t, logs);
    if (TOP) {
      for (int i = tid; i < nheads; i += 256) {
        const uint64_t k = heads[i];
        if (k && keys_above(heads, nheads, k) == a.K - 1) least = k;  // distinct but for 0
      }
      __syncthreads();
      const uint64_t from = least;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (first[i] >= from) buf[atomicAdd(&count, 1)] = first[i];
      for (int i = tid + AHEAD * 256; i < all; i += 256) {
        const uint64_t k = keys[i];
        if (k >= from) buf[atomicAdd(&count, 1)] = k;
      }
      __syncthreads();
      const int n = count;
      const float lg = s == 0.f ? INFINITY : logf(s);
      rank_keys<256>(buf, n, a.K, [&](int r, uint64_t k) { put_top(a, row, r, k, m, lg); });
      for (int k = n + tid; k < a.K; k += 256) {
        a.top_logp[(int64_t)row * a.K + k] = -INFINITY;
        a.top_ids[(int64_t)row * a.K + k] = -1;
      }
    }
    __syncthreads();
  }
}

// The gradient of log probabilities and entropies: every element of x is read and of dx written once.
// g_logp / g_ent may be null (no gradient of that output).
template <typename T, int TPB, int NV, bool ENT>
__global__ void __launch_bounds__(TPB) vocab_bwd_kernel(const VocabArgs a, const float* __restrict__ g_logp,
                                                        const float* __restrict__ g_ent, T* __restrict__ dx) {
  constexpr int N = Vec<T>::N, PART = TPB * NV * N;
  const int items = a.rows * a.nparts;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int row = a.nparts == 1 ? item : item / a.nparts, p0 = (item - row * a.nparts) * PART;
    const int end = min(a.V, p0 + PART), tid = thread_again(threadIdx.x);
    const int64_t tok = whole(a.tok, a.tok64, row);
    T* out = dx + (int64_t)row * a.V;
    const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
    // nothing flows into padding or a row without a token left; a token outside the vocabulary has no gradient
    const bool none = tok < 0 || st.y == 0.f, bad = tok >= a.V;
    if (none || bad) {
      float f[N];
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = tok < 0 || !bad ? 0.f : NAN;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int base = p0 + v * TPB * N;
        if (base < end) vec_st_block(out + base, tid, TPB, end - base, f);
      }
      continue;
    }
    u32x4_t raw[NV];
    load_part<T, TPB, NV, 0>(static_cast<const T*>(a.x) + (int64_t)row * a.stride, tid, p0, end, raw);
    fix_part<T, TPB, NV, 0>(raw, tid, p0, end);
    const float g = (g_logp ? g_logp[row] : 0.f) * a.scale, h = ENT ? g_ent[row] * a.scale : 0.f;
    // -[g + h (log p + H)] p = (A + B d) 2^d, with log p = ln2 d - log s
    const float A = -(g + h * (st.w - st.z)) * st.y, B = -h * kLn2 * st.y;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int base = p0 + v * TPB * N;
      float f[N];
      vec_unpack_again<T>(raw[v], f);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = (f[j] - st.x) * a.c, p = exp2_fast(d);
        f[j] = ENT ? (A + B * fmaxf(d, kLow)) * p : A * p;
        if (base + tid * N + j == (int)tok) f[j] += g;
      }
      if (base < end) vec_st_block(out + base, tid, TPB, end - base, f);
    }
  }
}

// ---------------------------------------------------------------- distillation
namespace {

// (The loops over a list are not unrolled: the row is in registers meanwhile, and what they took is taken from the
// blocks that fit a CU.)
// A row's teacher list in LDS, K rounded up to Kp, a multiple of 4
struct Teacher {
  float *q, *logq, *x;  // probabilities, their logs, the student's logits at the ids
  int* ids;             // -1: nothing there
};
__device__ __forceinline__ Teacher teacher_lds(float* lds, int Kp) {
  return {lds, lds + Kp, lds + 2 * Kp, reinterpret_cast<int*>(lds + 3 * Kp)};
}

// The list's ids, logits (in logq) and the student's logits at them, by all threads.  bad / any: set where an id
// lies outside the vocabulary / where there is one.
template <typename T>
__device__ __forceinline__ void teacher_load(const DistillArgs& a, int row, const T* x, int Kp, Teacher l) {
#pragma unroll 1
  for (int k = threadIdx.x; k < Kp; k += blockDim.x) {
    int64_t id = -1;
    float t = -INFINITY;
    if (k < a.K) {
      const int64_t at = (int64_t)row * a.K + k;
      id = whole(a.ids, a.ids64, at);
      t = a.teacher_bf16 ? bf16_to_f32(static_cast<const uint16_t*>(a.teacher)[at])
                         : static_cast<const float*>(a.teacher)[at];
    }
    const bool in = id >= 0 && id < a.v.V;
    l.ids[k] = in ? (int)id : id < 0 ? -1 : -2;
    l.logq[k] = id < 0 ? -INFINITY : t;
    l.x[k] = in ? elem_f32(x[id]) : 0.f;
  }
}

// q and log q from the list's logits, by the first wave (its lanes read what they write).  Returns 0: nothing to
// learn, 1: a list, 2: an id outside the vocabulary.
__device__ __forceinline__ int teacher_softmax(const DistillArgs& a, int Kp, Teacher l) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY, s = 0.f;
  bool bad = false;
#pragma unroll 1
  for (int k = lane; k < Kp; k += 64) {
    m = fmaxf(m, l.logq[k]);
    bad |= l.ids[k] == -2;
  }
  m = finite_max(wave64_max(m));
#pragma unroll 1
  for (int k = lane; k < Kp; k += 64) s += exp2_fast((l.logq[k] - m) * a.v.c);
  s = wave64_sum(s);
  const float inv = s == 0.f ? 0.f : 1.f / s, ls = logf(s);
#pragma unroll 1
  for (int k = lane; k < Kp; k += 64) {
    const float t = l.logq[k];
    l.q[k] = l.ids[k] < 0 ? 0.f : exp2_fast((t - m) * a.v.c) * inv;
    l.logq[k] = (t - m) * a.v.scale - ls;
  }
  return __ballot(bad) != 0 ? 2 : s != 0.f ? 1 : 0;
}

// sum_k q_k (log q_k - log p_{id_k}), in every lane of the first wave
__device__ __forceinline__ float row_kl(const DistillArgs& a, int Kp, Teacher l, float R, float logs, bool empty) {
  float kl = 0.f;
#pragma unroll 1
  for (int k = threadIdx.x & 63; k < Kp; k += 64) {
    const float qk = l.q[k];
    if (qk == 0.f) continue;  // NaN is not 0: it reaches the loss
    const float lp = empty ? -INFINITY : __builtin_fmaf(l.x[k] - R, a.v.scale, -logs);
    kl += qk * (l.logq[k] - lp);
  }
  return wave64_sum(kl);
}

// What entry k takes off the gradient at its token: the first of equal ids takes the probabilities of all, added
// in their order, the others (and empty entries) nothing: -1.
__device__ __forceinline__ float token_share(const Teacher& l, int Kp, int k) {
  const int id = l.ids[k];
  if (id < 0) return -1.f;
  float sum = 0.f;
  int first = Kp;
  const int4* ids = reinterpret_cast<const int4*>(l.ids);
  const float4* q = reinterpret_cast<const float4*>(l.q);
#pragma unroll 1
  for (int j = 0; j < Kp / 4; ++j) {
    const int4 i = ids[j];
    const float4 p = q[j];
    if (i.w == id) first = min(first, 4 * j + 3);
    if (i.z == id) first = min(first, 4 * j + 2);
    if (i.y == id) first = min(first, 4 * j + 1);
    if (i.x == id) first = min(first, 4 * j);
    sum += i.x == id ? p.x : 0.f;
    sum += i.y == id ? p.y : 0.f;
    sum += i.z == id ? p.z : 0.f;
    sum += i.w == id ? p.w : 0.f;
  }
  return first == k ? sum : -1.f;  // a NaN probability is kept: it is not below 0
}

}  // namespace

// Loss and gradient in one pass: the whole row is in the block's registers.  loss_rows[row] = w T^2 KL.
// AHEAD: one block fills the CU (1024 threads of up to 128 registers); it walks over the rows, and each vector's
// registers take the next row's load as soon as its gradient is stored, or memory would idle while it computes.
template <typename T, int TPB, int NV, bool AHEAD>
__global__ void __launch_bounds__(TPB) distill_fused_kernel(const DistillArgs a, T* __restrict__ dx) {
  constexpr int N = Vec<T>::N;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ float red[3 * (TPB / 64)];
  __shared__ int state;
  const int V = a.v.V, Kp = (a.K + 3) & ~3;
  const Teacher l = teacher_lds(lds, Kp);
  const T* base = static_cast<const T*>(a.v.x);
  u32x4_t raw[NV];
  if (AHEAD && blockIdx.x < a.v.rows) load_part<T, TPB, NV, sure_vectors(NV)>(base + (int64_t)blockIdx.x * a.v.stride, threadIdx.x, 0, V, raw);
  for (int row = blockIdx.x; row < a.v.rows; row += gridDim.x) {
    const float w = a.v.weight ? a.v.weight[row] : a.w;
    const T* x = base + (int64_t)row * a.v.stride;
    T* out = dx + (int64_t)row * V;
    const int tid = thread_again(threadIdx.x);
    int st = 0;
    float coef = 0.f, R = 0.f, inv = 0.f, loss = 0.f;
    if (w != 0.f) {
      if (!AHEAD) load_part<T, TPB, NV, sure_vectors(NV)>(x, tid, 0, V, raw);
      teacher_load(a, row, x, Kp, l);
      __syncthreads();
      if (threadIdx.x < 64) {
        st = teacher_softmax(a, Kp, l);
        if (threadIdx.x == 0) state = st;
      }
      float s, t;
      part_stats<T, TPB, NV, false>(raw, tid, V, a.v.c, red, R, s, t);
      if (TPB == 64) __syncthreads();
      st = state;  // behind a barrier of part_stats
      const bool empty = s == 0.f;
      inv = empty ? 0.f : 1.f / s;
      coef = st == 2 ? NAN : st == 0 || empty ? 0.f : w * a.temp;
      if (threadIdx.x < 64) loss = st == 1 ? w * a.temp * a.temp * row_kl(a, Kp, l, R, logf(s), empty) : coef;
    } else if (!AHEAD) {
#pragma unroll
      for (int v = 0; v < NV; ++v) raw[v] = u32x4_t{0u, 0u, 0u, 0u};  // not the last row's: its registers end there
    }
    if (threadIdx.x == 0) a.loss_rows[row] = loss;
    const bool dense = coef != 0.f && coef == coef;  // uniform
    const float ci = coef * inv;
    const T* next = row + gridDim.x < (unsigned)a.v.rows ? x + (int64_t)gridDim.x * a.v.stride : nullptr;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[N];
      if (dense) {
        vec_unpack_again<T>(raw[v], f);
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = ci * exp2_fast((f[j] - R) * a.v.c);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = coef;
      }
      if (v * TPB * N < V) vec_st_block(out + v * TPB * N, tid, TPB, V - v * TPB * N, f);
      if (AHEAD && next)
        raw[v] = v < sure_vectors(NV) ? vec_ld(next + v * TPB * N, (uint32_t)(tid * N))
                                      : vec_ld_near<T>(next, (v * TPB + tid) * N, V, Vec<T>::kNegInf);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (dense) {
      // at the teacher's tokens, over what the dense pass wrote
      __syncthreads();
      for (int k = threadIdx.x; k < Kp; k += TPB) {
        const float q = token_share(l, Kp, k);
        if (!(q < 0.f)) elem_st(out + l.ids[k], coef * (exp2_fast((l.x[k] - R) * a.v.c) * inv - q));
      }
    }
    __syncthreads();  // the list's place is the next row's
  }
}

// Row losses, probabilities q [rows, K] and gradient factors (w T; 0: no gradient, NaN: a bad id) from the
// rows' statistics: one wave a row.
template <typename T>
__global__ void __launch_bounds__(64) distill_loss_kernel(const DistillArgs a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int Kp = (a.K + 3) & ~3;
  const Teacher l = teacher_lds(lds, Kp);
  for (int row = blockIdx.x; row < a.v.rows; row += gridDim.x) {
    const float w = a.v.weight ? a.v.weight[row] : a.w;
    float loss = 0.f, coef = 0.f;
    if (w != 0.f) {
      teacher_load(a, row, static_cast<const T*>(a.v.x) + (int64_t)row * a.v.stride, Kp, l);
      __syncthreads();
      const int st = teacher_softmax(a, Kp, l);
      const float4 r = reinterpret_cast<const float4*>(a.v.stats)[row];  // R, 1 / s, log s, -
      const bool empty = r.y == 0.f;
      coef = st == 2 ? NAN : st == 0 || empty ? 0.f : w * a.temp;
      loss = st == 1 ? w * a.temp * a.temp * row_kl(a, Kp, l, r.x, r.z, empty) : coef;
    }
    if (a.q)
      for (int k = threadIdx.x; k < a.K; k += 64) a.q[(int64_t)row * a.K + k] = coef == 0.f ? 0.f : l.q[k];
    if (threadIdx.x == 0) {
      a.loss_rows[row] = loss;
      if (a.coef) a.coef[row] = coef;
    }
    __syncthreads();
  }
}

// The gradient from the saved statistics, factors and probabilities, times the upstream scalar g
template <typename T, int TPB, int NV>
__global__ void __launch_bounds__(TPB) distill_bwd_kernel(const DistillArgs a, const float* __restrict__ g,
                                                          T* __restrict__ dx) {
  constexpr int N = Vec<T>::N, PART = TPB * NV * N;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int Kp = (a.K + 3) & ~3;
  const Teacher l = teacher_lds(lds, Kp);
  const int items = a.v.rows * a.v.nparts;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int row = a.v.nparts == 1 ? item : item / a.v.nparts, p0 = (item - row * a.v.nparts) * PART;
    const int end = min(a.v.V, p0 + PART), tid = thread_again(threadIdx.x);
    const T* x = static_cast<const T*>(a.v.x) + (int64_t)row * a.v.stride;
    T* out = dx + (int64_t)row * a.v.V;
    const float own = a.coef[row], coef = own == 0.f ? 0.f : own * g[0];
    if (own == 0.f || coef != coef) {
      float f[N];
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = coef;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int base = p0 + v * TPB * N;
        if (base < end) vec_st_block(out + base, tid, TPB, end - base, f);
      }
      continue;
    }
    u32x4_t raw[NV];
    load_part<T, TPB, NV, 0>(x, tid, p0, end, raw);
    for (int k = threadIdx.x; k < Kp; k += TPB) {
      const int64_t at = (int64_t)row * a.K + k;
      l.q[k] = k < a.K ? a.q[at] : 0.f;
      l.ids[k] = k < a.K ? (int)max((int64_t)-1, whole(a.ids, a.ids64, at)) : -1;
    }
    const float4 st = reinterpret_cast<const float4*>(a.v.stats)[row];
    fix_part<T, TPB, NV, 0>(raw, tid, p0, end);
    const float ci = coef * st.y;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int base = p0 + v * TPB * N;
      float f[N];
      vec_unpack_again<T>(raw[v], f);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = ci * exp2_fast((f[j] - st.x) * a.v.c);
      if (base < end) vec_st_block(out + base, tid, TPB, end - base, f);
    }
    __syncthreads();  // the list is there, and the dense stores are in front of those below
    for (int k = threadIdx.x; k < Kp; k += TPB) {
      const int id = l.ids[k];
      if (id < p0 || id >= end) continue;
      const float q = token_share(l, Kp, k);
      if (!(q < 0.f)) elem_st(out + id, coef * (exp2_fast((elem_f32(x[id]) - st.x) * a.v.c) * st.y - q));
    }
    __syncthreads();
  }
}

// loss = sum of the rows' losses, in one order and 64 bits
__global__ void __launch_bounds__(1024) rows_sum_kernel(const float* __restrict__ r, int n, float* __restrict__ out) {
  __shared__ double part[16];
  double s = 0.;
  int i = threadIdx.x;
  for (; i + 7 * 1024 < n; i += 8 * 1024) {  // eight loads in flight
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = r[i + 1024 * j];
#pragma unroll
    for (int j = 0; j < 8; ++j) s += (double)v[j];
  }
  float v[7];
#pragma unroll
  for (int j = 0; j < 7; ++j) v[j] = i + 1024 * j < n ? r[i + 1024 * j] : 0.f;
#pragma unroll
  for (int j = 0; j < 7; ++j) s += (double)v[j];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  s = threadIdx.x < 16 ? part[threadIdx.x] : 0.;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (threadIdx.x == 0) out[0] = (float)s;
}

// x *= g[0], unless that is exactly 1 (then nothing is read or written); x is 16-byte aligned
template <typename T>
__global__ void __launch_bounds__(1024) scale_unless_one_kernel(T* __restrict__ x, int64_t n,
                                                                const float* __restrict__ g) {
  constexpr int N = Vec<T>::N;
  const float s = g[0];
  if (s == 1.f) return;
  for (int64_t i = ((int64_t)blockIdx.x * 1024 + threadIdx.x) * N; i < n; i += (int64_t)gridDim.x * 1024 * N) {
    if (i + N <= n) {
      float f[N];
      vec_unpack<T>(vec_ld(x + i), f);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] *= s;
      vec_st(x + i, 0, f);
    } else {
      for (int64_t k = i; k < n; ++k) elem_st(x + k, elem_f32(x[k]) * s);
    }
  }
}

// ---------------------------------------------------------------- host
namespace {

constexpr int kMaxGrid = 1 << 20;
int grid_of(int64_t items) { return (int)std::min<int64_t>(items, kMaxGrid); }

// threads, vectors a thread, parts of a row and their length
struct Shape {
  int tpb, nv, nparts, len;
};

// Rows that one wave's registers hold take one wave each: up to 16 vectors a lane (16384 rows in bf16 of 3000: 22 us,
// streamed by blocks 41; of 5000: 31 and 48; of 8000: 49 and 53; 256 rows of 5000: 5.1 and, in parts, 7.1).  With top
// alternatives a wave is on its own for longer, which takes rows enough to hide it: for up to kFewTop of them 16384 rows
// in bf16 of 8000, top 5: 69 us, streamed 87; 256 rows of 4096: 8.0 and 6.5; for more of them 16384 rows of 6000, top 20:
// 85 and 96, of 8000 107 and 100; 2000 rows of 5000 17.1 and 16.9; 256 rows of 3000 9.7 and 7.7.
// Longer rows take a block, in parts where the list of their alternatives asks for it (kTopVecs) or rows are so few that
// there would be less than kFewParts blocks.
constexpr int kFewParts = 512;

template <typename T>
Shape stats_shape(int64_t rows, int64_t V, int K) {
  constexpr int N = Vec<T>::N;
  const int most_nv = !K ? 16 : K <= kFewTop ? (rows >= 1024 ? 16 : 8) : rows >= 4096 ? 12 : rows >= 1024 ? 8 : 4;
  for (int nv = 1; nv <= most_nv; nv += nv < 8 ? nv : 2)
    if (V <= 64 * N * nv) return {64, nv, 1, (int)V};
  const int64_t vecs = (V + 256 * N - 1) / (256 * N), most = K ? kTopVecs : vecs;
  int64_t parts = std::max((vecs + most - 1) / most, std::min((vecs + 1) / 2, (kFewParts + rows - 1) / rows));
  const int64_t per = (vecs + parts - 1) / parts;
  parts = (vecs + per - 1) / per;
  return {256, 0, (int)parts, (int)std::min<int64_t>(per * 256 * N, V)};
}

template <typename T, bool ENT, bool TOP>
void stats_launch(const VocabArgs& a, Shape s, hipStream_t st) {
  const int grid = grid_of((int64_t)a.rows * a.nparts);
  if (s.tpb == 64) {
#define GO(NV)                                                                                              \
  if (s.nv == NV)                                                                                           \
    launch(vocab_stats_kernel<T, NV, ENT, TOP>, grid, 64, TOP ? (size_t)top_room<T, NV>(a.K) * 8 : 0, st, a)
    GO(1); GO(2); GO(4); GO(8);
    GO(10); GO(12); GO(14); GO(16);
#undef GO
    return;
  }
  launch(vocab_stream_kernel<T, ENT, TOP>, grid, 256, 0, st, a);
  if (a.nparts == 1) return;
  const size_t jl = TOP ? ((size_t)a.K * a.K + (size_t)a.nparts * heads_of(a.nparts, a.K)) * 8 : 0;
  launch(vocab_join_kernel<T, TOP>, grid_of(a.rows), 256, jl, st, a);
}

template <typename T>
void stats_all(VocabArgs& a, hipStream_t st) {
  const Shape s = stats_shape<T>(a.rows, a.V, a.K);
  a.part_len = s.len;
  const bool ent = a.ent != nullptr;
  if (a.K > 0) {
    if (ent) stats_launch<T, true, true>(a, s, st);
    else stats_launch<T, false, true>(a, s, st);
  } else {
    if (ent) stats_launch<T, true, false>(a, s, st);
    else stats_launch<T, false, false>(a, s, st);
  }
}

// the dense gradient passes (their reads and writes need no join): a wave a row where it holds it
template <typename T>
Shape bwd_shape(int64_t V) {
  constexpr int N = Vec<T>::N;
  for (int nv = 1; nv <= 4; nv *= 2)
    if (V <= 64 * N * nv) return {64, nv, 1, (int)V};
  const int len = 256 * N * 4;
  return {256, 4, (int)((V + len - 1) / len), len};
}

// The fewest threads that hold the row in 64 registers each, in few of them: 16 vectors a thread take 119 registers
// and 4 blocks of 256 fit a CU, 10 take 89 and 5 do (1500 rows of 50003 in bf16: 512 x 16 72 us, 512 x 14 69; 2048 rows of
// 10000 in f32: 256 x 16 37 us, 256 x 10 34).  A wave alone pays for up to 10 vectors a lane where rows are many
// (16384 rows in bf16 of 3000: 64 x 8 44 us, 256 x 2 56; of 5000: 64 x 10 68, 256 x 4 78; of 7000: 64 x 14 97, 256 x 4
// 90; 256 rows of 3000: 8.4 and 6.9).
template <typename T>
Shape fused_shape(int64_t rows, int64_t V) {
  constexpr int N = Vec<T>::N;
  for (int nv = 1; nv <= (rows >= 1024 ? 10 : 4); nv += nv < 8 ? nv : 2)
    if (V <= 64 * N * nv) return {64, nv, 1, (int)V};
  for (int nv = 2; nv <= 16; nv += nv < 8 ? nv : 2)
    if (V <= 256 * N * nv) return {256, nv, 1, (int)V};
  for (int tpb = 512; tpb <= 1024; tpb *= 2)
    for (int nv = 10; nv <= 16; nv += 2)
      if (V <= tpb * N * nv) return {tpb, nv, 1, (int)V};
  return {0, 0, 0, 0};
}

template <typename T, int TPB, int NV>
void fused_go(const DistillArgs& a, T* dx, hipStream_t st) {
  constexpr bool AHEAD = TPB == 1024;
  const int grid = std::min(grid_of(a.v.rows), AHEAD ? 256 : kMaxGrid);
  launch(distill_fused_kernel<T, TPB, NV, AHEAD>, grid, TPB, (size_t)((a.K + 3) & ~3) * 16, st, a, dx);
}

template <typename T>
void fused_launch(const DistillArgs& a, void* dx, hipStream_t st) {
  const Shape s = fused_shape<T>(a.v.rows, a.v.V);
  T* d = static_cast<T*>(dx);
#define GO(TPB, NV) \
  if (s.tpb == TPB && s.nv == NV) return fused_go<T, TPB, NV>(a, d, st)
  GO(64, 1); GO(64, 2); GO(64, 4); GO(64, 8); GO(64, 10);
  GO(256, 2); GO(256, 4); GO(256, 8); GO(256, 10); GO(256, 12); GO(256, 14); GO(256, 16);
  GO(512, 10); GO(512, 12); GO(512, 14); GO(512, 16);
  GO(1024, 10); GO(1024, 12); GO(1024, 14); GO(1024, 16);
#undef GO
}

template <typename T>
void vocab_bwd_launch(VocabArgs a, const float* g_logp, const float* g_ent, void* dx, hipStream_t st) {
  const Shape s = bwd_shape<T>(a.V);
  a.nparts = s.nparts;
  const int grid = grid_of((int64_t)a.rows * a.nparts);
  T* d = static_cast<T*>(dx);
#define GO(TPB, NV)                                                                                       \
  do {                                                                                                    \
    if (g_ent) launch(vocab_bwd_kernel<T, TPB, NV, true>, grid, TPB, 0, st, a, g_logp, g_ent, d);             \
    else launch(vocab_bwd_kernel<T, TPB, NV, false>, grid, TPB, 0, st, a, g_logp, g_ent, d);                  \
  } while (0)
  if (s.tpb == 256) GO(256, 4);
  else if (s.nv == 1) GO(64, 1);
  else if (s.nv == 2) GO(64, 2);
  else GO(64, 4);
#undef GO
}

template <typename T>
void distill_bwd_launch(DistillArgs a, const float* g, void* dx, hipStream_t st) {
  const Shape s = bwd_shape<T>(a.v.V);
  a.v.nparts = s.nparts;
  const int grid = grid_of((int64_t)a.v.rows * a.v.nparts);
  const size_t lds = (size_t)((a.K + 3) & ~3) * 16;
  T* d = static_cast<T*>(dx);
#define GO(TPB, NV) launch(distill_bwd_kernel<T, TPB, NV>, grid, TPB, lds, st, a, g, d)
  if (s.tpb == 256) GO(256, 4);
  else if (s.nv == 1) GO(64, 1);
  else if (s.nv == 2) GO(64, 2);
  else GO(64, 4);
#undef GO
}

}  // namespace

int vocab_parts(bool bf16, int64_t rows, int64_t V, int K) {
  return (bf16 ? stats_shape<uint16_t>(rows, V, K) : stats_shape<float>(rows, V, K)).nparts;
}

void vocab_stats(VocabArgs a, hipStream_t st) {
  a.bf16 ? stats_all<uint16_t>(a, st) : stats_all<float>(a, st);
}

void vocab_bwd(const VocabArgs& a, const float* g_logp, const float* g_ent, void* dx, hipStream_t st) {
  a.bf16 ? vocab_bwd_launch<uint16_t>(a, g_logp, g_ent, dx, st) : vocab_bwd_launch<float>(a, g_logp, g_ent, dx, st);
}

bool distill_fits(bool bf16, int64_t V) {
  return (bf16 ? fused_shape<uint16_t>(1, V) : fused_shape<float>(1, V)).tpb != 0;
}

void distill_fused(const DistillArgs& a, void* dx, float* loss, hipStream_t st) {
  a.v.bf16 ? fused_launch<uint16_t>(a, dx, st) : fused_launch<float>(a, dx, st);
  launch(rows_sum_kernel, 1, 1024, 0, st, a.loss_rows, a.v.rows, loss);
}

void distill_loss(const DistillArgs& a, float* loss, hipStream_t st) {
  const int grid = grid_of(a.v.rows);
  const size_t lds = (size_t)((a.K + 3) & ~3) * 16;
  if (a.v.bf16) launch(distill_loss_kernel<uint16_t>, grid, 64, lds, st, a);
  else launch(distill_loss_kernel<float>, grid, 64, lds, st, a);
  launch(rows_sum_kernel, 1, 1024, 0, st, a.loss_rows, a.v.rows, loss);
}

void distill_bwd(const DistillArgs& a, const float* g, void* dx, hipStream_t st) {
  a.v.bf16 ? distill_bwd_launch<uint16_t>(a, g, dx, st) : distill_bwd_launch<float>(a, g, dx, st);
}

void scale_unless_one(void* x, bool bf16, int64_t n, const float* g, hipStream_t st) {
  // two blocks a CU: mostly they read one number and end, in 2 us
  const int64_t per = (int64_t)1024 * (bf16 ? 8 : 4);
  const int grid = (int)std::min<int64_t>(512, (n + per - 1) / per);
  if (bf16) launch(scale_unless_one_kernel<uint16_t>, grid, 1024, 0, st, static_cast<uint16_t*>(x), n, g);
  else launch(scale_unless_one_kernel<float>, grid, 1024, 0, st, static_cast<float*>(x), n, g);
}

}  // namespace tfx
