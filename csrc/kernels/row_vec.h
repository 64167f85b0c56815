// Rows of any width, alignment and row stride read as 16-byte vectors.
//
// A row of a [rows, width] matrix starts at any element address (odd widths, slices of a wider
// matrix), so a vector load here is a 16-byte load with the alignment of one element: gfx950's
// global loads take any address, and a misaligned one costs no more than the extra cache line it
// touches.  The last vector of a row is read as the row's last 16 bytes and shifted into place when it is
// used (vec_ld_near, vec_fix): one load like all others, with no per-element loads and no branch around it.
#pragma once
#include <stdexcept>
#include <tuple>

#include "tfx_common.h"

namespace tfx {

// A launch that says itself whether the runtime took it.  (What hipGetLastError holds behind <<<>>> may be the error of an
// earlier call of another's, which is its owner's to take.)
template <typename... P, typename... A>
void launch(void (*kernel)(P...), dim3 grid, int threads, size_t lds, hipStream_t s, A... args) {
  std::tuple<P...> held(args...);
  const hipError_t e = std::apply(
      [&](auto&... v) {
        void* at[] = {const_cast<void*>(static_cast<const void*>(&v))...};
        return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(threads), at, lds, s);
      },
      held);
  if (e == hipSuccess) return;
  (void)hipGetLastError();  // this launch's
  throw std::runtime_error(hipGetErrorString(e));
}

template <typename T>
struct Vec;  // elements of a 16-byte vector
template <>
struct Vec<float> {
  static constexpr int N = 4;
  typedef uint32_t raw __attribute__((ext_vector_type(4), aligned(4)));
  static constexpr uint32_t kNegInf = 0xff800000u;  // -inf in every element of a word
};
template <>
struct Vec<uint16_t> {  // bf16
  static constexpr int N = 8;
  typedef uint32_t raw __attribute__((ext_vector_type(4), aligned(2)));
  static constexpr uint32_t kNegInf = 0xff80ff80u;
};

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// Elements e ... of `p`.  A uniform p and a 32-bit offset are one scalar and one vector register of the load;
// added up in 64 bits they would be two vector registers for each vector of a row.
// ONCE: the line is not kept in the caches for a later reader.
template <typename T, bool ONCE = false>
__device__ __forceinline__ u32x4_t vec_ld(const T* p, uint32_t e = 0) {
  const auto* at = reinterpret_cast<const typename Vec<T>::raw*>(reinterpret_cast<const char*>(p) + (uint32_t)(e * sizeof(T)));
  return ONCE ? __builtin_nontemporal_load(at) : *at;
}

__device__ __forceinline__ float elem_f32(float v) { return v; }
__device__ __forceinline__ float elem_f32(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ void elem_st(float* p, float v) { *p = v; }
__device__ __forceinline__ void elem_st(uint16_t* p, float v) { *p = f32_to_bf16(v); }

// Elements e .. e+N-1 of a row that ends at `end` (e may lie past it), in two steps.  vec_ld_near loads, with no branch
// and nothing done to what it loaded, so that it can be in flight long before it is used: 16 bytes at e, or the row's
// last 16 where those would leave the row.  vec_fix moves these into place, with `fill` at and behind the end; vectors
// that end inside the row it leaves as they are.  e is a multiple of N.  ONCE as in vec_ld.
// SHORT: the row may be shorter than one vector; then vec_ld_near gathers it.
template <typename T, bool SHORT = false, bool ONCE = false>
__device__ __forceinline__ u32x4_t vec_ld_near(const T* row, int e, int end, uint32_t fill) {
  constexpr int N = Vec<T>::N;
  if (!SHORT || end >= N) return vec_ld<T, ONCE>(row, (uint32_t)min(e, end - N));
  u32x4_t v = {fill, fill, fill, fill};
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (e + j >= end) continue;
    if constexpr (sizeof(T) == 2) {
      const uint32_t b = row[e + j];
      v[j >> 1] = (j & 1) ? ((v[j >> 1] & 0xffffu) | (b << 16)) : ((v[j >> 1] & 0xffff0000u) | b);
    } else {
      v[j] = __float_as_uint(row[e + j]);
    }
  }
  return v;
}

template <typename T, bool SHORT = false>
__device__ __forceinline__ u32x4_t vec_fix(u32x4_t v, int e, int end, uint32_t fill) {
  constexpr int N = Vec<T>::N;
  if (SHORT && end < N) return v;
  if (end % N == 0) {  // uniform: a vector is whole or past the end
    if (e >= end) v = u32x4_t{fill, fill, fill, fill};
    return v;
  }
  int sh = e - min(e, end - N);  // elements to drop at the front
  if (sizeof(T) == 2) {
    const uint32_t bits = (sh & 1) * 16;
    const u32x4_t w = v;
    v.x = __builtin_amdgcn_alignbit(w.y, w.x, bits);
    v.y = __builtin_amdgcn_alignbit(w.z, w.y, bits);
    v.z = __builtin_amdgcn_alignbit(w.w, w.z, bits);
    v.w = __builtin_amdgcn_alignbit(fill, w.w, bits);
    sh >>= 1;
  }
  if (sh & 1) v = u32x4_t{v.y, v.z, v.w, fill};
  if (sh & 2) v = u32x4_t{v.z, v.w, fill, fill};
  if (sh >= 4) v = u32x4_t{fill, fill, fill, fill};
  return v;
}

// both at once
template <typename T, bool SHORT = false>
__device__ __forceinline__ u32x4_t vec_ld_tail(const T* row, int e, int end, uint32_t fill) {
  return vec_fix<T, SHORT>(vec_ld_near<T, SHORT>(row, e, end, fill), e, end, fill);
}

template <typename T>
__device__ __forceinline__ void vec_unpack(u32x4_t v, float* f) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(v[i] << 16);
      f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
  }
}

// ... from the packed words, not from what an earlier pass over them unpacked: the compiler would keep every f32 of
// that alive, twice the registers of a bf16 row
template <typename T>
__device__ __forceinline__ void vec_unpack_again(u32x4_t& v, float* f) {
  asm volatile("" : "+v"(v));
  vec_unpack<T>(v, f);
}

// ... and in a branch: v itself stays one value on both of its sides
template <typename T>
__device__ __forceinline__ void vec_unpack_aside(u32x4_t v, float* f) {
  vec_unpack_again<T>(v, f);
}

template <typename T>
__device__ __forceinline__ void vec_st(T* p, uint32_t e, const float* f) {
  typename Vec<T>::raw r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) r[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    else r[i] = __float_as_uint(f[i]);
  }
  *reinterpret_cast<typename Vec<T>::raw*>(reinterpret_cast<char*>(p) + (uint32_t)(e * sizeof(T))) = r;
}
// Elements t * N ... of the next threads * N elements at p, those in front of `left` only
template <typename T>
__device__ __forceinline__ void vec_st_block(T* p, int t, int threads, int left, const float* f) {
  constexpr int N = Vec<T>::N;
  if (left >= threads * N || (t + 1) * N <= left) {  // the first uniform
    vec_st(p, (uint32_t)(t * N), f);
    return;
  }
  if (left % N == 0 || t * N >= left) return;
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (t * N + j < left) elem_st(p + t * N + j, f[j]);
}

// The thread's number anew: what is computed from it stays inside the loop that it is used in.  Hoisted out of a
// loop over rows, the offsets and bounds of all vectors of a row would take more registers than the row.
__device__ __forceinline__ int thread_again(int t) {
  asm volatile("" : "+v"(t));
  return t;
}

// Over each L lanes (8, 16, 32 or 64), the result in all of them: DPP steps inside 16, the LDS crossbar beyond.
// Groups may be inactive, as a whole.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp_f<0xB1>(v);
  v += dpp_f<0x4E>(v);
  v += dpp_f<0x141>(v);
  if (L >= 16) v += dpp_f<0x140>(v);
  if (L >= 32) v += __shfl_xor(v, 16, 64);
  if (L >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
  v = fmaxf(v, dpp_f<0xB1>(v));
  v = fmaxf(v, dpp_f<0x4E>(v));
  v = fmaxf(v, dpp_f<0x141>(v));
  if (L >= 16) v = fmaxf(v, dpp_f<0x140>(v));
  if (L >= 32) v = fmaxf(v, __shfl_xor(v, 16, 64));
  if (L >= 64) v = fmaxf(v, __shfl_xor(v, 32, 64));
  return v;
}
__device__ __forceinline__ float wave64_sum(float v) { return lanes_sum<64>(v); }
__device__ __forceinline__ float wave64_max(float v) { return lanes_max<64>(v); }

}  // namespace tfx
