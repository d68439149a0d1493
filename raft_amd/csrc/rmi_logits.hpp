// Building blocks of the operators over rows of logits (rmi_top_k, rmi_distill_*, rmi_sample):
// rank order as integer keys, sums over a workgroup, sweeps over one row, and the cut of a row
// in rank order by count or by mass.
#pragma once

#include <type_traits>

#include "rmi_device.hpp"

namespace rmi {
namespace logits {

constexpr float kInf   = __builtin_inff();
constexpr double kLn2  = 0.693147180559945309417232121458;
constexpr double kLog2e = 1.44269504088896340735992468100;

// Temperatures a call accepts: wide enough for every use, narrow enough that 1 / T and the
// products with it are normal fp32 numbers.
constexpr double kMinTemperature = 1e-6;
constexpr double kMaxTemperature = 1e6;

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline bool is_logits_dtype(int d) { return d == RMI_F16 || d == RMI_BF16 || d == RMI_F32; }
inline int bad_dtype(int d)
{
  return d >= 0 && d < RMI_DTYPE_COUNT_ ? RMI_ERR_UNSUPPORTED : RMI_ERR_BAD_ENUM;
}
// Shape rules shared by the entry points: indices are 32 bits, one workgroup row each.
inline int check_shape(int64_t n_rows, int64_t n_cols, int64_t ld)
{
  if (n_rows < 0 || n_cols < 0 || n_cols > INT32_MAX - 65536 || n_rows > INT32_MAX) return RMI_ERR_BAD_SHAPE;
  if (n_rows > 1 && ld < n_cols) return RMI_ERR_BAD_SHAPE;
  return RMI_OK;
}

// ---- elements ---------------------------------------------------------------------------------

// 16 bytes at any element's address, cached: rows are swept more than once.
__device__ __forceinline__ u32x4 load16c(const void* p)
{
  return *reinterpret_cast<const u32x4_unaligned*>(p);
}

template <class T>
__device__ __forceinline__ float widen(const T* p)
{
  return (float)In<T>::ld(p);
}

// Rank order as an unsigned number: larger value, larger key; -0 and +0 share a key; NaN is 0,
// behind -inf.  Only the bits that tell values of the type apart are kept (bf16: the upper 16 of
// fp32, fp16: 19), so a search over keys has no more steps than it needs.
template <class T>
constexpr int kKeyBits = 32;
template <>
inline constexpr int kKeyBits<bf16_t> = 16;
template <>
inline constexpr int kKeyBits<f16_t> = 19;

template <class T>
__device__ __forceinline__ u32 key_of(float x)
{
  const u32 b = as_u32(x + 0.0f);
  const u32 k = (b >> 31) ? ~b : b | 0x80000000u;
  return x == x ? k >> (32 - kKeyBits<T>) : 0u;
}
// The value of a key, where it is not NaN's.
template <class T>
__device__ __forceinline__ float value_of(u32 key)
{
  constexpr int low = 32 - kKeyBits<T>;
  // the bits below the kept ones are zero in the value: ones in a negative number's complement
  const u32 k = key << low;
  return as_f32((k >> 31) ? k & 0x7fffffffu : ~(k | ((1u << low) - 1)));
}
// Key and index as one number that is larger for what ranks first; no two are equal.
__device__ __forceinline__ u64 entry_of(u32 key, u32 index) { return ((u64)key << 32) | (u32)~index; }
__device__ __forceinline__ u32 entry_index(u64 e) { return ~(u32)e; }
__device__ __forceinline__ u32 entry_key(u64 e) { return (u32)(e >> 32); }

// ---- a workgroup's sums -------------------------------------------------------------------------

template <class T, class F>
__device__ __forceinline__ T wave_all(T v, F f)
{
  v = f(v, xchg<0>(v));
  v = f(v, xchg<1>(v));
  v = f(v, xchg<2>(v));
  v = f(v, xchg<3>(v));
  v = f(v, xchg<4>(v));
  v = f(v, xchg<5>(v));
  return v;
}

// f over all threads of a workgroup of W waves, in wave order (the same bits every time); `box`
// holds W values and is free again after the next barrier.
template <int W, class T, class F>
__device__ __forceinline__ T block_all(T v, F f, T* box)
{
  v = wave_all(v, f);
  if constexpr (W > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = v;
    __syncthreads();
    v = box[0];
#pragma unroll
    for (int w = 1; w < W; ++w) v = f(v, box[w]);
  }
  return v;
}

struct AddF {
  template <class T>
  __device__ __forceinline__ T operator()(T a, T b) const
  {
    return a + b;
  }
};
struct MaxF {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ __forceinline__ u32 operator()(u32 a, u32 b) const { return a > b ? a : b; }
};

// Sum over the threads before this one; `total` gets the sum over all of them.
template <int W, class T>
__device__ __forceinline__ T block_before(T v, T* box, T& total)
{
  const int lane = threadIdx.x & 63;
  T s            = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T o = __shfl_up(s, d, 64);
    if (lane >= d) s += o;
  }
  __syncthreads();
  if (lane == 63) box[threadIdx.x >> 6] = s;
  __syncthreads();
  T before = s - v;
  total    = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += box[w];
    total += box[w];
  }
  return before;
}

// ---- sweeps -------------------------------------------------------------------------------------

// f(x, index) for every element of the row, in no order.
template <class T, int THREADS, class F>
__device__ __forceinline__ void sweep(const T* row, int n, F f)
{
  constexpr int VEC = In<T>::VEC;
  const int nv      = n / VEC;
  for (int v = threadIdx.x; v < nv; v += THREADS) {
    const u32x4 w = load16c(row + (int64_t)v * VEC);
    static_for<VEC>([&](auto j) { f((float)In<T>::template get<j>(w), v * VEC + j); });
  }
  for (int i = nv * VEC + threadIdx.x; i < n; i += THREADS) f(widen(row + i), i);
}

// Visits the row in index order, a tile of THREADS vectors at a time: g(first index, values,
// count) in every thread, count elements from that index on, until g returns false (in every
// thread alike).  All threads call g for every tile.
template <class T, int THREADS, class G>
__device__ __forceinline__ void ordered_sweep(const T* row, int n, G g)
{
  constexpr int VEC = In<T>::VEC;
  for (int base = 0; base < n; base += THREADS * VEC) {
    const int at = base + (int)threadIdx.x * VEC;
    float x[VEC];
    int count = n - at;
    count     = count < 0 ? 0 : (count > VEC ? VEC : count);
    if (count == VEC) {
      const u32x4 w = load16c(row + at);
      static_for<VEC>([&](auto j) { x[j] = (float)In<T>::template get<j>(w); });
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = j < count ? widen(row + at + j) : 0.0f;
    }
    if (!g(at, x, count)) return;
  }
}

// ---- the cut of a row in rank order -----------------------------------------------------------

// The elements with a key above `key`, and of those that have it some first ones in index order.
struct Cut {
  u32 key;
  u64 above;  // the weight of the elements with a larger key
  u64 with;   // the weight of the elements with this key
};

constexpr int kBins = 256;

// The largest key such that the elements with this key or a larger one weigh `target` or more
// (target >= 1, and at most the weight of all elements).  Every sweep of the row splits the range
// of keys that is left into 256 parts and adds the elements' weights up in LDS: one sweep for each
// 8 bits of the range.  The weights are whole numbers, so the order of the additions does not
// matter.  weigh(x, index) is 0 for elements that do not count.
template <class T, int THREADS, class F>
__device__ Cut find_cut(const T* row, int n, u32 max_key, u64 target, F weigh, u64* bins /* kBins + 2 */)
{
  u32 lo = 0, hi = max_key;
  u64 above = 0;
  for (;;) {
    const u32 width = hi - lo;
    const int bits  = width == 0 ? 0 : 32 - __builtin_clz(width);
    const int shift = bits > 8 ? bits - 8 : 0;
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += THREADS) bins[b] = 0;
    if (threadIdx.x == 0) {  // where the weights do not reach the target: all elements
      bins[kBins]     = above;
      bins[kBins + 1] = 0;
    }
    __syncthreads();
    sweep<T, THREADS>(row, n, [&](float x, int i) {
      const u32 k = key_of<T>(x);
      if (k < lo || k > hi) return;
      const u64 w = weigh(x, i);
      if (w != 0) atomicAdd((unsigned long long*)&bins[(k - lo) >> shift], (unsigned long long)w);
    });
    __syncthreads();
    if (threadIdx.x < 64) {  // the first wave: from the last bin down, four bins a lane
      const int l = 63 - (int)threadIdx.x;
      u64 own[4], sum = 0;
#pragma unroll
      for (int j = 3; j >= 0; --j) sum += own[j] = bins[4 * l + j];
      u64 upto = sum;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const u64 o = __shfl_up(upto, d, 64);
        if ((int)threadIdx.x >= d) upto += o;
      }
      u64 before = above + upto - sum;
      if (before < target && above + upto >= target) {  // one lane
        int b = 3;
#pragma unroll
        for (int j = 3; j > 0; --j) {
          if (b == j && before + own[j] < target) {
            before += own[j];
            b = j - 1;
          }
        }
        bins[kBins]     = before;
        bins[kBins + 1] = (u64)(4 * l + b);
      }
    }
    __syncthreads();
    above     = bins[kBins];
    const u32 b = (u32)bins[kBins + 1];
    const u64 w = bins[b];
    lo += b << shift;
    const u32 last = lo + ((1u << shift) - 1);
    hi             = hi < last ? hi : last;
    if (shift == 0) return Cut{lo, above, w};
  }
}

}  // namespace logits
}  // namespace rmi
