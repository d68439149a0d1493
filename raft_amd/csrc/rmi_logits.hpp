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

// Workgroups over rows (or pieces of them) as a grid of two dimensions: a launch holds fewer than 2^32
// threads in each.
inline dim3 grid_of(int64_t blocks)
{
  const int64_t x = blocks < (1 << 20) ? blocks : (1 << 20);
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
__device__ __forceinline__ int64_t block_of_grid() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

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

// f over the first W lanes' values, for all lanes (W a power of two, at most 16).
template <int W, class T, class F>
__device__ __forceinline__ T lanes_all(T v, F f)
{
  static_assert(W <= 16 && (W & (W - 1)) == 0, "within a row of 16 lanes");
  if constexpr (W > 1) v = f(v, xchg<0>(v));
  if constexpr (W > 2) v = f(v, xchg<1>(v));
  if constexpr (W > 4) v = f(v, xchg<2>(v));
  if constexpr (W > 8) v = f(v, xchg<3>(v));
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
  } else {
    const u64 w  = __builtin_bit_cast(u64, v);
    const u32 lo = (u32)__builtin_amdgcn_readfirstlane((int)(u32)w);
    const u32 hi = (u32)__builtin_amdgcn_readfirstlane((int)(u32)(w >> 32));
    return __builtin_bit_cast(T, ((u64)hi << 32) | lo);
  }
}

// f over all threads of a workgroup of W waves (the same bits every time); `box` holds W values and is
// free again after the next barrier.  Lane w of every wave takes wave w's value: a few steps instead of
// a walk over all of them, whose instructions count where a kernel runs its code once.
template <int W, class T, class F>
__device__ __forceinline__ T block_all(T v, F f, T* box)
{
  v = wave_all(v, f);
  if constexpr (W > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lanes_all<W>(box[threadIdx.x & (W - 1)], f);
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
  const T own     = box[lane & (W - 1)];
  total           = lanes_all<W>(own, AddF{});
  const T earlier = lanes_all<W>((lane & (W - 1)) < (int)(threadIdx.x >> 6) ? own : (T)0, AddF{});
  return earlier + (s - v);
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

// The same element by element, four at a time: a fifth of the code and of the registers, for ways that are
// rarely taken in a kernel that has others.
template <class T, int THREADS, class F>
__device__ __forceinline__ void narrow_sweep(const T* row, int n, F f)
{
  for (int first = threadIdx.x; first < n; first += 4 * THREADS) {
    float x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = first + u * THREADS;
      x[u]        = widen(row + (i < n ? i : first));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (first + u * THREADS < n) f(x[u], first + u * THREADS);
  }
}

// Visits the row in index order, a tile of VEC elements a thread at a time: g(first index, values,
// count) in every thread, count elements from that index on, until g returns false (in every
// thread alike).  All threads call g for every tile.
template <class T, int THREADS, int VEC = In<T>::VEC, class G>
__device__ __forceinline__ void ordered_sweep(const T* row, int n, G g)
{
  for (int base = 0; base < n; base += THREADS * VEC) {
    const int at = base + (int)threadIdx.x * VEC;
    float x[VEC];
    int count = n - at;
    count     = count < 0 ? 0 : (count > VEC ? VEC : count);
    if (VEC == In<T>::VEC && count == VEC) {
      if constexpr (VEC == In<T>::VEC) {
        const u32x4 w = load16c(row + at);
        static_for<VEC>([&](auto j) { x[j] = (float)In<T>::template get<j>(w); });
      }
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
template <class T, int THREADS, bool NARROW = false, class F>
__device__ __forceinline__ Cut find_cut(const T* row, int n, u32 max_key, u64 target, F weigh, u64* bins /* kBins + 2 */)
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
    auto add = [&](float x, int i) {
      const u32 k = key_of<T>(x);
      if (k < lo || k > hi) return;
      const u64 w = weigh(x, i);
      if (w != 0) atomicAdd((unsigned long long*)&bins[(k - lo) >> shift], (unsigned long long)w);
    };
    if constexpr (NARROW)
      narrow_sweep<T, THREADS>(row, n, add);
    else
      sweep<T, THREADS>(row, n, add);
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

// ---- candidates: the elements that may be among the first k -------------------------------------

// Where the aligned 16-byte vectors of a row lie: `head` elements come before them, `nv` vectors
// follow, and what is left after them is shorter than a vector.  Reads of aligned vectors run at
// the full rate whatever the row's length and stride are; rows that are written start their vectors on
// a cache line (ALIGN = 128), so that no line is stored in parts.
template <class T, int ALIGN = 16>
struct Vectors {
  int head, nv;
  __device__ __forceinline__ Vectors(const T* row, int n)
  {
    const int off = (int)((ALIGN - (reinterpret_cast<uintptr_t>(row) & (ALIGN - 1))) & (ALIGN - 1)) / (int)sizeof(T);
    head          = off < n ? off : n;
    nv            = (n - head) / In<T>::VEC;
  }
  // The index of this thread's element outside the vectors, or -1 (there are fewer than ALIGN bytes in
  // front and fewer than a vector behind).
  __device__ __forceinline__ int extra(int n) const
  {
    const int t = (int)threadIdx.x;
    const int i = t < head ? t : t + nv * In<T>::VEC;
    return i < n && t < ALIGN / (int)sizeof(T) + In<T>::VEC ? i : -1;
  }
};

// The bits of 8 (or 4) tokens from `i` on.
__device__ __forceinline__ u32 mask_bits(const u32* allowed, int i, int words)
{
  const int w  = i >> 5;
  const u32 lo = allowed[w];
  const u32 hi = allowed[w + 1 < words ? w + 1 : w];
  return __builtin_amdgcn_alignbit(hi, lo, (u32)i & 31u);
}

// A t such that at least `need` of the wave's 64 G keys are t or more, and about as many as that: the
// largest with zeros below bit 16; 0 if there are fewer such keys than zero.  A step compares the G keys
// and counts over the lanes by scalar instructions, without a trip to LDS.  What is wanted mostly lies within
// two powers of two (2^24 keys) of the largest key: nine steps then do, sixteen otherwise.
template <int G>
__device__ __forceinline__ u32 wave_rank(const u32 (&key)[G], int need)
{
  auto have = [&](u32 t) {
    int n = 0;
#pragma unroll
    for (int g = 0; g < G; ++g) n += __popcll(__ballot(key[g] >= t));
    return n;
  };
  u32 top = key[0];
#pragma unroll
  for (int g = 1; g < G; ++g) top = top > key[g] ? top : key[g];
  top       = __builtin_amdgcn_readfirstlane(wave_all(top, MaxF{}));
  u32 t     = top > 0x01000000u ? (top - 0x01000000u) & 0xffff0000u : 0u;
  u32 first = 0x00800000u;  // t + 2^24 is above all keys but for the bits below bit 16
  if (t == 0 || have(t) < need) {
    t     = 0;
    first = 0x80000000u;
  }
#pragma unroll 1
  for (u32 bit = first; bit >= 0x10000u; bit >>= 1)
    if (have(t + bit) >= need) t += bit;
  return t;
}

// What a workgroup of W waves keeps in LDS while it looks for candidates: whole vectors that hold
// one (`hits`), and the candidates themselves.
template <int W>
struct CandidateBox {
  static constexpr int kHits    = 128 * W;
  static constexpr int kEntries = 256 * W;
  u64 entries[kEntries];
  u32x4 hit[kHits];
  int hit_at[kHits];  // the index of a vector's first element
  u32 bins[kBins];
  u32 word[W];
  float max[W];
  int hits;
  int count;
  u32 edge;
};

// How the elements of a row are looked at: kEvery for top_k (NaN and -inf have a rank too), kReal
// where only what is above -inf counts, kMasked where a bit mask says more.
enum class Look { kEvery, kReal, kMasked };

// 32-bit ordered key of an fp32 value: the one that candidates are compared by, whatever the type.
__device__ __forceinline__ u32 key32(float x) { return key_of<float>(x); }

// Keeps of the candidates those that may still be among the first k: their keys are counted in 256
// equal parts of the range between the least and the largest of them, and everything below the part
// that holds the k-th is dropped.  Returns the lower edge of that part; box.count is the new count.
template <int W>
__device__ __forceinline__ u32 thin_out(CandidateBox<W>& box, int count, int k, u32 lo, u32 hi)
{
  constexpr int THREADS = 64 * W;
  constexpr int EACH    = CandidateBox<W>::kEntries / THREADS;
  const u32 width    = hi - lo;
  const int bits     = width == 0 ? 0 : 32 - __builtin_clz(width);
  const int shift    = bits > 8 ? bits - 8 : 0;
  u64 own[EACH];
  for (int b = threadIdx.x; b < kBins; b += THREADS) box.bins[b] = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = e * THREADS + (int)threadIdx.x;
    own[e]      = i < count ? box.entries[i] : 0;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (e * THREADS + (int)threadIdx.x < count) atomicAdd(&box.bins[(entry_key(own[e]) - lo) >> shift], 1u);
  __syncthreads();
  if (threadIdx.x < 64) {
    const int l = 63 - (int)threadIdx.x;
    u32 bin[4], sum = 0;
#pragma unroll
    for (int j = 3; j >= 0; --j) sum += bin[j] = box.bins[4 * l + j];
    u32 upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const u32 o = (u32)__shfl_up((int)upto, d, 64);
      if ((int)threadIdx.x >= d) upto += o;
    }
    u32 before = upto - sum;
    if (before < (u32)k && upto >= (u32)k) {  // one lane: count >= k
      int b = 3;
#pragma unroll
      for (int j = 3; j > 0; --j) {
        if (b == j && before + bin[j] < (u32)k) {
          before += bin[j];
          b = j - 1;
        }
      }
      box.edge  = lo + ((u32)(4 * l + b) << shift);
      box.count = 0;
    }
  }
  __syncthreads();
  const u32 edge = box.edge;
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (e * THREADS + (int)threadIdx.x < count && entry_key(own[e]) >= edge)
      box.entries[atomicAdd(&box.count, 1)] = own[e];
  __syncthreads();
  return edge;
}

// From here on the wave's maxima ignore signalling NaNs as they ignore quiet ones (bit 9 of the MODE
// register, IEEE, off).  With it on, fmaxf needs an instruction per element that makes them quiet
// first.  Called once, at the start of a kernel.
__device__ __forceinline__ void maxima_ignore_nan() { __builtin_amdgcn_s_setreg(1 | (9 << 6), 0); }

__device__ __forceinline__ float max3(float a, float b, float c)
{
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// The largest of a vector's elements, NaN ignored (NaN if there is nothing else).
template <int N>
__device__ __forceinline__ float max_of(const float (&x)[N])
{
  static_assert(N == 4 || N == 8, "vectors of 4 or 8 elements");
  if constexpr (N == 8)
    return max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max3(x[6], x[7], x[7]));
  else
    return max3(max3(x[0], x[1], x[2]), x[3], x[3]);
}

// a b rounded, always: a product that the compiler joined with a later difference would be another number
// than the one that terms were taken against.
__device__ __forceinline__ float product(float a, float b)
{
#pragma clang fp contract(off)
  return a * b;
}

// A running maximum and sum of exp2((x - m) c) of the elements that one thread sees.  The terms are
// exp2(fma(x, c, -r)) with r = fl(m c): one rounding each, and r's own is taken back from the whole
// sum (residue()).  That rounding is in the exponent, 2^-25 of |r| at most: from
// |r| = 2^17 on, where it reaches 2^-8 (and 128, beyond which nothing is left of a sum, at 2^32), the
// difference x - m is taken first.
struct Running {
  static constexpr float kLarge = 0x1p17f;
  float m = -kInf;
  float r = -kInf;  // nothing yet: the careful way
  float s = 0;
  __device__ __forceinline__ static float ref(float m) { return fabsf(m) < kInf ? m : 0.0f; }
  // of r = fl(ref(m) c): whether differences are taken first
  __device__ __forceinline__ static bool large(float r) { return !(fabsf(r) < kLarge); }
  // What a sum that belongs to m is multiplied by to belong to `to`; r and q are their products with c.
  __device__ __forceinline__ static float moved(float m, float r, float to, float q, float c)
  {
    if (__builtin_expect(!large(fmaxf(fabsf(r), fabsf(q))), 1)) return __builtin_amdgcn_exp2f(r - q);
    if (!(m > -kInf)) return 1.0f;  // a sum of nothing, or of NaN alone
    // from r to m c, on to `to` c, and from there to q
    const float off = (large(q) ? 0.0f : fmaf(ref(to), c, -q)) - (large(r) ? 0.0f : fmaf(ref(m), c, -r));
    return __builtin_amdgcn_exp2f((ref(m) - ref(to)) * c + off);
  }
  __device__ __forceinline__ void raise(float to, float c)
  {
    if (to > m) {
      const float q = product(ref(to), c);
      s *= moved(m, r, to, q, c);
      m = to;
      r = q;
    }
  }
  // After raise() with at least the largest of them.
  template <int N, int V>
  __device__ __forceinline__ void add(const float (&x)[N][V], float c)
  {
    float t[2] = {0, 0};
    if (__builtin_expect(!large(r), 1)) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) t[j & 1] += __builtin_amdgcn_exp2f(fmaf(x[i][j], c, -r));
    } else {
      const float at = ref(m);
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) t[j & 1] += __builtin_amdgcn_exp2f((x[i][j] - at) * c);
    }
    s += t[0] + t[1];
  }
  // This thread's sum against the maximum `top` of all; top's own r is fl(ref(top) c).
  __device__ __forceinline__ double against(float top, float c) const
  {
    return (double)(s * moved(m, r, top, product(ref(top), c), c));
  }
  // The power of two that a sum held against fl(m c) is short of the sum held against m itself, exactly.  With it
  // c = fl(log2(e) / T) multiplies nothing but distances from m, so that what c is off by does not grow with |m|.
  __device__ __forceinline__ static double residue(float top, float c)
  {
    const float m = ref(top), q = product(m, c);
    return large(q) ? 0.0 : (double)q - (double)m * (double)c;
  }
  // log of sum exp(x / T) from all = the sum over the threads of against(top)
  __device__ __forceinline__ static double log_sum(float top, float c, double inv_t, double all)
  {
    if (all == all && fabsf(top) == kInf) return (double)top;
    return (double)ref(top) * inv_t + residue(top, c) * kLn2 + log(all);
  }
};

// Descending, `size` (a power of two) entries.
template <int THREADS>
__device__ __forceinline__ void sort_entries(u64* e, int size)
{
  __syncthreads();
  for (int len = 2; len <= size; len <<= 1) {
    for (int d = len >> 1; d > 0; d >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += THREADS) {
        const int a = 2 * i - (i & (d - 1));
        const u64 x = e[a], y = e[a + d];
        if ((x < y) == ((a & len) == 0)) {
          e[a]     = y;
          e[a + d] = x;
        }
      }
      // Where partners are at most 64 apart, now and in the next step, a wave's 64 pairs are the same 128 entries
      // again, and its own accesses are in order.
      if (d > 64 || (d == 1 && len > 64)) {
        __syncthreads();
      } else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
  __syncthreads();
}

// The same with one entry in every thread's register (`size` at most THREADS, at least 64; threads from `size` on
// bring nothing and get nothing): partners in one wave meet by a permute, the others in `e`.
template <int THREADS>
__device__ __forceinline__ u64 sort_one_each(u64 own, int size, u64* e)
{
  const int tid = (int)threadIdx.x;
  for (int len = 2; len <= size; len <<= 1) {
    const bool falls = (tid & len) == 0;
    for (int d = len >> 1; d > 0; d >>= 1) {
      u64 other;
      if (d >= 64) {
        if (tid < size) e[tid] = own;
        __syncthreads();
        other = tid < size ? e[tid ^ d] : 0;
        __syncthreads();
      } else {
        const int from = ((tid ^ d) & 63) << 2;
        const u32 lo   = (u32)__builtin_amdgcn_ds_bpermute(from, (int)(u32)own);
        const u32 hi   = (u32)__builtin_amdgcn_ds_bpermute(from, (int)(u32)(own >> 32));
        other          = (u64)hi << 32 | lo;
      }
      const bool larger = ((tid & d) == 0) == falls;
      own               = (own > other) == larger ? own : other;
    }
  }
  return own;
}

struct Found {
  bool all;    // the box holds the candidates; otherwise they did not fit and it is of no use
  int count;   // how many
  u32 tau;     // every element with a key32 of tau or more is in the box; 0: every element
  float max;   // of the elements that count
};

// One pass over a row that leaves in `box` at least its first k elements (k <= 64 W, or all there
// are), unordered, with keys of 32 bits.  The first NV loads of every thread set a threshold: every
// wave takes the (k / W)-th largest of its 256 maxima over NV / 4 vectors, and the least of the waves' is
// passed by k elements or more.  From then on a vector costs its maximum and a comparison; the few that
// pass are put aside whole and looked at element by element between the batches, all lanes at once (an
// element taken out where it is found costs a whole wave some twenty instructions).  The threshold is
// raised when twice k elements have gathered.  A vector's registers are loaded again as soon as it has been
// looked at, so NV loads per thread are in flight throughout.  `run`, if wanted, is the thread's sum of
// exponentials for the log-sum-exp, from the same loads.
template <class T, int W, int NV, Look LOOK, bool SUM>
__device__ __forceinline__ Found stream_candidates(const T* row, int n, int k, const u32* allowed, float c,
                                                   CandidateBox<W>& box, Running& run, bool sum = true)
{
  constexpr int THREADS = 64 * W;
  constexpr int VEC     = In<T>::VEC;
  constexpr int GROUP   = NV / 4;
  const int words       = (n + 31) >> 5;
  const Vectors<T> vs(row, n);
  const T* body   = row + vs.head;
  const int last  = vs.nv > 0 ? vs.nv - 1 : 0;
  const int tid   = (int)threadIdx.x;

  float ext       = -kInf;
  const int ext_i = vs.extra(n);
  bool ext_on     = ext_i >= 0;
  if (ext_on) {
    ext = widen(row + ext_i);
    if (LOOK == Look::kMasked && ((allowed[ext_i >> 5] >> (ext_i & 31)) & 1u) == 0) ext_on = false;
    if (LOOK != Look::kEvery && !(ext > -kInf)) ext_on = false;
  }
  if (!ext_on) ext = -kInf;
  if (SUM && sum && ext_on) {
    const float one[1][1] = {{ext}};
    run.raise(ext, c);
    run.add(one, c);
  }
  float seen_max = ext > -kInf ? ext : -kInf;

  // Vectors are addressed by a byte offset from the batch's first one, which is the same for all lanes:
  // no 64-bit arithmetic per load.  Offsets are held within the row.
  constexpr int BATCH = THREADS * NV;
  u32x4 now[NV];
  auto fetch = [&](int first, int i) {
    const int left = last - first;
    const u32 room = (u32)(left < BATCH ? left : BATCH) * 16u;
    u32 off        = (u32)(i * THREADS + tid) * 16u;
    off            = off < room ? off : room;
    const char* p  = reinterpret_cast<const char*>(body + (int64_t)first * VEC) + off;
    if constexpr (LOOK == Look::kEvery) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    else return *reinterpret_cast<const u32x4*>(p);  // sampling may come back to the row
  };
  // The elements of a vector; what does not count is -inf.
  auto unpack = [&](const u32x4& w, int v, float(&x)[VEC]) {
    static_for<VEC>([&](auto j) { x[j] = (float)In<T>::template get<j>(w); });
    if constexpr (LOOK == Look::kMasked) {
      const int at   = v < last ? v : last;
      const u32 bits = mask_bits(allowed, vs.head + at * VEC, words);
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = (bits >> j) & 1u ? x[j] : -kInf;
    }
  };
  auto put = [&](float x, int i) {
    const int at = atomicAdd(&box.count, 1);
    if (at < CandidateBox<W>::kEntries) box.entries[at] = entry_of(key32(x), (u32)i);
  };
  // without a threshold (tau = 0) every element passes, NaN too
  auto value_at = [](u32 key) { return key != 0 ? as_f32((key >> 31) ? key & 0x7fffffffu : ~key) : -kInf; };

  if (tid == 0) box.count = box.hits = 0;
  if (vs.nv > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) now[i] = fetch(0, i);
  }
  u32 tau        = 0;
  float at_least = -kInf;
  bool fits      = true;
  float m[NV];
  // the vectors' maxima, and their share of the sum, two vectors at a time
  auto take_in = [&](int first, bool whole) {
    constexpr int PAIR = 2;
#pragma unroll
    for (int i = 0; i < NV; i += PAIR) {
      if (!whole && first + i * THREADS >= vs.nv) {
        m[i] = m[i + 1] = -kInf;
        continue;
      }
      float x[PAIR][VEC];
#pragma unroll
      for (int p = 0; p < PAIR; ++p) unpack(now[i + p], first + (i + p) * THREADS + tid, x[p]);
      if (!whole && first + (i + PAIR) * THREADS > vs.nv) {  // the same for all lanes
#pragma unroll
        for (int p = 0; p < PAIR; ++p)
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            x[p][j] = first + (i + p) * THREADS + tid < vs.nv ? x[p][j] : -kInf;
      }
#pragma unroll
      for (int p = 0; p < PAIR; ++p) m[i + p] = max_of(x[p]);
      const float most = max3(m[i], m[i + 1], -kInf);
      seen_max         = max3(seen_max, most, most);
      if (SUM && sum) {
        run.raise(most, c);
        run.add(x, c);
      }
    }
  };
  // puts vectors aside that hold a candidate, and loads the next batch in their place.  The places are
  // counted over the wave's lanes; one lane takes room for all of them.
  auto put_aside = [&](int first, bool whole, bool more) {
    u32 on = 0;
    int total = 0, place[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = first + i * THREADS + tid;
      // a vector of NaN alone has rank, too, where everything passes
      const bool hit = (m[i] >= at_least || (LOOK == Look::kEvery && tau == 0 && fits)) && (whole || v < vs.nv);
      const u64 all  = __ballot(hit);
      place[i]       = total + (int)__builtin_amdgcn_mbcnt_hi((u32)(all >> 32), __builtin_amdgcn_mbcnt_lo((u32)all, 0u));
      total += __popcll(all);
      on |= hit ? 1u << i : 0u;
    }
    if (total != 0) {
      int base = 0;
      if ((tid & 63) == 0) base = atomicAdd(&box.hits, total);
      base = __builtin_amdgcn_readfirstlane(base);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = base + place[i];
        if (((on >> i) & 1u) != 0 && at < CandidateBox<W>::kHits) {
          box.hit[at]    = now[i];
          box.hit_at[at] = vs.head + (first + i * THREADS + tid) * VEC;
        }
      }
    }
    if (more) {
#pragma unroll
      for (int i = 0; i < NV; ++i) now[i] = fetch(first + BATCH, i);
    }
  };
  auto first_threshold = [&]() {
    u32 key[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float o = g == 0 ? ext : -kInf;  // the element outside the vectors counts with the first
#pragma unroll
      for (int i = g * GROUP; i < (g + 1) * GROUP; ++i) o = max3(o, m[i], m[i]);
      key[g] = o > -kInf ? key32(o) : 0u;
    }
    tau = wave_rank<4>(key, (k + W - 1) / W);
    if ((tid & 63) == 0) box.word[tid >> 6] = tau;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) tau = tau < box.word[w] ? tau : box.word[w];
    at_least = value_at(tau);
    if (ext_on && (tau == 0 || ext >= at_least)) put(ext, ext_i);
  };
  // between two batches: the vectors put aside are looked at element by element
  auto gather = [&](bool more) {
    __syncthreads();
    const int hits = box.hits;
    __syncthreads();  // every wave has read it before a fast one adds the next batch's
    if (hits > CandidateBox<W>::kHits) {  // what is left of the row is read for its maximum and sum
      fits     = false;
      at_least = __builtin_nanf("");
    } else if (hits > (more ? CandidateBox<W>::kHits / 4 : 0)) {
      const T* flat = reinterpret_cast<const T*>(box.hit);
      for (int i = tid; i < hits * VEC; i += THREADS) {
        const float x = (float)In<T>::ld(flat + i);
        const int at  = box.hit_at[i / VEC] + i % VEC;
        bool on       = LOOK == Look::kEvery ? (tau == 0 || x >= at_least) : (x > -kInf && x >= at_least);
        if (LOOK == Look::kMasked && on) on = ((allowed[at >> 5] >> (at & 31)) & 1u) != 0;
        if (on) put(x, at);
      }
      __syncthreads();
      const int count = box.count;
      if (tid == 0) box.hits = 0;
      if (count > CandidateBox<W>::kEntries) {
        fits     = false;
        at_least = __builtin_nanf("");
      } else if (more && count >= 2 * k && count >= THREADS) {
        u32 top = 0, low = ~0u;
        for (int i = tid; i < count; i += THREADS) {
          const u32 e = entry_key(box.entries[i]);
          top         = top > e ? top : e;
          low         = low < e ? low : e;
        }
        top = block_all<W>(top, MaxF{}, box.word);
        low = ~block_all<W>(~low, MaxF{}, box.word);
        tau = thin_out<W>(box, count, k, low, top);
        if (tau < 0x00800000u) tau = 0;  // at or below the key of -inf: NaN's and -inf's own ranks
        at_least = value_at(tau);
      }
      __syncthreads();
    }
  };
  int first = 0;
  for (; first + BATCH <= vs.nv; first += BATCH) {
    take_in(first, true);
    if (first == 0) first_threshold();
    const bool more = first + BATCH < vs.nv;
    put_aside(first, true, more);
    gather(more);
  }
  if (first < vs.nv || vs.nv == 0) {
    take_in(first, false);
    if (first == 0) first_threshold();
    put_aside(first, false, false);
    gather(false);
  }
  const float top = block_all<W>(seen_max, MaxF{}, box.max);
  __syncthreads();
  return Found{fits, box.count, tau, top};
}

}  // namespace logits
}  // namespace rmi
