// rmi_distill_loss / rmi_distill_grad (include/rmi_reduce.h):
// the loss of a row of student logits against a teacher's stored best logits, and its gradient.
//
//   p_j = exp(t_j / T - L),  q_v = exp((z_v - m) / T) / s,  m = max z,  s = sum_v exp((z_v - m) / T)
//   loss = scale * sum_j p_j (log p_j - (z_{i_j} - m) / T + log s)
//   dz_v = c * (P q_v - sum_{j: i_j = v} p_j),  c = g * scale / T,  P = sum_j p_j
//
// Memory is the bound: with the gradient a row is read once and written once where a workgroup's registers
// hold it, which is why rows are not split (q needs the whole row's s).  Measured: 4096 x 32000 bf16 100 us (83 at
// the rate of a copy, 6.5 TB/s); 4096 x 131072 bf16 393 us (332).  In two calls the row is read twice: 1000 x
// 50001 f32 109 us (90).  Rows beyond the registers are read twice in one call: 4096 x 152064 bf16 523 us (385),
// 1024 x 131072 f32 240 us (167).
#include "rmi_logits.hpp"
#include "rmi_normalize.hpp"

namespace rmi {
namespace logits {
namespace {

struct DistillArgs {
  const void* z;
  const void* t;
  const int32_t* index;
  const float* t_lse;
  const float* row_grad;
  float* loss;       // null: the backward call
  float* stats;      // written by the forward call, read by the backward one
  void* grad;
  int64_t ld, ld_grad;
  int n_rows, n_cols, k;
  int t_dtype;
  float c;           // log2(e) / T
  double inv_t, scale;
};

__device__ __forceinline__ double teacher(const DistillArgs& a, int64_t at)
{
  switch (a.t_dtype) {
    case RMI_F16: return (double)widen(static_cast<const f16_t*>(a.t) + at);
    case RMI_BF16: return (double)widen(static_cast<const bf16_t*>(a.t) + at);
    default: return (double)static_cast<const float*>(a.t)[at];
  }
}

// VEC values as one 16-byte vector, rounded to nearest even.
template <class T>
__device__ __forceinline__ u32x4 pack(const float (&y)[In<T>::VEC])
{
  u32x4 w;
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = as_u32(y[j]);
  } else if constexpr (std::is_same_v<T, bf16_t>) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const pair p = {(__bf16)y[2 * j], (__bf16)y[2 * j + 1]};  // one v_cvt_pk_bf16_f32
      w[j]         = __builtin_bit_cast(u32, p);
    }
  } else {
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const pair p = {(_Float16)y[2 * j], (_Float16)y[2 * j + 1]};
      w[j]         = __builtin_bit_cast(u32, p);
    }
  }
  return w;
}

// What the first wave of a workgroup keeps in LDS of a row's teacher; `slot` is a hash table that finds
// out whether a token is listed twice.
struct TeacherBox {
  double* p;
  float* z;
  int* index;
  int* slot;
  int slots;  // a power of two, at least 2 k
  __device__ __forceinline__ TeacherBox(void* lds, int k, int slots_) : slots(slots_)
  {
    p     = static_cast<double*>(lds);
    z     = reinterpret_cast<float*>(p + k);
    index = reinterpret_cast<int*>(z + k);
    slot  = index + k;
  }
  static int slots_of(int k)
  {
    int n = 64;
    while (n < 2 * k) n *= 2;
    return n;
  }
  static size_t bytes(int k) { return (size_t)k * 16 + (size_t)slots_of(k) * 4; }
};

// A row's teacher, by one wave, in 64 bits: its entries in box.index (-1: not used) and box.p (t / T), and
// the logarithm that its probabilities are taken against.
__device__ __forceinline__ double teacher_norm(const DistillArgs& a, int64_t r, TeacherBox& box)
{
  double best = -kInf;
  for (int j = (int)(threadIdx.x & 63); j < a.k; j += 64) {
    const int64_t at = r * a.k + j;
    int i            = a.index[at];
    i                = i >= 0 && i < a.n_cols ? i : -1;
    const double t   = teacher(a, at) * a.inv_t;
    box.index[j]     = i;
    box.p[j]         = t;
    if (i >= 0) best = fmax(best, t);
  }
  if (a.t_lse != nullptr) return (double)a.t_lse[r];
  best             = wave_all(best, [](double x, double y) { return fmax(x, y); });
  const double ref = best > -kInf ? best : 0.0;
  double sum       = 0;
  for (int j = (int)(threadIdx.x & 63); j < a.k; j += 64)
    if (box.index[j] >= 0) sum += exp(box.p[j] - ref);
  return ref + log(wave_all(sum, AddF{}));
}

// q of one logit, in 64 bits.  A sum of +inf leaves q = 0 for every finite logit, also where its own exponential
// passes the largest number.
__device__ __forceinline__ double share_of(const DistillArgs& a, float z, double m, double s)
{
  if (s == (double)kInf) return z == kInf ? (double)__builtin_nanf("") : 0.0;
  return s == 0 ? 0.0 : exp(((double)z - m) * a.inv_t) / s;
}

// The teacher of one row, by one wave, in 64 bits: p_j in box.p (0 for unused entries), the
// student's logits at its places in box.z, read before any of them is overwritten.  Returns their
// mass; `twice` tells whether a token is listed more than once.
template <class T>
__device__ __forceinline__ double teacher_in(const DistillArgs& a, int64_t r, const T* row, TeacherBox& box, bool& twice)
{
  const int lane    = (int)(threadIdx.x & 63);
  const double norm = teacher_norm(a, r, box);
  for (int j = lane; j < box.slots; j += 64) box.slot[j] = -1;
  for (int j = lane; j < a.k; j += 64) box.z[j] = box.index[j] >= 0 ? widen(row + box.index[j]) : 0.0f;
  double mass = 0;
  bool again  = false;
  for (int j = lane; j < a.k; j += 64) {
    const int i    = box.index[j];
    const double p = i >= 0 && norm != -kInf ? exp(box.p[j] - norm) : 0.0;
    box.p[j]       = p;
    mass += p;
    if (i >= 0) {  // at most half of the table is taken, so every search ends
      int h = (int)((u32)i * 2654435769u) & (box.slots - 1);
      for (;;) {
        const int was = atomicCAS(&box.slot[h], -1, i);
        if (was == -1) break;
        if (was == i) {
          again = true;
          break;
        }
        h = (h + 1) & (box.slots - 1);
      }
    }
  }
  twice = __ballot(again) != 0;
  return wave_all(mass, AddF{});
}

// The loss of a row, by the same wave: sum_j p_j (log p_j - (z_j - m) / T + log s).
__device__ __forceinline__ double loss_of(const DistillArgs& a, const TeacherBox& box, double m, double log_s)
{
  double loss = 0;
  for (int j = (int)(threadIdx.x & 63); j < a.k; j += 64) {
    const double p = box.p[j];
    if (p != 0) loss += p * (log(p) - (((double)box.z[j] - m) * a.inv_t - log_s));
  }
  return wave_all(loss, AddF{});
}

// s: the sum of exponentials against m = Running::ref(top)
__device__ __forceinline__ void write_loss(const DistillArgs& a, const TeacherBox& box, int64_t r, float top, double s)
{
  const double log_s = log(s);
  const double loss  = loss_of(a, box, (double)Running::ref(top), log_s);
  if ((threadIdx.x & 63) != 0) return;
  a.loss[r] = (float)(loss * a.scale);
  if (a.stats != nullptr) {
    a.stats[2 * r]     = s == 0 ? -kInf : Running::ref(top);
    a.stats[2 * r + 1] = (float)log_s;
  }
}

// The gradient at the listed tokens, over the dense part that has been written there.
template <class T>
__device__ __forceinline__ void patch(const DistillArgs& a, const TeacherBox& box, T* out, double c, double mass, double m,
                                      double s, bool twice)
{
  for (int j = (int)(threadIdx.x & 63); j < a.k; j += 64) {
    const int i = box.index[j];
    if (i < 0) continue;
    double p = box.p[j];
    if (twice) {  // every entry of a token writes the whole sum
      p = 0;
      for (int o = 0; o < a.k; ++o)
        if (box.index[o] == i) p += box.p[o];
    }
    Put<T>::st(out + i, (float)(c * (mass * share_of(a, box.z[j], m, s) - p)));
  }
}

// The sum of exponentials of one thread's elements, two vectors at a time, against the largest of its
// first two vectors: no maxima after that, which are a third of the instructions.  Any reference gives the
// sum as long as it neither grows much nor sinks: what a thread's elements say about that is seen in the sum
// itself, which is at least 1 with a reference out of its own elements.  If it is not, or is 2^30 or more, or
// the reference is too large for one fused step, the thread goes over its elements again and raises the
// reference as it goes.  Below 2^30 the row's maximum is 30 powers of two above the reference at most: exponents
// keep the precision that the errors of a log-sum-exp are counted with, no thread's sum is lost where a
// larger reference joins it, and the gradient's factor c P / s stays far from the denormal numbers.
struct Guess {
  static constexpr float kMost = 0x1p30f;
  Running run;
  template <int V>
  __device__ __forceinline__ void first(const float (&x)[2][V], float ext, float c)
  {
    const float m = max3(max_of(x[0]), max_of(x[1]), ext);
    const float r = product(m, c);
    run.m         = Running::large(r) ? 0.0f : m;
    run.r         = Running::large(r) ? 0.0f : r;
  }
  template <int V>
  __device__ __forceinline__ void add(const float (&x)[2][V], float c)
  {
    float t[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) t[j & 1] += __builtin_amdgcn_exp2f(fmaf(x[i][j], c, -run.r));
    run.s += t[0] + t[1];
  }
  __device__ __forceinline__ bool doubtful() const { return !(run.s >= 0.5f && run.s < kMost); }
};

// dense part of the gradient: f exp((x - m) / T), f = c P / s.  The factor is multiplied, for results of 16
// bits too: in the exponent (one instruction less an element, no time less) it would be rounded at the size of
// m c, which 16 bits show from |m| / T = 6000 on.
template <class T>
struct Dense {
  float f, r, ref, c;
  bool large, zero;
  __device__ __forceinline__ Dense(float top, float c_, double factor, double mass, double s) : c(c_)
  {
    ref   = Running::ref(top);
    r     = product(ref, c);
    large = Running::large(r);
    // a row without a finite logit has q = 0 everywhere; without a teacher its gradient is zero
    zero = mass == 0;
    f    = s == 0 || zero ? 0.0f : (float)(factor * mass) / (float)s;
    if (s == (double)kInf) {  // exp2(-inf) for every finite logit, however large, and NaN for +inf
      r     = kInf;
      large = false;
    }
  }
  __device__ __forceinline__ float one(float x) const
  {
    if (zero) return 0.0f;
    return f * __builtin_amdgcn_exp2f(large ? (x - ref) * c : fmaf(x, c, -r));
  }
  __device__ __forceinline__ u32x4 operator()(const u32x4& w) const
  {
    constexpr int VEC = In<T>::VEC;
    if (zero) return u32x4{0, 0, 0, 0};
    float x[VEC];
    static_for<VEC>([&](auto j) { x[j] = (float)In<T>::template get<j>(w); });
    if (large) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = f * __builtin_amdgcn_exp2f((x[j] - ref) * c);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = f * __builtin_amdgcn_exp2f(fmaf(x[j], c, -r));
    }
    return pack<T>(x);
  }
};

// A sum of exponentials that belongs to the maximum m, against the maximum `top` of all.
__device__ __forceinline__ double against(float m, double sum, float top, float c)
{
  if (!(m > -kInf)) return sum;  // nothing, or NaN alone
  return sum * (double)Running::moved(m, product(Running::ref(m), c), top, product(Running::ref(top), c), c);
}
// A wave's maximum and sum into LDS.
__device__ __forceinline__ void share(const Running& run, float c, float* max, double* sum)
{
  const float m  = wave_all(run.m, MaxF{});
  const double s = wave_all(run.against(m, c), AddF{});
  if ((threadIdx.x & 63) == 0) {
    max[threadIdx.x >> 6] = m;
    sum[threadIdx.x >> 6] = s;
  }
}
// What share() left there, as one: lane w of every wave takes wave w's.
template <int W>
__device__ __forceinline__ void joined(const float* max, const double* sum, float c, float& top, double& all)
{
  const int lane = (int)(threadIdx.x & 63);
  float m        = lane < W ? max[lane] : -kInf;
  double s       = lane < W ? sum[lane] : 0.0;
  top            = wave_all(m, MaxF{});
  all            = wave_all(against(m, s, top, c), AddF{});
}
// The sum against `top` itself, for the listed tokens, the loss and the statistics, from the one against
// fl(top c) that the terms of the dense part belong to.
__device__ __forceinline__ double exact_sum(float top, double all, float c) { return all * exp2(Running::residue(top, c)); }
__device__ __forceinline__ double factor_of(const DistillArgs& a, int64_t r)
{
  return (a.row_grad != nullptr ? (double)a.row_grad[r] : 1.0) * a.scale * a.inv_t;
}

// Loss and gradient of rows that fit into the registers of a workgroup (NV vectors a thread): a row is
// read once and written once.  The first wave does the teacher's part before its own share of the row, and
// the rest of it when its registers are free again.
template <class T, int W, int NV>
__global__ __launch_bounds__(64 * W, NV > 8 ? 4 : 8) void distill_rows_kernel(DistillArgs a, int slots)
{
  constexpr int THREADS = 64 * W;
  constexpr int VEC     = In<T>::VEC;
  extern __shared__ double lds[];
  __shared__ float max[W];
  __shared__ double sum[W];
  __shared__ double mass_box;
  maxima_ignore_nan();
  TeacherBox box(lds, a.k, slots);
  const int tid   = (int)threadIdx.x;
  const int n     = a.n_cols;
  const bool lead = tid < 64;
  const int64_t r = block_of_grid();
  if (r >= a.n_rows) return;
  const T* row    = static_cast<const T*>(a.z) + r * a.ld;
  T* out          = static_cast<T*>(a.grad) + r * a.ld_grad;
  const Vectors<T, 128> vs(out, n);  // whole lines where the gradient is stored
  bool twice = false;
  if (lead) {
    const double mass = teacher_in(a, r, row, box, twice);
    if (tid == 0) mass_box = mass;
  }
  u32x4 now[NV];
  if (vs.nv > 0) {
    const char* body = reinterpret_cast<const char*>(row + vs.head);
    const u32 room   = (u32)(vs.nv - 1) * 16u;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      u32 off = (u32)(i * THREADS + tid) * 16u;
      off     = off < room ? off : room;
      now[i]  = load16(body + off);
    }
  }
  const int ext_i = vs.extra(n);
  const float ext = ext_i >= 0 ? widen(row + ext_i) : -kInf;
  auto pair = [&](int i, float(&x)[2][VEC]) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
      static_for<VEC>([&](auto j) { x[p][j] = (float)In<T>::template get<j>(now[i + p]); });
    if ((i + 2) * THREADS > vs.nv) {  // behind the last vector: -inf
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[p][j] = (i + p) * THREADS + tid < vs.nv ? x[p][j] : -kInf;
    }
  };
  Guess sums;
#pragma unroll
  for (int i = 0; i < NV; i += 2) {
    if (i > 0 && i * THREADS >= vs.nv) continue;
    float x[2][VEC];
    pair(i, x);
    if (i == 0) sums.first(x, ext, a.c);
    sums.add(x, a.c);
  }
  sums.run.s += __builtin_amdgcn_exp2f(fmaf(ext, a.c, -sums.run.r));
  // the vectors stay packed: without this the compiler keeps the unpacked elements of the first pass for
  // the next ones, twice the registers of a 16-bit type
#pragma unroll
  for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(now[i]));
  if (sums.doubtful()) {
    sums.run = Running{};
    const float one[1][1] = {{ext}};
    sums.run.raise(ext, a.c);
    sums.run.add(one, a.c);
#pragma unroll
    for (int i = 0; i < NV; i += 2) {
      if (i * THREADS >= vs.nv) continue;
      float x[2][VEC];
      pair(i, x);
      sums.run.raise(max3(max_of(x[0]), max_of(x[1]), -kInf), a.c);
      sums.run.add(x, a.c);
    }
  }
  const Running& run = sums.run;
  share(run, a.c, max, sum);
  __syncthreads();
  float top;
  double all;
  joined<W>(max, sum, a.c, top, all);
  const double mass = mass_box;
  const double c    = factor_of(a, r);
  const Dense<T> dense(top, a.c, c, mass, all);
#pragma unroll
  for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(now[i]));
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i * THREADS >= vs.nv) continue;
    const u32x4 y = dense(now[i]);
    if (i * THREADS + tid < vs.nv) store16<true>(out + vs.head + (int64_t)(i * THREADS + tid) * VEC, y);
  }
  if (ext_i >= 0) {
    Put<T>::st(out + ext_i, dense.one(ext));
  }
  __syncthreads();  // the dense part is written before the listed tokens'
  if (lead) {
    const double s = exact_sum(top, all, a.c);
    write_loss(a, box, r, top, s);
    if (mass != 0) patch(a, box, out, c, mass, (double)Running::ref(top), s, twice);
  }
}

// The gradient from the statistics of an earlier forward pass: nothing joins a row's parts, so every
// workgroup takes one piece of a row, NV vectors a thread, in the order of memory.  (A workgroup that walks
// a whole row keeps a thousand rows open at once: 1000 x 50001 f32: 92 us against 77, and 72 now.  Six
// waves a SIMD leave it too few registers by five, which costs 4 us.)  Its first wave works the teacher's probabilities
// out again and corrects the listed tokens that lie in the piece.
template <class T, int W, int NV>
__global__ __launch_bounds__(64 * W, 5) void distill_grad_kernel(DistillArgs a, int pieces)
{
  constexpr int THREADS = 64 * W;
  constexpr int VEC     = In<T>::VEC;
  extern __shared__ double lds[];
  __shared__ double mass_box;
  const int tid   = (int)threadIdx.x;
  const int n     = a.n_cols;
  const bool lead = tid < 64;
  const int64_t r = block_of_grid() / pieces;
  const int piece = (int)(block_of_grid() % pieces);
  if (r >= a.n_rows) return;
  const T* row    = static_cast<const T*>(a.z) + r * a.ld;
  T* out          = static_cast<T*>(a.grad) + r * a.ld_grad;
  const Vectors<T, 128> vs(out, n);  // whole lines where the gradient is stored
  // vectors [from, to) of the row; the first piece also has the elements outside the vectors
  const int per  = ((n / VEC + pieces - 1) / pieces + 63) & ~63;  // a wave's stores cover whole lines
  const int from = min(piece * per, vs.nv);
  const int to   = min(from + per, vs.nv);
  u32x4 now[NV];
  if (from < to) {
    const char* body = reinterpret_cast<const char*>(row + vs.head + (int64_t)from * VEC);
    const u32 room   = (u32)(to - from - 1) * 16u;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      u32 off = (u32)(i * THREADS + tid) * 16u;
      off     = off < room ? off : room;
      now[i]  = load16(body + off);
    }
  }
  const int ext_i = piece == 0 ? vs.extra(n) : -1;
  const float ext = ext_i >= 0 ? widen(row + ext_i) : -kInf;
  const float top = a.stats[2 * r];
  const double m  = (double)Running::ref(top);
  const double s  = exp((double)a.stats[2 * r + 1]);
  // against fl(m c), as the terms are
  const double all = s * exp2(-Running::residue(top, a.c));
  TeacherBox box(lds, a.k, 0);
  const int lo    = vs.head + from * VEC, hi = vs.head + to * VEC;
  auto mine       = [&](int i) { return (i >= lo && i < hi) || (piece == 0 && i >= 0 && (i < vs.head || i >= vs.head + vs.nv * VEC)); };
  if (lead) {
    const double norm = teacher_norm(a, r, box);
    double mass       = 0;
    for (int j = tid; j < a.k; j += 64) {
      const int i    = box.index[j];
      const double p = i >= 0 && norm != -kInf ? exp(box.p[j] - norm) : 0.0;
      box.p[j]       = p;
      mass += p;
      if (mine(i)) box.z[j] = widen(row + i);
    }
    mass = wave_all(mass, AddF{});
    if (tid == 0) mass_box = mass;
  }
  __syncthreads();  // the logits at the listed tokens are read before any of the piece is overwritten
  const double mass = mass_box;
  const double c    = factor_of(a, r);
  const Dense<T> dense(top, a.c, c, mass, all);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = from + i * THREADS + tid;
    if (from + i * THREADS >= to) continue;
    const u32x4 y = dense(now[i]);
    if (v < to) store16<true>(out + vs.head + (int64_t)v * VEC, y);
  }
  if (ext_i >= 0) Put<T>::st(out + ext_i, dense.one(ext));
  __syncthreads();  // the dense part is written before the listed tokens'
  if (!lead || mass == 0) return;
  for (int j = tid; j < a.k; j += 64) {
    const int i = box.index[j];
    if (!mine(i)) continue;
    double p = 0;  // the same token may be listed more than once: every entry writes the whole sum
    for (int o = 0; o < a.k; ++o)
      if (box.index[o] == i) p += box.p[o];
    Put<T>::st(out + i, (float)(c * (mass * share_of(a, box.z[j], m, s) - p)));
  }
}

// One workgroup per row that is streamed, for the sum of its exponentials; if the gradient is wanted too,
// the row, too long for a workgroup's registers, is read a second time.
template <class T, int W, bool GRAD>
__global__ __launch_bounds__(64 * W, 4) void distill_stream_kernel(DistillArgs a, int slots)
{
  constexpr int THREADS = 64 * W;
  constexpr int VEC     = In<T>::VEC;
  constexpr int NV      = 4;
  extern __shared__ double lds[];
  __shared__ float max[W];
  __shared__ double sum[W];
  __shared__ double mass_box;
  maxima_ignore_nan();
  TeacherBox box(lds, a.k, slots);
  const int tid   = (int)threadIdx.x;
  const int n     = a.n_cols;
  const bool lead = tid < 64;
  const int64_t r = block_of_grid();
  if (r >= a.n_rows) return;
  const T* row    = static_cast<const T*>(a.z) + r * a.ld;
  T* out          = GRAD ? static_cast<T*>(a.grad) + r * a.ld_grad : nullptr;
  const Vectors<T, GRAD ? 128 : 16> vs(GRAD ? out : row, n);  // whole lines where the gradient is stored
  const T* body   = row + vs.head;
  const int last  = vs.nv > 0 ? vs.nv - 1 : 0;
  constexpr int BATCH = THREADS * NV;
  auto fetch = [&](int first, int i, auto keep) {
    const int left = last - first;
    const u32 room = (u32)(left < BATCH ? left : BATCH) * 16u;
    u32 off        = (u32)(i * THREADS + tid) * 16u;
    off            = off < room ? off : room;
    const char* p  = reinterpret_cast<const char*>(body + (int64_t)first * VEC) + off;
    // a row that is read again is kept in the caches
    if constexpr (keep) return load16c(p);
    else return load16(p);
  };
  const int ext_i = vs.extra(n);
  const float ext = ext_i >= 0 ? widen(row + ext_i) : -kInf;
  bool twice      = false;
  if (lead) {
    const double mass = teacher_in(a, r, row, box, twice);
    if (tid == 0) mass_box = mass;
  }
  float top;
  double all;
  {
    Running run;
    {
      const float one[1][1] = {{ext}};
      run.raise(ext, a.c);
      if (ext_i >= 0) run.add(one, a.c);
    }
    using keep = std::integral_constant<bool, GRAD>;
    u32x4 now[NV];
    auto take_in = [&](int first, bool whole) {
#pragma unroll
      for (int i = 0; i < NV; i += 2) {
        if (!whole && first + i * THREADS >= vs.nv) continue;
        float x[2][VEC];
#pragma unroll
        for (int p = 0; p < 2; ++p)
          static_for<VEC>([&](auto j) { x[p][j] = (float)In<T>::template get<j>(now[i + p]); });
        if (!whole && first + (i + 2) * THREADS > vs.nv) {
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int j = 0; j < VEC; ++j) x[p][j] = first + (i + p) * THREADS + tid < vs.nv ? x[p][j] : -kInf;
        }
        // loaded again as soon as the vectors are taken out of the registers
        if (whole) {
          const int next = first + BATCH <= last ? first + BATCH : last;
#pragma unroll
          for (int p = 0; p < 2; ++p) now[i + p] = fetch(next, i + p, keep{});
        }
        run.raise(max3(max_of(x[0]), max_of(x[1]), -kInf), a.c);
        run.add(x, a.c);
      }
    };
    if (vs.nv > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) now[i] = fetch(0, i, keep{});
    }
    int first = 0;
    for (; first + BATCH <= vs.nv; first += BATCH) take_in(first, true);
    if (first < vs.nv) take_in(first, false);
    share(run, a.c, max, sum);
    __syncthreads();
    joined<W>(max, sum, a.c, top, all);
  }
  double s = 0;
  if (lead) {
    s = exact_sum(top, all, a.c);
    write_loss(a, box, r, top, s);
  }
  if constexpr (GRAD) {
    const double mass = mass_box;
    const double c    = factor_of(a, r);
    const Dense<T> dense(top, a.c, c, mass, all);
    // The next batch is asked for before this one is stored: loads and stores are counted together, in
    // order, so loads behind the stores would wait for them.
    u32x4 now[NV], next[NV];
    if (vs.nv > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) now[i] = fetch(0, i, std::false_type{});
    }
    for (int first = 0; first < vs.nv; first += BATCH) {
      const int ahead = first + BATCH <= last ? first + BATCH : last;
#pragma unroll
      for (int i = 0; i < NV; ++i) next[i] = fetch(ahead, i, std::false_type{});
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = first + i * THREADS + tid;
        const u32x4 y = dense(now[i]);
        if (v < vs.nv) store16<true>(out + vs.head + (int64_t)v * VEC, y);
        now[i] = next[i];
      }
    }
    if (ext_i >= 0) {
      Put<T>::st(out + ext_i, dense.one(ext));
    }
    __syncthreads();
    if (lead && !dense.zero) patch(a, box, out, c, mass, (double)Running::ref(top), s, twice);
  }
}

template <class T, int W, int NV>
void launch_rows(const DistillArgs& a, int slots, size_t lds, hipStream_t st)
{
  hipLaunchKernelGGL((distill_rows_kernel<T, W, NV>), grid_of(a.n_rows), dim3(64 * W), lds, st, a, slots);
}

template <class T>
int launch(const DistillArgs& a, hipStream_t st)
{
  const int slots       = TeacherBox::slots_of(a.k);
  const size_t lds      = TeacherBox::bytes(a.k);
  const int64_t vectors = (int64_t)a.n_cols / In<T>::VEC;
  const dim3 grid = grid_of(a.n_rows);
  const bool few = a.n_rows <= 512 && vectors >= 1024;
  if (a.loss == nullptr) {
    constexpr int W = 4, NV = 8;
    const int pieces = vectors > 0 ? (int)((vectors + 64 * W * NV - 1) / (64 * W * NV)) : 1;
    hipLaunchKernelGGL((distill_grad_kernel<T, W, NV>), grid_of(a.n_rows * (int64_t)pieces), dim3(64 * W), lds, st,
                       a, pieces);
  } else if (a.grad == nullptr) {
    if (few)
      hipLaunchKernelGGL((distill_stream_kernel<T, 16, false>), grid, dim3(1024), lds, st, a, slots);
    else
      hipLaunchKernelGGL((distill_stream_kernel<T, 4, false>), grid, dim3(256), lds, st, a, slots);
  } else if (vectors > 16384) {
    hipLaunchKernelGGL((distill_stream_kernel<T, 8, true>), grid, dim3(512), lds, st, a, slots);
  } else if (vectors > 8192) {
    launch_rows<T, 16, 16>(a, slots, lds, st);
  } else if (vectors > 4096) {
    launch_rows<T, 16, 8>(a, slots, lds, st);
  } else if (vectors > 2048 && !few) {
    launch_rows<T, 8, 8>(a, slots, lds, st);
  } else if (vectors > 1024) {
    launch_rows<T, 16, 4>(a, slots, lds, st);
  } else {
    launch_rows<T, 4, 4>(a, slots, lds, st);
  }
  return hipGetLastError() == hipSuccess ? RMI_OK : RMI_ERR_LAUNCH;
}

int run(int dtype, int t_dtype, int64_t n_rows, int64_t n_cols, int64_t ld, int64_t k, double temperature,
        double scale, DistillArgs a, void* stream)
{
  if (!is_logits_dtype(dtype)) return bad_dtype(dtype);
  if (!is_logits_dtype(t_dtype)) return bad_dtype(t_dtype);
  int rc = check_shape(n_rows, n_cols, ld);
  if (rc != RMI_OK) return rc;
  if (k < 0 || k > RMI_DISTILL_MAX) return RMI_ERR_BAD_SHAPE;
  if (a.grad != nullptr && n_rows > 1 && a.ld_grad < n_cols) return RMI_ERR_BAD_SHAPE;
  // in place every row lies where it was: with another distance one row's gradient would run over another's logits
  if (a.grad != nullptr && a.grad == a.z && n_rows > 1 && n_cols > 0 && a.ld_grad != ld) return RMI_ERR_BAD_SHAPE;
  if (!(temperature >= kMinTemperature && temperature <= kMaxTemperature) || !(scale - scale == 0))
    return RMI_ERR_UNSUPPORTED;
  if (n_rows == 0 || (n_cols == 0 && a.loss == nullptr)) return RMI_OK;
  if (n_cols > 0 && a.z == nullptr) return RMI_ERR_NULL;
  if (k > 0 && (a.t == nullptr || a.index == nullptr)) return RMI_ERR_NULL;
  const size_t es = rmi_dtype_size(dtype);
  if (!aligned(a.z, es) || !aligned(a.grad, es) || !aligned(a.t, rmi_dtype_size(t_dtype)) || !aligned(a.index, 4) ||
      !aligned(a.t_lse, 4) || !aligned(a.loss, 4) || !aligned(a.stats, 4) || !aligned(a.row_grad, 4))
    return RMI_ERR_ALIGNMENT;
  a.ld      = ld;
  a.n_rows  = (int)n_rows;
  a.n_cols  = (int)n_cols;
  a.k       = (int)k;
  a.t_dtype = t_dtype;
  a.inv_t   = 1.0 / temperature;
  a.scale   = scale;
  a.c       = (float)(kLog2e / temperature);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case RMI_F16: return launch<f16_t>(a, st);
    case RMI_BF16: return launch<bf16_t>(a, st);
    default: return launch<float>(a, st);
  }
}

}  // namespace
}  // namespace logits
}  // namespace rmi

extern "C" {

int rmi_distill_loss(int dtype,
                     int t_dtype,
                     int64_t n_rows,
                     int64_t n_cols,
                     int64_t ld,
                     int k,
                     double temperature,
                     double scale,
                     const void* logits,
                     const void* t_values,
                     const int32_t* t_indices,
                     const float* t_lse,
                     float* loss,
                     float* stats,
                     const float* row_grad,
                     void* grad,
                     int64_t ld_grad,
                     void* stream)
{
  using namespace rmi::logits;
  if (n_rows > 0 && loss == nullptr) return RMI_ERR_NULL;
  DistillArgs a{};
  a.z        = logits;
  a.t        = t_values;
  a.index    = t_indices;
  a.t_lse    = t_lse;
  a.row_grad = row_grad;
  a.loss     = loss;
  a.stats    = stats;
  a.grad     = grad;
  a.ld_grad  = ld_grad;
  return run(dtype, t_dtype, n_rows, n_cols, ld, k, temperature, scale, a, stream);
}

int rmi_distill_grad(int dtype,
                     int t_dtype,
                     int64_t n_rows,
                     int64_t n_cols,
                     int64_t ld,
                     int k,
                     double temperature,
                     double scale,
                     const void* logits,
                     const void* t_values,
                     const int32_t* t_indices,
                     const float* t_lse,
                     const float* stats,
                     const float* row_grad,
                     void* grad,
                     int64_t ld_grad,
                     void* stream)
{
  using namespace rmi::logits;
  if (n_rows > 0 && n_cols > 0 && (stats == nullptr || grad == nullptr)) return RMI_ERR_NULL;
  DistillArgs a{};
  a.z        = logits;
  a.t        = t_values;
  a.index    = t_indices;
  a.t_lse    = t_lse;
  a.row_grad = row_grad;
  a.stats    = const_cast<float*>(stats);
  a.grad     = grad;
  a.ld_grad  = ld_grad;
  return run(dtype, t_dtype, n_rows, n_cols, ld, k, temperature, scale, a, stream);
}

}  // extern "C"
