// rmi_distill_loss / rmi_distill_grad / rmi_distill_workspace_bytes (include/rmi_reduce.h):
// the loss of a row of student logits against a teacher's stored best logits, and its gradient.
//
//   p_j = exp(t_j / T - L),  q_v = exp((z_v - m) / T) / s,  m = max z,  s = sum_v exp((z_v - m) / T)
//   loss = scale * sum_j p_j (log p_j - (z_{i_j} - m) / T + log s)
//   dz_v = c * (P q_v - sum_{j: i_j = v} p_j),  c = g * scale / T,  P = sum_j p_j
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

// A running (max, sum of exponentials) of part of a row.
struct MaxSum {
  float m = -kInf;
  float s = 0;
};
__device__ __forceinline__ float finite_or_zero(float m) { return fabsf(m) < kInf ? m : 0.0f; }

// One workgroup per row: the running maximum and sum of the row (or the caller's), the teacher's
// probabilities in 64 bits, the loss, and a second sweep that writes the gradient.  The teacher's
// entries are written over the dense gradient after a barrier.
template <class T, int THREADS, bool FORWARD, bool GRAD>
__global__ __launch_bounds__(THREADS) void distill_kernel(DistillArgs a)
{
  constexpr int W   = THREADS / 64;
  constexpr int VEC = In<T>::VEC;
  __shared__ double p_of[RMI_DISTILL_MAX];
  __shared__ int32_t i_of[RMI_DISTILL_MAX];
  __shared__ float z_of[RMI_DISTILL_MAX];
  __shared__ double box[W];
  const int r  = blockIdx.x;
  const T* row = static_cast<const T*>(a.z) + (int64_t)r * a.ld;
  const int n  = a.n_cols;

  // the teacher's entries; the student's logits at their places are read before any is overwritten
  double best = -kInf;
  for (int j = threadIdx.x; j < a.k; j += THREADS) {
    const int64_t at = (int64_t)r * a.k + j;
    int i            = a.index[at];
    i                = i >= 0 && i < n ? i : -1;
    const double t   = teacher(a, at) * a.inv_t;
    i_of[j]          = i;
    p_of[j]          = t;
    z_of[j]          = i >= 0 ? widen(row + i) : 0.0f;
    if (i >= 0) best = fmax(best, t);
  }
  double norm;
  if (a.t_lse != nullptr) {
    norm = (double)a.t_lse[r];
  } else {
    best         = block_all<W>(best, [](double x, double y) { return fmax(x, y); }, box);
    const double ref = best > -kInf ? best : 0.0;
    double sum   = 0;
    for (int j = threadIdx.x; j < a.k; j += THREADS)
      if (i_of[j] >= 0) sum += exp(p_of[j] - ref);
    sum  = block_all<W>(sum, AddF{}, box);
    norm = ref + log(sum);
  }

  double m, log_s;
  float s;
  if constexpr (FORWARD) {
    MaxSum ms;
    sweep<T, THREADS>(row, n, [&](float x, int) {
      if (x > ms.m) {
        const float ref = finite_or_zero(x);
        ms.s *= __builtin_amdgcn_exp2f((ms.m - ref) * a.c);
        ms.m = x;
      }
      ms.s += __builtin_amdgcn_exp2f((x - finite_or_zero(ms.m)) * a.c);
    });
    const float top = block_all<W>(ms.m, MaxF{}, reinterpret_cast<float*>(box));
    const float ref = finite_or_zero(top);
    const float own = ms.m > -kInf ? ms.s * __builtin_amdgcn_exp2f((ms.m - ref) * a.c) : ms.s;
    const double all = block_all<W>((double)own, AddF{}, box);
    m     = (double)ref;
    log_s = log(all);
    s     = (float)all;
    if (a.stats != nullptr && threadIdx.x == 0) {
      a.stats[2 * (int64_t)r]     = all == 0 ? -kInf : ref;
      a.stats[2 * (int64_t)r + 1] = (float)log_s;
    }
  } else {
    m     = (double)finite_or_zero(a.stats[2 * (int64_t)r]);
    log_s = (double)a.stats[2 * (int64_t)r + 1];
    s     = (float)exp(log_s);
  }

  double loss = 0, mass = 0;
  for (int j = threadIdx.x; j < a.k; j += THREADS) {
    double p = 0;
    if (i_of[j] >= 0 && norm != -kInf) {
      const double log_p = p_of[j] - norm;
      p                  = exp(log_p);
      if (p != 0) loss += p * (log_p - (((double)z_of[j] - m) * a.inv_t - log_s));
    }
    p_of[j] = p;
    mass += p;
  }
  if constexpr (FORWARD) {
    loss = block_all<W>(loss, AddF{}, box);
    if (threadIdx.x == 0) a.loss[r] = (float)(loss * a.scale);
  }
  if constexpr (GRAD) {
    mass           = block_all<W>(mass, AddF{}, box);
    const double g = a.row_grad != nullptr ? (double)a.row_grad[r] : 1.0;
    const double c = g * a.scale * a.inv_t;
    // a row without a finite logit has q = 0 everywhere; without a teacher its gradient is zero
    const double dense = mass == 0 ? 0.0 : (s == 0 ? 0.0 : c * mass / (double)s);
    const float f      = (float)dense;
    const float ref    = (float)m;
    T* out             = static_cast<T*>(a.grad) + (int64_t)r * a.ld_grad;
    const bool zero    = mass == 0;
    const int nv       = n / VEC;
    for (int v = threadIdx.x; v < nv; v += THREADS) {
      const u32x4 w = load16c(row + (int64_t)v * VEC);
      u32x4 y;
      static_for<VEC>([&](auto j) {
        const float x = (float)In<T>::template get<j>(w);
        Put<T>::template at<j>(y, zero ? 0.0f : f * __builtin_amdgcn_exp2f((x - ref) * a.c));
      });
      store16<false>(out + (int64_t)v * VEC, y);
    }
    for (int i = nv * VEC + threadIdx.x; i < n; i += THREADS)
      Put<T>::st(out + i, zero ? 0.0f : f * __builtin_amdgcn_exp2f((widen(row + i) - ref) * a.c));
    __syncthreads();
    if (zero) return;
    for (int j = threadIdx.x; j < a.k; j += THREADS) {
      const int i = i_of[j];
      if (i < 0) continue;
      double p = 0;  // the same token may be listed more than once: every entry writes the whole sum
      for (int o = 0; o < a.k; ++o)
        if (i_of[o] == i) p += p_of[o];
      const double q = s == 0 ? 0.0 : exp(((double)z_of[j] - m) * a.inv_t) / (double)s;
      Put<T>::st(out + i, (float)(c * (mass * q - p)));
    }
  }
}

template <class T>
int launch(const DistillArgs& a, hipStream_t st)
{
  const dim3 grid((unsigned)a.n_rows), block(256);
  if (a.loss == nullptr)
    hipLaunchKernelGGL((distill_kernel<T, 256, false, true>), grid, block, 0, st, a);
  else if (a.grad != nullptr)
    hipLaunchKernelGGL((distill_kernel<T, 256, true, true>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((distill_kernel<T, 256, true, false>), grid, block, 0, st, a);
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

size_t rmi_distill_workspace_bytes(int, int64_t, int64_t, int) { return 0; }

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
                     void*,
                     size_t,
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
