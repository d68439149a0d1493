// rmi_sample / rmi_sample_workspace_bytes (include/rmi_reduce.h): one token of every row of
// logits, drawn with a given random number after temperature, top-k, top-p and min-p.
#include "rmi_logits.hpp"

namespace rmi {
namespace logits {
namespace {

struct SampleArgs {
  const void* logits;
  const u32* allowed;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int32_t* token;
  float* logprob;
  int64_t ld, ld_allowed;
  int n_rows, n_cols;
  int bits;  // the weight of the row's maximum is 2^bits
};

// exp((x - m) / T) as a whole number of 2^-bits: sums of such weights do not depend on how a row
// is split or in which order it is added up, and they are exact.  n_cols * 2^bits stays below 2^63.
struct Weights {
  double m, c, one;
  float top;
  __device__ __forceinline__ u64 operator()(float x) const
  {
    // 2^52 + w holds w in its low bits; x == m also where both are infinite
    const double t = x == top ? 0.0 : ((double)x - m) * c;
    const double w = t > -64.0 ? exp2(t) : 0.0;
    return __builtin_bit_cast(u64, fma(w, one, 4503599627370496.0)) & 0xfffffffffffffull;
  }
};

// One workgroup per row: one sweep for the maximum, sweeps for the cut by count and by mass, one
// for the total, and one in index order that ends at the token.
template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a)
{
  constexpr int W   = THREADS / 64;
  constexpr int VEC = In<T>::VEC;
  __shared__ u64 bins[kBins + 2];
  __shared__ u64 box[W];
  __shared__ u64 found[2];
  const int64_t r    = block_of_grid();
  if (r >= a.n_rows) return;
  const T* row       = static_cast<const T*>(a.logits) + r * a.ld;
  const int n        = a.n_cols;
  const u32* allowed = a.allowed != nullptr ? a.allowed + r * a.ld_allowed : nullptr;
  auto eligible      = [&](float x, int i) {
    return x > -kInf && (allowed == nullptr || ((allowed[i >> 5] >> (i & 31)) & 1u) != 0);
  };

  const float temperature = a.temperature != nullptr ? a.temperature[r] : 1.0f;
  const bool greedy       = !(temperature > 0.0f);
  float m                 = -kInf;
  u64 count               = 0;
  sweep<T, THREADS>(row, n, [&](float x, int i) {
    if (eligible(x, i)) {
      m = fmaxf(m, x);
      ++count;
    }
  });
  m     = block_all<W>(m, MaxF{}, reinterpret_cast<float*>(box));
  count = block_all<W>(count, AddF{}, box);
  if (count == 0) {
    if (threadIdx.x == 0) {
      a.token[r] = -1;
      if (a.logprob != nullptr) a.logprob[r] = -kInf;
    }
    return;
  }
  const u32 top = key_of<T>(m);
  Weights weight;
  weight.m   = (double)m;
  weight.top = m;
  weight.c   = kLog2e / (greedy ? 1.0 : (double)temperature);
  weight.one = (double)((u64)1 << a.bits);

  // the cut in rank order: every element with a key above `key`, and with it up to index `last`
  u32 key  = 0;
  int last = n;
  u64 take = ~(u64)0;  // elements with the key itself
  const int want = greedy ? 1 : (a.top_k != nullptr ? a.top_k[r] : 0);
  u64 with       = 0;  // how many there are
  if (want > 0 && (u64)want < count) {
    const Cut c = find_cut<T, THREADS>(
      row, n, top, (u64)want, [&](float x, int i) { return (u64)(eligible(x, i) ? 1 : 0); }, bins);
    key  = c.key;
    take = (u64)want - c.above;
    with = c.with;
  }
  const float top_p = !greedy && a.top_p != nullptr ? a.top_p[r] : 1.0f;
  if (top_p < 1.0f) {
    u64 all = 0;
    sweep<T, THREADS>(row, n, [&](float x, int i) {
      if (!eligible(x, i)) return;
      const u32 k = key_of<T>(x);
      if (k > key || (k == key && take == ~(u64)0)) all += weight(x);
    });
    all = block_all<W>(all, AddF{}, box);
    if (take != ~(u64)0) all += take * weight(value_of<T>(key));
    // an element is kept if the mass before it is below top_p of all
    u64 goal = (u64)ceil((double)top_p * (double)all);
    goal     = goal < 1 ? 1 : goal;
    if (goal < all) {
      const Cut c = find_cut<T, THREADS>(
        row, n, top, goal, [&](float x, int i) { return eligible(x, i) ? weight(x) : (u64)0; }, bins);
      const u64 each = weight(value_of<T>(c.key));
      key            = c.key;
      take           = (goal - c.above + each - 1) / each;
      with           = c.with / each;
    }
  }
  if (take < with) {  // where the last of the equal elements is that is kept
    u64 seen = 0;
    ordered_sweep<T, THREADS>(row, n, [&](int at, const float(&x)[VEC], int cnt) {
      u64 ties = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (j < cnt && key_of<T>(x[j]) == key && eligible(x[j], at + j)) ++ties;
      u64 all;
      u64 rank = seen + block_before<W>(ties, box, all);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (j < cnt && key_of<T>(x[j]) == key && eligible(x[j], at + j) && ++rank == take) found[0] = (u64)(at + j);
      seen += all;
      return seen < take;
    });
    __syncthreads();
    last = (int)found[0];
  }
  const float min_p = !greedy && a.min_p != nullptr ? a.min_p[r] : 0.0f;
  const double least = min_p > 0.0f ? fmin((double)min_p, 1.0) * weight.one : 0.0;
  auto kept = [&](float x, int i) -> u64 {
    if (!eligible(x, i)) return 0;
    const u32 k = key_of<T>(x);
    if (k < key || (k == key && i > last)) return 0;
    const u64 w = weight(x);
    return (double)w >= least ? w : 0;
  };
  u64 all = 0;
  sweep<T, THREADS>(row, n, [&](float x, int i) { all += kept(x, i); });
  all = block_all<W>(all, AddF{}, box);
  // the first element, in index order, whose cumulative mass exceeds u * all
  const double at_u = (double)a.u[r] * (double)all;
  u64 goal          = at_u > 0 ? (at_u < (double)all ? (u64)at_u : all - 1) : 0;
  goal              = goal < all ? goal : all - 1;
  u64 seen          = 0;
  ordered_sweep<T, THREADS>(row, n, [&](int at, const float(&x)[VEC], int cnt) {
    u64 own[VEC], sum = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum += own[j] = j < cnt ? kept(x[j], at + j) : 0;
    u64 tile;
    u64 upto = seen + block_before<W>(sum, box, tile);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if (upto <= goal && upto + own[j] > goal) {
        found[0] = (u64)(at + j);
        found[1] = own[j];
      }
      upto += own[j];
    }
    seen += tile;
    return seen <= goal;
  });
  __syncthreads();
  if (threadIdx.x == 0) {
    a.token[r] = (int32_t)found[0];
    if (a.logprob != nullptr) a.logprob[r] = (float)log((double)found[1] / (double)all);
  }
}

template <class T>
int launch(const SampleArgs& a, hipStream_t st)
{
  hipLaunchKernelGGL((sample_kernel<T, 1024>), grid_of(a.n_rows), dim3(1024), 0, st, a);
  return hipGetLastError() == hipSuccess ? RMI_OK : RMI_ERR_LAUNCH;
}

}  // namespace
}  // namespace logits
}  // namespace rmi

extern "C" {

size_t rmi_sample_workspace_bytes(int, int64_t, int64_t) { return 0; }

int rmi_sample(int dtype,
               int64_t n_rows,
               int64_t n_cols,
               int64_t ld,
               const void* logits,
               const uint32_t* allowed,
               int64_t ld_allowed,
               const float* temperature,
               const int32_t* top_k,
               const float* top_p,
               const float* min_p,
               const float* u,
               int32_t* token,
               float* logprob,
               void*,
               size_t,
               void* stream)
{
  using namespace rmi;
  using namespace rmi::logits;
  if (!is_logits_dtype(dtype)) return bad_dtype(dtype);
  int rc = check_shape(n_rows, n_cols, ld);
  if (rc != RMI_OK) return rc;
  if (allowed != nullptr && n_rows > 1 && ld_allowed < (n_cols + 31) / 32) return RMI_ERR_BAD_SHAPE;
  if (n_rows == 0) return RMI_OK;
  if (u == nullptr || token == nullptr || (n_cols > 0 && logits == nullptr)) return RMI_ERR_NULL;
  if (!rmi::logits::aligned(logits, rmi_dtype_size(dtype)) || !rmi::logits::aligned(allowed, 4) ||
      !rmi::logits::aligned(temperature, 4) || !rmi::logits::aligned(top_k, 4) || !rmi::logits::aligned(top_p, 4) ||
      !rmi::logits::aligned(min_p, 4) || !rmi::logits::aligned(u, 4) || !rmi::logits::aligned(token, 4) ||
      !rmi::logits::aligned(logprob, 4))
    return RMI_ERR_ALIGNMENT;
  SampleArgs a{};
  a.logits      = logits;
  a.allowed     = allowed;
  a.temperature = temperature;
  a.top_k       = top_k;
  a.top_p       = top_p;
  a.min_p       = min_p;
  a.u           = u;
  a.token       = token;
  a.logprob     = logprob;
  a.ld          = ld;
  a.ld_allowed  = ld_allowed;
  a.n_rows      = (int)n_rows;
  a.n_cols      = (int)n_cols;
  int log_n     = 0;
  while (((int64_t)1 << log_n) < n_cols) ++log_n;
  a.bits = 62 - log_n < 50 ? 62 - log_n : 50;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case RMI_F16: return launch<f16_t>(a, st);
    case RMI_BF16: return launch<bf16_t>(a, st);
    default: return launch<float>(a, st);
  }
}

}  // extern "C"
