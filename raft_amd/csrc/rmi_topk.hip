// rmi_top_k / rmi_top_k_workspace_bytes (include/rmi_reduce.h): the k elements of every row that
// rank first, in rank order, and the row's log-sum-exp.
#include "rmi_logits.hpp"

namespace rmi {
namespace logits {
namespace {

struct TopKArgs {
  const void* in;
  void* values;
  int32_t* indices;
  float* lse;
  int64_t ld;
  int n_rows, n_cols, k;
  float scale;   // log2(e) / T
  double inv_t;
};

// Descending, `size` (a power of two) entries.
template <int THREADS>
__device__ __forceinline__ void sort_entries(u64* e, int size)
{
  for (int len = 2; len <= size; len <<= 1) {
    for (int d = len >> 1; d > 0; d >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < size / 2; i += THREADS) {
        const int a = 2 * i - (i & (d - 1));
        const u64 x = e[a], y = e[a + d];
        if ((x < y) == ((a & len) == 0)) {
          e[a]     = y;
          e[a + d] = x;
        }
      }
    }
  }
  __syncthreads();
}

// One workgroup per row.  The row is swept for its maximum, for the sum of its exponentials, for
// the key of its k-th element (8 bits of the key a sweep) and for the elements themselves.
template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void top_k_kernel(TopKArgs a)
{
  constexpr int W   = THREADS / 64;
  constexpr int VEC = In<T>::VEC;
  __shared__ u64 bins[kBins + 2];
  __shared__ u64 entries[RMI_TOP_K_MAX];
  __shared__ u64 box[W];
  __shared__ int filled;
  const int r   = blockIdx.x;
  const T* row  = static_cast<const T*>(a.in) + (int64_t)r * a.ld;
  const int n   = a.n_cols;
  float m       = -kInf;
  u32 top       = 0;
  sweep<T, THREADS>(row, n, [&](float x, int) {
    m           = fmaxf(m, x);
    const u32 k = key_of<T>(x);
    top         = top > k ? top : k;
  });
  m   = block_all<W>(m, MaxF{}, reinterpret_cast<float*>(box));
  top = block_all<W>(top, MaxF{}, reinterpret_cast<u32*>(box));
  if (a.lse != nullptr) {
    const float ref = fabsf(m) < kInf ? m : 0.0f;
    float s         = 0;
    sweep<T, THREADS>(row, n, [&](float x, int) { s += __builtin_amdgcn_exp2f((x - ref) * a.scale); });
    const double all = block_all<W>((double)s, AddF{}, reinterpret_cast<double*>(box));
    if (threadIdx.x == 0)
      a.lse[r] = all == all && fabsf(m) == kInf ? m : (float)((double)ref * a.inv_t + log(all));
  }
  const Cut cut = find_cut<T, THREADS>(row, n, top, (u64)a.k, [](float, int) { return (u64)1; }, bins);
  const int want = a.k - (int)cut.above;  // elements with the cut's own key, from the lowest index on
  int size = 1;
  while (size < a.k) size <<= 1;
  if (threadIdx.x == 0) filled = 0;
  for (int i = threadIdx.x; i < size; i += THREADS) entries[i] = 0;
  __syncthreads();
  int seen = 0;
  ordered_sweep<T, THREADS>(row, n, [&](int at, const float(&x)[VEC], int count) {
    int ties = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if (j >= count) continue;
      const u32 k = key_of<T>(x[j]);
      ties += k == cut.key;
      if (k > cut.key) entries[atomicAdd(&filled, 1)] = entry_of(k, (u32)(at + j));
    }
    if (seen < want) {
      int all;
      int rank = seen + block_before<W>(ties, reinterpret_cast<int*>(box), all);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (j >= count || key_of<T>(x[j]) != cut.key) continue;
        if (rank < want) entries[atomicAdd(&filled, 1)] = entry_of(cut.key, (u32)(at + j));
        ++rank;
      }
      seen += all;
    }
    return true;
  });
  sort_entries<THREADS>(entries, size);
  for (int j = threadIdx.x; j < a.k; j += THREADS) {
    const u32 i       = entry_index(entries[j]);
    const int64_t out = (int64_t)r * a.k + j;
    static_cast<T*>(a.values)[out] = row[i];
    a.indices[out]                 = (int32_t)i;
  }
}

template <class T>
int launch(const TopKArgs& a, hipStream_t st)
{
  hipLaunchKernelGGL((top_k_kernel<T, 256>), dim3((unsigned)a.n_rows), dim3(256), 0, st, a);
  return hipGetLastError() == hipSuccess ? RMI_OK : RMI_ERR_LAUNCH;
}

}  // namespace
}  // namespace logits
}  // namespace rmi

extern "C" {

size_t rmi_top_k_workspace_bytes(int, int64_t, int64_t, int) { return 0; }

int rmi_top_k(int dtype,
              int64_t n_rows,
              int64_t n_cols,
              int64_t ld,
              int k,
              double temperature,
              const void* in,
              void* values,
              int32_t* indices,
              float* lse,
              void*,
              size_t,
              void* stream)
{
  using namespace rmi;
  using namespace rmi::logits;
  if (!is_logits_dtype(dtype)) return bad_dtype(dtype);
  int rc = check_shape(n_rows, n_cols, ld);
  if (rc != RMI_OK) return rc;
  if (k < 1 || k > RMI_TOP_K_MAX || k > n_cols) return RMI_ERR_BAD_SHAPE;
  if (!(temperature >= kMinTemperature && temperature <= kMaxTemperature)) return RMI_ERR_UNSUPPORTED;
  if (n_rows == 0) return RMI_OK;
  if (in == nullptr || values == nullptr || indices == nullptr) return RMI_ERR_NULL;
  const size_t es = rmi_dtype_size(dtype);
  if (!aligned(in, es) || !aligned(values, es) || !aligned(indices, 4) || !aligned(lse, 4))
    return RMI_ERR_ALIGNMENT;
  TopKArgs a{};
  a.in      = in;
  a.values  = values;
  a.indices = indices;
  a.lse     = lse;
  a.ld      = ld;
  a.n_rows  = (int)n_rows;
  a.n_cols  = (int)n_cols;
  a.k       = k;
  a.inv_t   = 1.0 / temperature;
  a.scale   = (float)(kLog2e / temperature);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case RMI_F16: return launch<f16_t>(a, st);
    case RMI_BF16: return launch<bf16_t>(a, st);
    default: return launch<float>(a, st);
  }
}

}  // extern "C"
