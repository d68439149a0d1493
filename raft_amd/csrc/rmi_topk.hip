// rmi_top_k (include/rmi_reduce.h): the k elements of every row that
// rank first, in rank order, and the row's log-sum-exp.
//
// A row has to be read once; nothing else is large, so memory is the bound (a read of this chip: 7.1 TB/s).
// Any k elements give a threshold that the k-th cannot lie below, and in a long row few elements pass one that was
// found early: the pass costs a maximum and a comparison a vector.  The log-sum-exp is summed in the same pass
// against a reference near the maximum.  Measured: 4096 x 32000 bf16, k 64 with the sum: 60 us (39 to
// read; vector instructions are issued in two thirds of the cycles); 1024 x 131072 f32, k 256: 107 us (78); one row of
// 32000 bf16: 9 us, all of it launch and steps.
#include "rmi_logits.hpp"
#include "rmi_normalize.hpp"

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

// What a row's candidates do not fit: the key of the k-th element by sweeps of the row, 8 bits of
// the key a sweep, then the elements above it and the first ones that have it, in index order.
template <class T, int W>
__device__ __forceinline__ void gather_exact(const T* row, int n, int k, float max, CandidateBox<W>& box)
{
  constexpr int THREADS = 64 * W;
  constexpr int VEC     = In<T>::VEC;
  const Cut cut     = find_cut<T, THREADS>(row, n, key_of<T>(max), (u64)k, [](float, int) { return (u64)1; }, box.entries);
  const int want    = k - (int)cut.above;  // elements with the cut's own key, from the lowest index on
  __syncthreads();
  if (threadIdx.x == 0) box.count = 0;
  __syncthreads();
  int seen = 0;
  ordered_sweep<T, THREADS>(row, n, [&](int at, const float(&x)[VEC], int count) {
    int ties = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if (j >= count) continue;
      const u32 key = key_of<T>(x[j]);
      ties += key == cut.key;
      if (key > cut.key) box.entries[atomicAdd(&box.count, 1)] = entry_of(key32(x[j]), (u32)(at + j));
    }
    if (seen < want) {
      int all;
      int rank = seen + block_before<W>(ties, reinterpret_cast<int*>(box.word), all);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (j >= count || key_of<T>(x[j]) != cut.key) continue;
        if (rank < want) box.entries[atomicAdd(&box.count, 1)] = entry_of(key32(x[j]), (u32)(at + j));
        ++rank;
      }
      seen += all;
    }
    return true;
  });
  __syncthreads();
}

// One workgroup per row: one pass over the row for its candidates and its sum of exponentials; the
// candidates are thinned out to little more than k and sorted in LDS.
template <class T, int W, int NV, bool SUM>
__global__ __launch_bounds__(64 * W, 4) void top_k_kernel(TopKArgs a)
{
  constexpr int THREADS = 64 * W;
  __shared__ CandidateBox<W> box;
  __shared__ double sums[W];
  maxima_ignore_nan();
  const int64_t r = block_of_grid();
  if (r >= a.n_rows) return;
  const T* row = static_cast<const T*>(a.in) + r * a.ld;
  const int n  = a.n_cols;
  Running run;
  const Found f = stream_candidates<T, W, NV, Look::kEvery, SUM>(row, n, a.k, nullptr, a.scale, box, run);
  if constexpr (SUM) {
    const double all = block_all<W>(run.against(f.max, a.scale), AddF{}, sums);
    if (threadIdx.x == 0) a.lse[r] = (float)Running::log_sum(f.max, a.scale, a.inv_t, all);
  }
  int count = f.count;
  if (!f.all) {
    gather_exact<T, W>(row, n, a.k, f.max, box);
    count = a.k;
  } else if (count > THREADS && count > a.k) {
    thin_out<W>(box, count, a.k, f.tau, key32(f.max));
    count = box.count;
  }
  auto write = [&](int j, u64 e) {
    const u32 key     = entry_key(e);
    const u32 i       = entry_index(e);
    const int64_t out = r * a.k + j;
    // the key says the value but for the sign of a zero and the bits of a NaN
    if (key == 0 || key == 0x80000000u)
      static_cast<T*>(a.values)[out] = row[i];
    else
      Put<T>::st(static_cast<T*>(a.values) + out, value_of<float>(key));
    a.indices[out] = (int32_t)i;
  };
  if (count <= THREADS) {
    // a thread per candidate counts those that rank before it: no barrier, and every lane reads the
    // same place in LDS
    if ((int)(threadIdx.x & ~63u) >= count) return;
    const u64 own = (int)threadIdx.x < count ? box.entries[threadIdx.x] : ~(u64)0;
    int rank      = 0;
#pragma unroll 4
    for (int i = 0; i < count; ++i) rank += box.entries[i] > own;
    if ((int)threadIdx.x < count && rank < a.k) write(rank, own);
    return;
  }
  int size = 1;
  while (size < count) size <<= 1;
  for (int i = count + (int)threadIdx.x; i < size; i += THREADS) box.entries[i] = 0;
  sort_entries<THREADS>(box.entries, size);
  for (int j = threadIdx.x; j < a.k; j += THREADS) write(j, box.entries[j]);
}

template <class T, int W, int NV>
int launch_rows(const TopKArgs& a, hipStream_t st)
{
  const dim3 grid = grid_of(a.n_rows), block(64 * W);
  if (a.lse != nullptr)
    hipLaunchKernelGGL((top_k_kernel<T, W, NV, true>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((top_k_kernel<T, W, NV, false>), grid, block, 0, st, a);
  return hipGetLastError() == hipSuccess ? RMI_OK : RMI_ERR_LAUNCH;
}

template <class T>
int launch(const TopKArgs& a, hipStream_t st)
{
  const int64_t vectors = (int64_t)a.n_cols / In<T>::VEC;
  // A workgroup of W waves sets its threshold from 256 W maxima, which is sharp while k is a quarter of
  // that; few long rows want all the loads that one CU can have in flight.
  const bool few = a.n_rows <= 512 && vectors >= 2048;
  if (a.k > 512 || few) return launch_rows<T, 16, 4>(a, st);
  if (a.k > 256) return launch_rows<T, 8, 8>(a, st);
  if (vectors > 2048) return launch_rows<T, 4, 16>(a, st);
  return vectors > 1024 ? launch_rows<T, 4, 8>(a, st) : launch_rows<T, 4, 4>(a, st);
}

}  // namespace
}  // namespace logits
}  // namespace rmi

extern "C" {

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
