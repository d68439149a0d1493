// raft::matrix::top_k: the k elements of every row that rank first, with their columns, in rank order (larger
// values first, NaN last, the lowest column on ties: the rule of raft::matrix::argmax), and the row's
// log-sum-exp at a temperature where it is asked for.  rmi_top_k in the reduction library; plain C++.
#pragma once

#include <cstdint>
#include <optional>

#include <raft/core/device_mdspan.hpp>
#include <raft/core/resource/cuda_stream.hpp>
#include <raft/linalg/detail/rmi_logits.hpp>

namespace raft::matrix {

// in: rows of float, __half or bfloat16_t, contiguous or strided; values, indices: n_rows x k, k <= 1024;
// lse: log(sum_v exp(in[i][v] / temperature)) of every row.
template <typename T, typename idx_t, typename layout_t>
void top_k(raft::resources const& handle,
           raft::device_matrix_view<const T, idx_t, layout_t> in,
           raft::device_matrix_view<T, idx_t, row_major> values,
           raft::device_matrix_view<std::int32_t, idx_t, row_major> indices,
           typename raft::detail::rmi::optional_vector<float, idx_t>::type lse = std::nullopt,
           double temperature                                                  = 1.0)
{
  namespace rmi = raft::detail::rmi;
  RAFT_EXPECTS(values.extent(0) == in.extent(0) && indices.extent(0) == in.extent(0),
               "top_k: the outputs must have as many rows as the input");
  RAFT_EXPECTS(values.extent(1) == indices.extent(1), "top_k: values and indices must have the same shape");
  RAFT_EXPECTS(values.extent(1) <= in.extent(1), "top_k: k must not exceed the number of columns");
  RAFT_EXPECTS((std::int64_t)values.extent(1) <= RMI_TOP_K_MAX, "top_k: k must not exceed %d", RMI_TOP_K_MAX);
  const std::int64_t ld = rmi::rows_apart(in, "top_k");
  float* const lse_ptr  = rmi::optional_ptr(lse, in.extent(0), "top_k");
  rmi::check(rmi_top_k(rmi::logits_dtype<T>(), (std::int64_t)in.extent(0), (std::int64_t)in.extent(1), ld,
                       (int)values.extent(1), temperature, in.data_handle(), values.data_handle(),
                       indices.data_handle(), lse_ptr, resource::get_cuda_stream(handle)),
             "rmi_top_k");
}

}  // namespace raft::matrix
