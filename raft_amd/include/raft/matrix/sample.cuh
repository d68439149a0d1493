// raft::matrix::sample_tokens: one column of every row of logits, drawn with the caller's random numbers from
// the softmax of the row after its temperature, top_k, top_p, min_p and mask.  rmi_sample in the reduction
// library; plain C++.
#pragma once

#include <cstdint>
#include <optional>

#include <raft/core/device_mdspan.hpp>
#include <raft/core/resource/cuda_stream.hpp>
#include <raft/linalg/detail/rmi_logits.hpp>

namespace raft::matrix {

// One setting for every row; what is left out changes nothing.
template <typename idx_t>
struct sampling_settings {
  std::optional<raft::device_vector_view<const float, idx_t>> temperature;   // not above 0: the row's arg-max
  std::optional<raft::device_vector_view<const std::int32_t, idx_t>> top_k;  // <= 0: all
  std::optional<raft::device_vector_view<const float, idx_t>> top_p;
  std::optional<raft::device_vector_view<const float, idx_t>> min_p;
  // bit v % 32 of word v / 32: whether column v may be chosen; ceil(n_cols / 32) words a row
  std::optional<raft::device_matrix_view<const std::uint32_t, idx_t, row_major>> allowed;
};

// u: numbers in [0, 1); token: the columns, -1 for a row with nothing to choose from; logprob: the log of the
// token's share of what is left.  Works in the handle's workspace, like a reduction: a graph that was recorded
// through a handle must not run beside other work of that handle.
template <typename T, typename idx_t, typename layout_t>
void sample_tokens(raft::resources const& handle,
                   raft::device_matrix_view<const T, idx_t, layout_t> logits,
                   raft::device_vector_view<const float, idx_t> u,
                   raft::device_vector_view<std::int32_t, idx_t> token,
                   typename raft::detail::rmi::optional_vector<float, idx_t>::type logprob = std::nullopt,
                   sampling_settings<idx_t> const& settings                                = {})
{
  namespace rmi    = raft::detail::rmi;
  const idx_t rows = logits.extent(0);
  RAFT_EXPECTS(u.extent(0) == rows && token.extent(0) == rows,
               "sample_tokens: one number and one token for every row are wanted");
  const std::int64_t ld            = rmi::rows_apart(logits, "sample_tokens");
  const std::int64_t words         = ((std::int64_t)logits.extent(1) + 31) / 32;
  const std::uint32_t* allowed_ptr = nullptr;
  if (settings.allowed.has_value()) {
    RAFT_EXPECTS(settings.allowed->extent(0) == rows && (std::int64_t)settings.allowed->extent(1) == words,
                 "sample_tokens: the mask must have ceil(n_cols / 32) words for every row");
    allowed_ptr = settings.allowed->data_handle();
  }
  const float* const temperature  = rmi::optional_ptr(settings.temperature, rows, "sample_tokens: temperature");
  const std::int32_t* const top_k = rmi::optional_ptr(settings.top_k, rows, "sample_tokens: top_k");
  const float* const top_p        = rmi::optional_ptr(settings.top_p, rows, "sample_tokens: top_p");
  const float* const min_p        = rmi::optional_ptr(settings.min_p, rows, "sample_tokens: min_p");
  float* const logprob_ptr        = rmi::optional_ptr(logprob, rows, "sample_tokens: logprob");
  hipStream_t stream              = resource::get_cuda_stream(handle);
  const int dtype                 = rmi::logits_dtype<T>();
  rmi::workspace_lease ws(&handle, stream,
                          rmi_sample_workspace_bytes(dtype, (std::int64_t)rows, (std::int64_t)logits.extent(1)));
  rmi::check(rmi_sample(dtype, (std::int64_t)rows, (std::int64_t)logits.extent(1), ld, logits.data_handle(),
                        allowed_ptr, words, temperature, top_k, top_p, min_p, u.data_handle(),
                        token.data_handle(), logprob_ptr, ws.data(), ws.size(), stream),
             "rmi_sample");
}

}  // namespace raft::matrix
