// raft::stats::distillation_loss / distillation_grad: the divergence of a student's rows of logits from the best
// logits that a teacher left for every row, and its gradient (rmi_distill_loss / rmi_distill_grad in the reduction
// library, where the formulas stand); plain C++.
#pragma once

#include <cstdint>
#include <optional>

#include <raft/core/device_mdspan.hpp>
#include <raft/core/resource/cuda_stream.hpp>
#include <raft/linalg/detail/rmi_logits.hpp>

namespace raft::stats {

// What a call may go without.  teacher_lse: the teacher's log-sum-exp over its whole vocabulary
// (raft::matrix::top_k at the same temperature); row_grad: the gradient that arrives at every row's loss.
template <typename idx_t>
struct distillation_settings {
  double temperature = 1.0;
  double scale       = 1.0;
  std::optional<raft::device_vector_view<const float, idx_t>> teacher_lse;
  std::optional<raft::device_vector_view<const float, idx_t>> row_grad;
};

namespace detail {
template <typename T, typename U, typename idx_t, typename layout_t>
void expect_teacher(raft::device_matrix_view<const T, idx_t, layout_t> logits,
                    raft::device_matrix_view<const U, idx_t, row_major> t_values,
                    raft::device_matrix_view<const std::int32_t, idx_t, row_major> t_indices,
                    const char* what)
{
  RAFT_EXPECTS(t_values.extent(0) == logits.extent(0) && t_indices.extent(0) == logits.extent(0),
               "%s: the teacher must have as many rows as the logits", what);
  RAFT_EXPECTS(t_values.extent(1) == t_indices.extent(1),
               "%s: the teacher's values and indices must have the same shape", what);
  RAFT_EXPECTS((std::int64_t)t_values.extent(1) <= RMI_DISTILL_MAX, "%s: at most %d entries of the teacher", what,
               RMI_DISTILL_MAX);
}
template <typename T, typename idx_t, typename a_t, typename b_t>
void expect_grad(raft::device_matrix_view<const T, idx_t, a_t> logits,
                 raft::device_matrix_view<T, idx_t, b_t> grad,
                 const char* what)
{
  RAFT_EXPECTS(grad.extent(0) == logits.extent(0) && grad.extent(1) == logits.extent(1),
               "%s: the gradient must have the logits' shape", what);
}
template <typename T, typename U, typename idx_t, typename layout_t>
void distillation_loss(raft::resources const& handle,
                       raft::device_matrix_view<const T, idx_t, layout_t> logits,
                       raft::device_matrix_view<const U, idx_t, row_major> t_values,
                       raft::device_matrix_view<const std::int32_t, idx_t, row_major> t_indices,
                       raft::device_vector_view<float, idx_t> loss,
                       float* stats,
                       T* grad,
                       std::int64_t ld_grad,
                       distillation_settings<idx_t> const& how)
{
  namespace rmi = raft::detail::rmi;
  expect_teacher(logits, t_values, t_indices, "distillation_loss");
  RAFT_EXPECTS(loss.extent(0) == logits.extent(0), "distillation_loss: one loss for every row is wanted");
  const std::int64_t ld  = rmi::rows_apart(logits, "distillation_loss");
  const float* const lse = rmi::optional_ptr(how.teacher_lse, logits.extent(0), "distillation_loss: teacher_lse");
  const float* const arrived = rmi::optional_ptr(how.row_grad, logits.extent(0), "distillation_loss: row_grad");
  rmi::check(rmi_distill_loss(rmi::logits_dtype<T>(), rmi::logits_dtype<U>(), (std::int64_t)logits.extent(0),
                              (std::int64_t)logits.extent(1), ld, (int)t_values.extent(1), how.temperature,
                              how.scale, logits.data_handle(), t_values.data_handle(), t_indices.data_handle(), lse,
                              loss.data_handle(), stats, arrived, grad, ld_grad,
                              resource::get_cuda_stream(handle)),
             "rmi_distill_loss");
}
}  // namespace detail

// The loss of every row, and its gradient in the same pass over the logits; `grad` may be the logits' own memory.
template <typename T, typename U, typename idx_t, typename layout_t, typename grad_layout_t>
void distillation_loss(raft::resources const& handle,
                       raft::device_matrix_view<const T, idx_t, layout_t> logits,
                       raft::device_matrix_view<const U, idx_t, row_major> t_values,
                       raft::device_matrix_view<const std::int32_t, idx_t, row_major> t_indices,
                       raft::device_vector_view<float, idx_t> loss,
                       raft::device_matrix_view<T, idx_t, grad_layout_t> grad,
                       distillation_settings<idx_t> const& how = {})
{
  detail::expect_grad(logits, grad, "distillation_loss");
  detail::distillation_loss(handle, logits, t_values, t_indices, loss, nullptr, grad.data_handle(),
                            raft::detail::rmi::rows_apart(grad, "distillation_loss"), how);
}

// The loss alone.
template <typename T, typename U, typename idx_t, typename layout_t>
void distillation_loss(raft::resources const& handle,
                       raft::device_matrix_view<const T, idx_t, layout_t> logits,
                       raft::device_matrix_view<const U, idx_t, row_major> t_values,
                       raft::device_matrix_view<const std::int32_t, idx_t, row_major> t_indices,
                       raft::device_vector_view<float, idx_t> loss,
                       distillation_settings<idx_t> const& how = {})
{
  detail::distillation_loss(handle, logits, t_values, t_indices, loss, nullptr, static_cast<T*>(nullptr),
                            std::int64_t{0}, how);
}

// The loss alone, and the two numbers of every row (n_rows x 2) from which distillation_grad starts.
template <typename T, typename U, typename idx_t, typename layout_t>
void distillation_loss_stats(raft::resources const& handle,
                             raft::device_matrix_view<const T, idx_t, layout_t> logits,
                             raft::device_matrix_view<const U, idx_t, row_major> t_values,
                             raft::device_matrix_view<const std::int32_t, idx_t, row_major> t_indices,
                             raft::device_vector_view<float, idx_t> loss,
                             raft::device_matrix_view<float, idx_t, row_major> stats,
                             distillation_settings<idx_t> const& how = {})
{
  RAFT_EXPECTS(stats.extent(0) == logits.extent(0) && stats.extent(1) == 2,
               "distillation_loss_stats: two numbers for every row are wanted");
  detail::distillation_loss(handle, logits, t_values, t_indices, loss, stats.data_handle(),
                            static_cast<T*>(nullptr), std::int64_t{0}, how);
}

// The gradient from the stats of an earlier distillation_loss_stats with the same logits, teacher and settings.
template <typename T, typename U, typename idx_t, typename layout_t, typename grad_layout_t>
void distillation_grad(raft::resources const& handle,
                       raft::device_matrix_view<const T, idx_t, layout_t> logits,
                       raft::device_matrix_view<const U, idx_t, row_major> t_values,
                       raft::device_matrix_view<const std::int32_t, idx_t, row_major> t_indices,
                       raft::device_matrix_view<const float, idx_t, row_major> stats,
                       raft::device_matrix_view<T, idx_t, grad_layout_t> grad,
                       distillation_settings<idx_t> const& how = {})
{
  namespace rmi = raft::detail::rmi;
  detail::expect_teacher(logits, t_values, t_indices, "distillation_grad");
  detail::expect_grad(logits, grad, "distillation_grad");
  RAFT_EXPECTS(stats.extent(0) == logits.extent(0) && stats.extent(1) == 2,
               "distillation_grad: two numbers for every row are wanted");
  const std::int64_t ld  = rmi::rows_apart(logits, "distillation_grad");
  const std::int64_t ldg = rmi::rows_apart(grad, "distillation_grad");
  const float* const lse = rmi::optional_ptr(how.teacher_lse, logits.extent(0), "distillation_grad: teacher_lse");
  const float* const arrived = rmi::optional_ptr(how.row_grad, logits.extent(0), "distillation_grad: row_grad");
  rmi::check(rmi_distill_grad(rmi::logits_dtype<T>(), rmi::logits_dtype<U>(), (std::int64_t)logits.extent(0),
                              (std::int64_t)logits.extent(1), ld, (int)t_values.extent(1), how.temperature,
                              how.scale, logits.data_handle(), t_values.data_handle(), t_indices.data_handle(), lse,
                              stats.data_handle(), arrived, grad.data_handle(), ldg,
                              resource::get_cuda_stream(handle)),
             "rmi_distill_grad");
}

}  // namespace raft::stats
