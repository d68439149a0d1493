// What the calls on rows of logits (matrix/top_k.cuh, matrix/sample.cuh, stats/distillation.cuh) share:
// element types, the distance between rows, optional views.
#pragma once

#include <cstdint>
#include <optional>
#include <type_traits>

#include <raft/core/device_mdspan.hpp>
#include <raft/linalg/detail/rmi_bridge.hpp>

namespace raft::detail::rmi {

template <typename T>
constexpr int logits_dtype()
{
  using value_t = std::remove_cv_t<T>;
  static_assert(std::is_same_v<value_t, float> || std::is_same_v<value_t, __half> ||
                  std::is_same_v<value_t, bfloat16_t>,
                "logits are float, __half or raft::bfloat16_t");
  return dtype<T>();
}

// Elements from one row to the next of a row-major matrix view, contiguous or strided
// (make_device_strided_matrix_view).
template <typename T, typename idx_t, typename layout_t>
std::int64_t rows_apart(const device_matrix_view<T, idx_t, layout_t>& m, const char* what)
{
  static_assert(std::is_same_v<layout_t, layout_c_contiguous> || std::is_same_v<layout_t, layout_stride>,
                "rows of logits are row-major");
  RAFT_EXPECTS(m.extent(1) <= 1 || m.stride(1) == 1, "%s: the elements of a row must lie side by side", what);
  return m.extent(0) > 1 ? (std::int64_t)m.stride(0) : (std::int64_t)m.extent(1);
}

// A view that the call may go without.  The index type follows the logits' (nothing is deduced here, so
// that a view or std::nullopt can be passed as it is).
template <typename T, typename idx_t>
struct optional_vector {
  using type = std::optional<device_vector_view<T, idx_t>>;
};

template <typename T, typename idx_t>
T* optional_ptr(const std::optional<device_vector_view<T, idx_t>>& v, idx_t n, const char* what)
{
  if (!v.has_value()) return nullptr;
  RAFT_EXPECTS(v->extent(0) == n, "%s: one value for every row is wanted", what);
  return v->data_handle();
}

}  // namespace raft::detail::rmi
