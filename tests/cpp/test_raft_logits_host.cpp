// Shape and argument errors of raft::matrix::top_k, raft::matrix::sample_tokens and raft::stats::distillation_*:
// raft::logic_error for shapes, raft::exception for what the library does not offer, before anything
// touches a device, so the pointers are never dereferenced.
#include <raft/core/device_mdspan.hpp>
#include <raft/core/resources.hpp>
#include <raft/matrix/sample.cuh>
#include <raft/matrix/top_k.cuh>
#include <raft/stats/distillation.cuh>

#include "check.hpp"

namespace {

template <typename T>
auto mat(int rows, int cols)
{
  return raft::make_device_matrix_view<T, int>(reinterpret_cast<T*>(0x1000), rows, cols);
}
template <typename T>
auto vec(int n)
{
  return raft::make_device_vector_view<T, int>(reinterpret_cast<T*>(0x2000), n);
}
template <typename T>
auto strided(int rows, int cols, int s0, int s1)
{
  using view = raft::device_matrix_view<T, int, raft::layout_stride>;
  return view{reinterpret_cast<T*>(0x1000), raft::matrix_extent<int>{rows, cols}, {s0, s1}};
}

}  // namespace

TEST_CASE(top_k_refuses)
{
  raft::resources h;
  const auto in = mat<const float>(3, 2000);
  using raft::matrix::top_k;
  CHECK_THROWS_AS(top_k(h, in, mat<float>(2, 4), mat<int>(3, 4)), raft::logic_error);
  CHECK_THROWS_AS(top_k(h, in, mat<float>(3, 4), mat<int>(2, 4)), raft::logic_error);
  CHECK_THROWS_AS(top_k(h, in, mat<float>(3, 4), mat<int>(3, 5)), raft::logic_error);
  CHECK_THROWS_AS(top_k(h, in, mat<float>(3, 0), mat<int>(3, 0)), raft::logic_error);
  CHECK_THROWS_AS(top_k(h, in, mat<float>(3, 1025), mat<int>(3, 1025)), raft::logic_error);
  CHECK_THROWS_AS(top_k(h, mat<const float>(3, 4), mat<float>(3, 5), mat<int>(3, 5)), raft::logic_error);
  CHECK_THROWS_AS(top_k(h, in, mat<float>(3, 4), mat<int>(3, 4), vec<float>(2)), raft::logic_error);
  CHECK_THROWS_AS(top_k(h, strided<const float>(3, 20, 40, 2), mat<float>(3, 4), mat<int>(3, 4)), raft::logic_error);
  CHECK_THROWS_AS(top_k(h, strided<const float>(3, 20, 10, 1), mat<float>(3, 4), mat<int>(3, 4)), raft::logic_error);
  CHECK_THROWS_AS(top_k(h, in, mat<float>(3, 4), mat<int>(3, 4), std::nullopt, 0.0), raft::exception);
}

TEST_CASE(sample_tokens_refuses)
{
  raft::resources h;
  const auto in = mat<const __half>(3, 100);
  const auto u  = vec<const float>(3);
  const auto to = vec<int>(3);
  using raft::matrix::sample_tokens;
  CHECK_THROWS_AS(sample_tokens(h, in, vec<const float>(2), to), raft::logic_error);
  CHECK_THROWS_AS(sample_tokens(h, in, u, vec<int>(4)), raft::logic_error);
  CHECK_THROWS_AS(sample_tokens(h, in, u, to, vec<float>(2)), raft::logic_error);
  CHECK_THROWS_AS(sample_tokens(h, strided<const __half>(3, 20, 40, 2), u, to), raft::logic_error);
  raft::matrix::sampling_settings<int> s;
  s.allowed = mat<const std::uint32_t>(3, 3);
  CHECK_THROWS_AS(sample_tokens(h, in, u, to, std::nullopt, s), raft::logic_error);
  s       = {};
  s.top_k = vec<const int>(2);
  CHECK_THROWS_AS(sample_tokens(h, in, u, to, std::nullopt, s), raft::logic_error);
  s       = {};
  s.top_p = vec<const float>(4);
  CHECK_THROWS_AS(sample_tokens(h, in, u, to, std::nullopt, s), raft::logic_error);
}

TEST_CASE(distillation_refuses)
{
  raft::resources h;
  const auto z    = mat<const float>(3, 100);
  const auto tv   = mat<const float>(3, 4);
  const auto ti   = mat<const int>(3, 4);
  const auto loss = vec<float>(3);
  const auto st   = mat<const float>(3, 2);
  using raft::stats::distillation_grad;
  using raft::stats::distillation_loss;
  using raft::stats::distillation_loss_stats;
  CHECK_THROWS_AS(distillation_loss(h, z, mat<const float>(2, 4), ti, loss), raft::logic_error);
  CHECK_THROWS_AS(distillation_loss(h, z, tv, mat<const int>(3, 5), loss), raft::logic_error);
  CHECK_THROWS_AS(distillation_loss(h, z, mat<const float>(3, 1025), mat<const int>(3, 1025), loss), raft::logic_error);
  CHECK_THROWS_AS(distillation_loss(h, z, tv, ti, vec<float>(2)), raft::logic_error);
  CHECK_THROWS_AS(distillation_loss(h, z, tv, ti, loss, mat<float>(3, 99)), raft::logic_error);
  CHECK_THROWS_AS(distillation_loss(h, z, tv, ti, loss, strided<float>(3, 100, 99, 1)), raft::logic_error);
  CHECK_THROWS_AS(distillation_loss_stats(h, z, tv, ti, loss, mat<float>(3, 1)), raft::logic_error);
  CHECK_THROWS_AS(distillation_grad(h, z, tv, ti, mat<const float>(2, 2), mat<float>(3, 100)), raft::logic_error);
  CHECK_THROWS_AS(distillation_grad(h, z, tv, ti, st, mat<float>(4, 100)), raft::logic_error);
  raft::stats::distillation_settings<int> how;
  how.teacher_lse = vec<const float>(2);
  CHECK_THROWS_AS(distillation_loss(h, z, tv, ti, loss, how), raft::logic_error);
  how             = {};
  how.temperature = -1.0;
  CHECK_THROWS_AS(distillation_loss(h, z, tv, ti, loss, how), raft::exception);
  CHECK_THROWS_AS(distillation_grad(h, z, tv, ti, st, mat<float>(3, 100), how), raft::exception);
}

int main() { return t::run_all(); }
