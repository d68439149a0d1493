// raft::matrix::top_k, raft::matrix::sample_tokens and raft::stats::distillation_* on the GPU against a sequential
// host evaluation in double precision: one after the other as a training step and a decoding step would
// call them, contiguous and strided, eagerly and from a graph that was recorded through a handle.
#include <raft/core/device_mdarray.hpp>
#include <raft/core/device_mdspan.hpp>
#include <raft/core/device_resources.hpp>
#include <raft/matrix/sample.cuh>
#include <raft/matrix/top_k.cuh>
#include <raft/stats/distillation.cuh>
#include <raft/util/cudart_utils.hpp>

#include <algorithm>
#include <cstdint>
#include <numeric>
#include <random>

#include "check.hpp"

namespace {

template <typename T>
std::vector<T> to_host(const T* d, size_t n, hipStream_t s)
{
  std::vector<T> h(n);
  raft::update_host(h.data(), d, n, s);
  RAFT_HIP_TRY(hipStreamSynchronize(s));
  return h;
}

std::vector<float> normal(size_t n, float sigma, unsigned long long seed)
{
  std::mt19937_64 g(seed);
  std::normal_distribution<float> d(0.0f, sigma);
  std::vector<float> v(n);
  for (auto& x : v)
    x = d(g);
  return v;
}

struct Buffers {
  int rows, cols, ld, k;
  raft::device_matrix<float, int, raft::row_major> student, teacher, values, stats, grad, grad2;
  raft::device_matrix<int, int, raft::row_major> indices;
  raft::device_vector<float, int> lse, loss, loss2, u, top_p, logprob;
  raft::device_vector<int, int> token;

  Buffers(raft::resources const& h, int rows_, int cols_, int ld_, int k_)
    : rows(rows_),
      cols(cols_),
      ld(ld_),
      k(k_),
      student(raft::make_device_matrix<float, int, raft::row_major>(h, rows_, ld_)),
      teacher(raft::make_device_matrix<float, int, raft::row_major>(h, rows_, ld_)),
      values(raft::make_device_matrix<float, int, raft::row_major>(h, rows_, k_)),
      stats(raft::make_device_matrix<float, int, raft::row_major>(h, rows_, 2)),
      grad(raft::make_device_matrix<float, int, raft::row_major>(h, rows_, cols_)),
      grad2(raft::make_device_matrix<float, int, raft::row_major>(h, rows_, ld_)),
      indices(raft::make_device_matrix<int, int, raft::row_major>(h, rows_, k_)),
      lse(raft::make_device_vector<float, int>(h, rows_)),
      loss(raft::make_device_vector<float, int>(h, rows_)),
      loss2(raft::make_device_vector<float, int>(h, rows_)),
      u(raft::make_device_vector<float, int>(h, rows_)),
      top_p(raft::make_device_vector<float, int>(h, rows_)),
      logprob(raft::make_device_vector<float, int>(h, rows_)),
      token(raft::make_device_vector<int, int>(h, rows_))
  {
  }

  // the teacher's best k, the student's loss with its gradient in one pass and in two, and a token of every row
  void run(raft::resources const& h, double temperature)
  {
    using raft::make_const_mdspan;
    auto z = raft::make_device_strided_matrix_view<const float, int, raft::row_major>(student.data_handle(), rows, cols, ld);
    auto t = raft::make_device_strided_matrix_view<const float, int, raft::row_major>(teacher.data_handle(), rows, cols, ld);
    auto g2 = raft::make_device_strided_matrix_view<float, int, raft::row_major>(grad2.data_handle(), rows, cols, ld);
    raft::matrix::top_k(h, t, values.view(), indices.view(), lse.view(), temperature);
    raft::stats::distillation_settings<int> how;
    how.temperature = temperature;
    how.scale       = temperature * temperature / rows;
    how.teacher_lse = make_const_mdspan(lse.view());
    auto tv = make_const_mdspan(values.view());
    auto ti = make_const_mdspan(indices.view());
    raft::stats::distillation_loss(h, z, tv, ti, loss.view(), grad.view(), how);
    raft::stats::distillation_loss_stats(h, z, tv, ti, loss2.view(), stats.view(), how);
    raft::stats::distillation_grad(h, z, tv, ti, make_const_mdspan(stats.view()), g2, how);
    raft::matrix::sampling_settings<int> s;
    s.top_p = make_const_mdspan(top_p.view());
    raft::matrix::sample_tokens(h, z, make_const_mdspan(u.view()), token.view(), logprob.view(), s);
  }

  std::vector<float> zh, th, uh, ph;
  void fill(unsigned long long seed, hipStream_t s)
  {
    zh = normal((size_t)rows * ld, 2.0f, seed);
    th = normal((size_t)rows * ld, 2.0f, seed + 1);
    std::mt19937_64 g(seed + 2);
    std::uniform_real_distribution<float> d(0.0f, 1.0f);
    uh.resize(rows), ph.resize(rows);
    for (int i = 0; i < rows; ++i)
      uh[i] = d(g), ph[i] = 0.5f + 0.5f * d(g);
    raft::update_device(student.data_handle(), zh.data(), zh.size(), s);
    raft::update_device(teacher.data_handle(), th.data(), th.size(), s);
    raft::update_device(u.data_handle(), uh.data(), uh.size(), s);
    raft::update_device(top_p.data_handle(), ph.data(), ph.size(), s);
    RAFT_HIP_TRY(hipStreamSynchronize(s));
  }

  // Sums of n terms in fp32 are off by less than n half steps; the lse of n terms by that and by the rounding
  // of max / T, which is below 2^4.  A token may only differ from the host's where u times the mass falls within
  // the host's own error of a border, which 1e-9 of the mass is far above.
  void check(double T, hipStream_t s) const
  {
    const auto v   = to_host(values.data_handle(), (size_t)rows * k, s);
    const auto ix  = to_host(indices.data_handle(), (size_t)rows * k, s);
    const auto ls  = to_host(lse.data_handle(), (size_t)rows, s);
    const auto lo  = to_host(loss.data_handle(), (size_t)rows, s);
    const auto lo2 = to_host(loss2.data_handle(), (size_t)rows, s);
    const auto g1  = to_host(grad.data_handle(), (size_t)rows * cols, s);
    const auto g2  = to_host(grad2.data_handle(), (size_t)rows * ld, s);
    const auto tok = to_host(token.data_handle(), (size_t)rows, s);
    const auto lpr = to_host(logprob.data_handle(), (size_t)rows, s);
    const double eps = std::ldexp(1.0, -24);
    const double rel = (cols + 64) * eps;  // of a sum of `cols` terms
    bool order = true, sums = true, losses = true, grads = true, tokens = true;
    for (int i = 0; i < rows; ++i) {
      const float* t = &th[(size_t)i * ld];
      const float* z = &zh[(size_t)i * ld];
      std::vector<int> rank(cols);
      std::iota(rank.begin(), rank.end(), 0);
      std::sort(rank.begin(), rank.end(), [&](int a, int b) { return t[a] != t[b] ? t[a] > t[b] : a < b; });
      double sum_t = 0, sum_z = 0;
      for (int c = 0; c < cols; ++c)
        sum_t += std::exp(t[c] / T), sum_z += std::exp(z[c] / T);
      const double L = std::log(sum_t), Z = std::log(sum_z);
      sums &= std::fabs(ls[i] - L) <= rel + 32 * eps;
      const double scale = T * T / rows;
      double want = 0, mass = 0, size = 0;
      std::vector<double> p(cols, 0.0);
      for (int j = 0; j < k; ++j) {
        order &= ix[(size_t)i * k + j] == rank[j] && v[(size_t)i * k + j] == t[rank[j]];
        const double lp = t[rank[j]] / T - L, pj = std::exp(lp);
        want += pj * (lp - (z[rank[j]] / T - Z));
        size += pj * (std::fabs(lp) + std::fabs(z[rank[j]] / T - Z) + 1);
        p[rank[j]] += pj;
        mass += pj;
      }
      losses &= std::fabs(lo[i] - scale * want) <= scale * size * 4 * (rel + 64 * eps);
      losses &= std::fabs(lo2[i] - scale * want) <= scale * size * 4 * (rel + 64 * eps);
      for (int c = 0; c < cols; ++c) {
        const double q = std::exp(z[c] / T - Z), d = scale / T * (q * mass - p[c]);
        const double tol = scale / T * (q * mass + p[c]) * 4 * (rel + 64 * eps);
        grads &= std::fabs(g1[(size_t)i * cols + c] - d) <= tol && std::fabs(g2[(size_t)i * ld + c] - d) <= tol;
      }
      // the nucleus
      std::iota(rank.begin(), rank.end(), 0);
      std::sort(rank.begin(), rank.end(), [&](int a, int b) { return z[a] != z[b] ? z[a] > z[b] : a < b; });
      std::vector<double> w(cols);
      double all = 0, before = 0, left = 0;
      for (int c = 0; c < cols; ++c)
        all += w[c] = std::exp((double)z[c] - z[rank[0]]);
      std::vector<char> keep(cols, 0);
      bool at_border = false;
      for (int j = 0; j < cols; ++j) {
        const double gap = before - ph[i] * all;
        at_border |= std::fabs(gap) < 1e-9 * all;
        if (j > 0 && gap >= 0) break;
        keep[rank[j]] = 1, left += w[rank[j]], before += w[rank[j]];
      }
      double run_sum = 0;
      int at = -1;
      for (int c = 0; c < cols && at < 0; ++c) {
        if (!keep[c]) continue;
        run_sum += w[c];
        at_border |= std::fabs(run_sum - uh[i] * left) < 1e-9 * left;
        if (run_sum > uh[i] * left) at = c;
      }
      if (!at_border) tokens &= tok[i] == at && std::fabs(lpr[i] - std::log(w[at] / left)) <= 1e-5;
    }
    CHECK(order);
    CHECK(sums);
    CHECK(losses);
    CHECK(grads);
    CHECK(tokens);
  }
};

void together(int rows, int cols, int ld, int k, double temperature)
{
  raft::resources h;
  auto s = raft::resource::get_cuda_stream(h);
  Buffers b(h, rows, cols, ld, k);
  b.fill(rows + cols, s);
  b.run(h, temperature);
  b.check(temperature, s);
}

void under_graph_capture()
{
  hipStream_t s;
  RAFT_HIP_TRY(hipStreamCreate(&s));
  {
    raft::resources h(s);
    Buffers b(h, 300, 9001, 9004, 20);
    b.fill(1, s);
    b.run(h, 1.5);  // the handle's workspace reaches its size
    b.check(1.5, s);
    void* const before = h.workspace(1);
    hipGraph_t graph;
    hipGraphExec_t exec;
    RAFT_HIP_TRY(hipStreamBeginCapture(s, hipStreamCaptureModeThreadLocal));
    b.run(h, 1.5);
    RAFT_HIP_TRY(hipStreamEndCapture(s, &graph));
    CHECK(h.workspace(1) == before);
    RAFT_HIP_TRY(hipGraphInstantiate(&exec, graph, nullptr, nullptr, 0));
    for (unsigned long long rep = 0; rep < 3; ++rep) {
      b.fill(50 + 3 * rep, s);
      RAFT_HIP_TRY(hipGraphLaunch(exec, s));
      b.check(1.5, s);
      b.run(h, 1.5);  // eager work between the replays
      b.check(1.5, s);
    }
    RAFT_HIP_TRY(hipGraphExecDestroy(exec));
    RAFT_HIP_TRY(hipGraphDestroy(graph));
  }
  RAFT_HIP_TRY(hipStreamDestroy(s));
}

// Types of storage, an empty matrix, a mask.
template <typename T>
void narrow(T one, T three, T two)
{
  raft::resources h;
  auto s   = raft::resource::get_cuda_stream(h);
  auto in  = raft::make_device_matrix<T, std::int64_t, raft::row_major>(h, 1, 3);
  auto out = raft::make_device_matrix<T, std::int64_t, raft::row_major>(h, 1, 2);
  auto ix  = raft::make_device_matrix<int, std::int64_t, raft::row_major>(h, 1, 2);
  auto u   = raft::make_device_vector<float, std::int64_t>(h, 1);
  auto to  = raft::make_device_vector<int, std::int64_t>(h, 1);
  auto ok  = raft::make_device_matrix<std::uint32_t, std::int64_t, raft::row_major>(h, 1, 1);
  const T x[3] = {one, three, two};
  const float half = 0.5f;
  const std::uint32_t third = 4;
  raft::update_device(in.data_handle(), x, 3, s);
  raft::update_device(u.data_handle(), &half, 1, s);
  raft::update_device(ok.data_handle(), &third, 1, s);
  auto z = raft::make_const_mdspan(in.view());
  raft::matrix::top_k(h, z, out.view(), ix.view());
  CHECK((to_host(ix.data_handle(), 2, s) == std::vector<int>{1, 2}));
  raft::matrix::sampling_settings<std::int64_t> how;
  how.allowed = raft::make_const_mdspan(ok.view());
  raft::matrix::sample_tokens(h, z, raft::make_const_mdspan(u.view()), to.view(), std::nullopt, how);
  CHECK((to_host(to.data_handle(), 1, s) == std::vector<int>{2}));
  raft::matrix::top_k(h, raft::make_device_matrix_view<const T, std::int64_t>(nullptr, 0, 3),
                      raft::make_device_matrix_view<T, std::int64_t>(nullptr, 0, 2),
                      raft::make_device_matrix_view<int, std::int64_t>(nullptr, 0, 2));
}

}  // namespace

TEST_CASE(TogetherSmall) { together(7, 33, 33, 5, 1.0); }
TEST_CASE(TogetherStrided) { together(20, 5001, 5010, 64, 2.0); }
TEST_CASE(TogetherManyRows) { together(400, 4500, 4500, 1, 0.7); }
TEST_CASE(UnderGraphCapture) { under_graph_capture(); }
TEST_CASE(Half) { narrow<__half>(__float2half(1.0f), __float2half(3.0f), __float2half(2.0f)); }
TEST_CASE(BFloat16)
{
  narrow<raft::bfloat16_t>(raft::bfloat16_t{0x3f80}, raft::bfloat16_t{0x4040}, raft::bfloat16_t{0x4000});
}

int main()
{
  int n = 0;
  if (hipGetDeviceCount(&n) != hipSuccess || n == 0) {
    std::printf("no GPU visible\n");
    return 2;
  }
  return t::run_all();
}
