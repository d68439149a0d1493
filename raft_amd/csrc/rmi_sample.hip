// rmi_sample / rmi_sample_workspace_bytes (include/rmi_reduce.h): one token of every row of
// logits, drawn with a given random number after temperature, top-k, top-p and min-p.
//
//   w_v = 2^bits exp((x_v - max) / T), right to 2^-42 of itself and rounded to a whole number,
//   K = what top_k, top_p, min_p and the mask leave,
//   token = the least v with sum_{v' in K, v' <= v} w_v' > u sum_{K} w
//
// The token must not depend on how a row is summed, so weights are whole numbers: sums of
// them are exact in any order.  One pass bound by memory decides every row whose kept tokens are few (greedy, top_k,
// a peaked nucleus).  The others cost an exact pass over all weights, some 20 vector instructions an element in
// 64 bits on the one CU that has the row (131072 elements: 20 us, half of the time in vector instructions), and for a wide
// nucleus a count of the distances before it.  Measured, 131072 tokens: one row of top_k and top_p 15 us, 256 rows of
// bf16: greedy 17, top_k 24, temperature alone 42, nucleus 89, nucleus with min_p 73 us (11.5 to read).
// The general way, for what neither decides, takes 400 us and more for such a row: top_k above 64 a wave (1024; 512
// in batches of more rows than CUs, 256 for rows of up to 1024 vectors), a top_p within some 5e-4 of 1, whose window reaches the row's light end, +inf, and
// more ties than the candidates have room for.
#include "rmi_logits.hpp"

namespace rmi {
int cu_count();  // rmi_api.hip

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
  struct Undecided* rest;
  int32_t* todo;  // whether a row is left to the second kernel
};

// What the first kernel leaves of a row that it could not decide.
struct Undecided {
  u64 base;          // exact mass of the first `known` bins
  double mass, off;  // the row's mass in fp32 and how far it may be off
  float max;
  int known;
};

// exp((x - m) / T) as a whole number of 2^-bits: sums of such weights do not depend on how a row
// is split or in which order it is added up, and they are exact.  n_cols * 2^bits stays below 2^63.
//
// With t = (x - m) log2(e) / T in 64 bits: t = k / 256 + f, 2^t = 2^(k >> 8) * table[k & 255] * 2^f,
// |f| <= 1/512, and 2^f = 1 + f l + (f l)^2 / 2 + (f l)^3 / 6 with l = ln 2, off by (f l)^4 / 24 < 2^-42.6.
// The last product adds 2^52, so the rounded weight stands in the low bits of the result.
constexpr int kTable = 256;
struct Weights {
  const double* table;  // 2^(bits + i / 256), in LDS
  double m, c;          // t = (x - m) c
  int bits;
  bool infinite;        // the maximum is +inf: whatever else there is weighs nothing
  // the weight + the bits of 2^52; not where the maximum is infinite
  __device__ __forceinline__ u64 raw(float x) const
  {
    constexpr double kRound = 6755399441055744.0 / 256.0;  // 1.5 * 2^52 / 256: what is added to it is rounded to 1 / 256
    constexpr double kL = kLn2, kL2 = kLn2 * kLn2 / 2, kL3 = kLn2 * kLn2 * kLn2 / 6;
    // -inf, NaN and what is too small for a weight end at -64
    const double t  = fmax(((double)x - m) * c, -64.0);
    const double up = t + kRound;
    const double f  = t - (up - kRound);
    const int k     = (int)(u32)__builtin_bit_cast(u64, up);
    const double p  = fma(fma(fma(kL3, f, kL2), f, kL), f, 1.0);
    return __builtin_bit_cast(u64, fma(__builtin_ldexp(table[k & (kTable - 1)], k >> 8), p, 4503599627370496.0));
  }
  __device__ __forceinline__ u64 operator()(float x) const
  {
    if (infinite) return x == kInf ? (u64)1 << bits : 0;
    return raw(x) & 0xfffffffffffffull;
  }
};

struct MaxI {
  __device__ __forceinline__ int operator()(int a, int b) const { return a > b ? a : b; }
};

struct Settings {
  float temperature, top_p, min_p, u;
  int top_k;
  bool greedy;
  __device__ __forceinline__ Settings(const SampleArgs& a, int64_t r)
  {
    temperature = a.temperature != nullptr ? a.temperature[r] : 1.0f;
    greedy      = !(temperature > 0.0f);
    if (greedy) temperature = 1.0f;
    top_k = greedy ? 1 : (a.top_k != nullptr ? a.top_k[r] : 0);
    top_p = !greedy && a.top_p != nullptr ? a.top_p[r] : 1.0f;
    top_p = top_p < 1.0f ? (top_p > 0.0f ? top_p : 0.0f) : 1.0f;  // a negative mass has no whole number
    min_p = !greedy && a.min_p != nullptr ? a.min_p[r] : 0.0f;
    min_p = min_p > 0.0f ? (min_p < 1.0f ? min_p : 1.0f) : 0.0f;
    u     = a.u[r];
  }
  // the mass that has to be passed: the first element whose cumulative mass exceeds it is taken
  __device__ __forceinline__ u64 goal(u64 all) const
  {
    const double at = (double)u * (double)all;
    return at > 0 ? (at < (double)all ? min((u64)at, all - 1) : all - 1) : 0;
  }
  // a prefix in rank order is kept as long as the mass before an element is below this
  __device__ __forceinline__ u64 nucleus(u64 all) const
  {
    const u64 mass = (u64)ceil((double)top_p * (double)all);
    return mass > 1 ? mass : 1;
  }
};

// What a workgroup keeps in LDS.
template <int W>
struct SampleBox {
  static constexpr int kSegments = 64 * W;
  CandidateBox<W> c;                          // its entries and hits make room for the bins
  u64 sorted[kSegments];                      // candidates in rank order; later the sums of the segments
  u64 mass[kSegments];
  double table[kTable];
  u64 box[W + 2];
  float fbox[W];
  u64 found[2];
  u64 last;
  int ibox[W];
  int window[3];
};

// One row of a workgroup of W waves; W_REST: those of the second kernel, which sets the width of the bins.
template <class T, int W, int W_REST, bool MASKED>
struct Row {
  static constexpr int THREADS = 64 * W;
  static constexpr int BINS    = 1024 * W_REST;  // of the distance from the maximum, in log2
  static constexpr int VEC     = In<T>::VEC;
  const SampleArgs& a;
  const T* row;
  const u32* allowed;
  SampleBox<W>& box;
  const Settings& set;
  Weights weight;
  int n;
  float max;
  u64 least;  // that a weight has to be, for min_p
  int64_t r;

  __device__ __forceinline__ bool eligible(float x, int i) const
  {
    return x > -kInf && (!MASKED || ((allowed[i >> 5] >> (i & 31)) & 1u) != 0);
  }
  __device__ __forceinline__ void answer(int token, u64 mass, u64 all) const
  {
    a.token[r] = token;
    if (a.logprob != nullptr) a.logprob[r] = (float)log((double)mass / (double)all);
  }

  // The token among the first `count` of box.sorted with their weights in box.mass, whose sum is `all`: the one, in
  // index order, whose cumulative mass passes the goal.
  __device__ __forceinline__ void choose(int count, u64 all) const
  {
    const u64 goal = set.goal(all);
    const int tid  = (int)threadIdx.x;
    if (count <= 256) {
      if ((tid & ~63) >= count) return;
      const u32 mine = tid < count ? entry_index(box.sorted[tid]) : 0;
      u64 upto       = 0;
#pragma unroll 4
      for (int o = 0; o < count; ++o) {
        const u32 other = entry_index(box.sorted[o]);
        upto += other <= mine ? box.mass[o] : 0;
      }
      if (tid < count && upto > goal && upto - box.mass[tid] <= goal) answer((int)mine, box.mass[tid], all);
      return;
    }
    // the least index at which the mass up to it passes the goal, by halving
    const u32 mine = tid < count ? entry_index(box.sorted[tid]) : ~0u;
    const u64 own  = tid < count ? box.mass[tid] : 0;
    u32 lo = 0, hi = (u32)n - 1;
    while (lo < hi) {
      const u32 mid  = lo + (hi - lo) / 2;
      const u64 upto = block_all<W>(mine <= mid ? own : (u64)0, AddF{}, box.box);
      if (upto > goal) hi = mid;
      else lo = mid + 1;
    }
    if (mine == lo) answer((int)mine, own, all);
  }

  // Candidates into rank order (count <= THREADS): few by counting for each those that rank before it, more by
  // sorting, which is a handful of steps to LDS against one for every candidate.
  __device__ __forceinline__ void order(int count) const
  {
    const int tid = (int)threadIdx.x;
    if (count <= 256) {
      if ((tid & ~63) < count) {
        const u64 own = tid < count ? box.c.entries[tid] : ~(u64)0;
        int rank      = 0;
#pragma unroll 4
        for (int i = 0; i < count; ++i) rank += box.c.entries[i] > own;
        if (tid < count) box.sorted[rank] = own;
      }
      __syncthreads();
      return;
    }
    int size = 512;
    while (size < count) size <<= 1;
    const u64 own = sort_one_each<THREADS>(tid < count ? box.c.entries[tid] : 0, size, box.sorted);
    if (tid < count) box.sorted[tid] = own;
    __syncthreads();
  }

  // The distance of an element from the maximum in parts of 48 / BINS powers of two.
  struct Bin {
    float c, r;
    // 0 for the maximum, and larger behind it
    __device__ __forceinline__ float place(float x) const
    {
      return fminf(fmaxf(fmaf(x, -c, r), 0.0f), (float)(BINS - 1));
    }
    __device__ __forceinline__ int operator()(float x) const { return (int)place(x); }
  };

  __device__ __forceinline__ Bin bins() const
  {
    const float per = (float)BINS / 48.0f;
    return Bin{(float)weight.c * per, (float)(weight.m * weight.c) * per};
  }

  // How many candidates are looked for where their number is not given.
  static constexpr int kNucleus = 12 * W;

  // From the candidates alone, if they are sure to hold all that is kept; false if they are not.  `sum`,
  // if there is a nucleus of the whole row, is the row's mass in fp32, right to within `off` of itself.
  // `base` and `known`: the exact mass of all values in the first `known` bins (see Bin).
  __device__ __forceinline__ bool from_candidates(const Found& f, double sum, double off, u64& base, int& known) const
  {
    const int tid = (int)threadIdx.x;
    int count     = f.count;
    if (!f.all) return false;
    if (set.greedy) {  // the largest entry
      u64 best = 0;
      for (int i = tid; i < count; i += THREADS) best = best > box.c.entries[i] ? best : box.c.entries[i];
      best = block_all<W>(best, [](u64 x, u64 y) { return x > y ? x : y; }, box.box);
      if (tid == 0) answer((int)entry_index(best), 1, 1);
      return true;
    }
    const bool by_k = set.top_k > 0;
    u32 tau        = f.tau;
    if (!by_k && tau != 0 && set.top_p < 1.0f && set.min_p <= 0.0f) {
      // a nucleus that is sure to hold more than the candidates needs no order of them.  All values in the bins
      // before that of tau are candidates.
      if (!(sum < 1e300) || !(off < 0.01)) return false;
      const Bin bin = bins();
      const int end = bin(value_of<float>(tau));
      u64 mass = 0, inside = 0;
      for (int i = tid; i < count; i += THREADS) {
        const float x = value_of<float>(entry_key(box.c.entries[i]));
        const u64 w   = weight(x);
        mass += w;
        inside += bin(x) < end ? w : 0;
      }
      mass = block_all<W>(mass, AddF{}, box.box);
      if ((double)mass < (double)set.top_p * sum * (1 - off)) {
        base  = block_all<W>(inside, AddF{}, box.box);
        known = end;
        return false;
      }
    }
    const int target = by_k ? set.top_k : kNucleus;
    if (count > target + target / 4 || count > THREADS) {  // fewer to put in order: one a thread at most
      tau   = thin_out<W>(box.c, count, target, tau, key32(f.max));
      count = box.c.count;
      if (count > THREADS) return false;
    }
    order(count);
    const int kept = by_k && set.top_k < count ? set.top_k : count;
    const u64 own  = tid < kept ? weight(value_of<float>(entry_key(box.sorted[tid]))) : 0;
    u64 all;
    const u64 before = block_before<W>(own, box.box, all);
    if (tid < kept) box.mass[tid] = own;
    // how many of the sorted candidates stay: at least `lo`, at most `hi`
    int lo = kept, hi = kept;
    bool open = !by_k && tau != 0;  // elements that are no candidates may belong to it
    if (set.top_p < 1.0f) {
      if (!open) {  // they are all there is
        const u64 goal = set.nucleus(all);
        lo = hi = block_all<W>(tid < kept && before < goal ? 1 : 0, AddF{}, box.ibox);
      } else {
        if (!(sum < 1e300) || !(off < 0.01)) return false;
        const double goal = (double)set.top_p * sum;
        lo = block_all<W>(tid < kept && (double)before < goal * (1 - off) ? 1 : 0, AddF{}, box.ibox);
        hi = block_all<W>(tid < kept && (double)before < goal * (1 + off) + 1 ? 1 : 0, AddF{}, box.ibox);
        // complete if the candidates' own mass passes the goal
        open = !((double)all >= goal * (1 + off) + 1);
        // for the other way: the last bin that is well inside, and the mass up to its end
        const Bin bin  = bins();
        const int mine = tid < kept ? bin(value_of<float>(entry_key(box.sorted[tid]))) : 0;
        const bool ends = tid + 1 < kept && mine != bin(value_of<float>(entry_key(box.sorted[tid + 1])));
        const int inside = block_all<W>(ends && (double)(before + own) < goal * 0.997 ? tid + 1 : 0, MaxI{}, box.ibox);
        if (inside > 0) {
          if (tid == inside - 1) {
            box.found[0] = before + own;
            box.found[1] = (u64)mine + 1;
          }
          __syncthreads();
          base  = box.found[0];
          known = (int)box.found[1];
        }
      }
    }
    if (set.min_p > 0.0f) {
      const int heavy = block_all<W>(tid < kept && own >= least ? 1 : 0, AddF{}, box.ibox);
      lo = lo < heavy ? lo : heavy;
      hi = hi < heavy ? hi : heavy;
      if (heavy < kept) open = false;  // what ranks behind the candidates weighs less still
    }
    lo = lo > 1 ? lo : 1;  // the first stays whatever top_p is
    if (lo != hi || open) return false;
    if (tid == lo - 1) box.last = before + own;
    __syncthreads();
    choose(lo, box.last);
    return true;
  }

  // The least value whose bin lies before b; NaN if there is none.  Bins fall as values rise.
  __device__ __forceinline__ float least_in(const Bin& bin, int b) const
  {
    u32 lo = key32(-3.402823466e38f), hi = key32(max);  // hi is one, and what lies before lo is none
    if (bin(max) >= b) return __builtin_nanf("");
    const u32 lane = threadIdx.x & 63;
    while (lo < hi) {  // 64 places between them at a time, all lanes alike
      const u32 step = (hi - lo) / 64 + 1;
      const u32 at   = hi - lo > lane * step ? lo + lane * step : hi;
      const u64 in   = __ballot(bin(value_of<float>(at)) < b);  // from some lane on
      const int from = in != 0 ? __builtin_ctzll(in) : 64;
      const u32 end  = from < 64 && hi - lo > from * step ? lo + from * step : hi;
      lo             = from > 0 ? lo + (from - 1) * step + 1 : lo;
      hi             = end;
    }
    return value_of<float>(lo);
  }

  static constexpr int kVectors = 4;                   // of a lane and segment
  static constexpr int kSegment = 64 * VEC * kVectors;     // elements that one wave adds up

  // A lane's vectors of one segment as they were loaded, with the mask's bits.
  struct Loaded {
    u32x4 w[kVectors];
    u32 bits;  // VEC of every vector
  };

  // g(segment, index of the first element, VEC elements) for every vector of the row that this wave has: the
  // waves take the segments in turn, and load the next one before they work on one.  What the mask
  // leaves out, or lies behind the row's end, is -inf; NaN is left as it is.
  template <class G>
  __device__ __forceinline__ void segments_of_wave(G g) const
  {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int whole = n / kSegment;
    const int words = (n + 31) >> 5;
    auto load = [&](int s) {
      Loaded l;
      l.bits = 0;
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        const int at = s * kSegment + (v * 64 + lane) * VEC;
        l.w[v]       = load16c(row + at);
        if (MASKED) l.bits |= (mask_bits(allowed, at, words) & ((1u << VEC) - 1)) << (v * VEC);
      }
      return l;
    };
    auto unpack = [&](const u32x4& w, u32 bits, float(&x)[VEC]) {
      static_for<VEC>([&](auto j) { x[j] = (float)In<T>::template get<j>(w); });
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (MASKED) x[j] = ((bits >> j) & 1u) != 0 ? x[j] : -kInf;
    };
    if (wave < whole) {
      Loaded now = load(wave);
      for (int s = wave; s < whole; s += W) {
        const Loaded next = load(s + W < whole ? s + W : s);
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
          float x[VEC];
          unpack(now.w[v], now.bits >> (v * VEC), x);
          g(s, s * kSegment + (v * 64 + lane) * VEC, x);
        }
        now = next;
      }
    }
    if (whole * kSegment < n && wave == whole % W) {  // the last, partly filled segment
#pragma unroll 1
      for (int v = 0; v < kVectors; ++v) {
        const int at = whole * kSegment + (v * 64 + lane) * VEC;
        float x[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          x[j] = at + j < n ? widen(row + at + j) : -kInf;
          x[j] = at + j < n && eligible(x[j], at + j) ? x[j] : -kInf;
        }
        g(whole, at, x);
      }
    }
  }

  // Without top_k, where what is kept is more than the candidates: one exact pass that adds up every
  // segment's weights.  For a nucleus a pass before it counts the elements by their distance from the
  // maximum; the counts say between which distances the nucleus has to end, and the few elements there are
  // put in order.  false if there are too many of them.
  __device__ __forceinline__ bool from_segments(double sum, double off, u64 base, int known) const
  {
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const int segments = (n + kSegment - 1) / kSegment;
    if (segments > SampleBox<W>::kSegments || weight.infinite) return false;
    const Bin bin      = bins();
    bool nucleus       = set.top_p < 1.0f;
    // what is kept whole, and what may be kept: values from here on (NaN: none)
    float above = -kInf, low = -kInf;
    if (nucleus) {
      if (!(sum < 1e300) || !(off < 0.01)) return false;
      u32* counts = reinterpret_cast<u32*>(&box.c);
      // (64 more for what does not count, one a lane, so that no two lanes meet there)
      static_assert(offsetof(CandidateBox<W>, bins) >= (BINS + 64) * sizeof(u32), "the bins fit into what is free");
      __syncthreads();
      for (int i = tid; i < BINS; i += THREADS) counts[i] = 0;
      __syncthreads();
      segments_of_wave([&](int, int, const float(&x)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) atomicAdd(&counts[x[j] > -kInf ? bin(x[j]) : BINS + lane], 1u);
      });
      __syncthreads();
      // Every thread has a few bins; the mass up to and with a bin, as if its elements lay in its middle.  That
      // would be far off for the few heaviest, whose mass is known.
      constexpr int EACH = BINS / THREADS;
      const double one   = (double)((u64)1 << weight.bits);
      double mass[EACH];
      double own = 0;
      u32 count[EACH];
#pragma unroll
      for (int e = 0; e < EACH; e += 4) {
        const u32x4 four = *reinterpret_cast<const u32x4*>(&counts[tid * EACH + e]);
#pragma unroll
        for (int f = 0; f < 4; ++f) count[e + f] = four[f];
      }
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int b   = tid * EACH + e;
        const float w = __builtin_amdgcn_exp2f(-((float)b + 0.5f) * (48.0f / BINS));
        mass[e]       = b >= known ? (double)count[e] * ((double)w * one) : 0.0;
        own += mass[e];
      }
      double ignored;
      double upto       = (double)base + block_before<W>(own, reinterpret_cast<double*>(box.box), ignored);
      const double goal = (double)set.top_p * sum;
      // Bins are 0.2 to 0.8 % wide, and the places of many values in theirs average out: to 1e-5 of the mass where
      // the values are fine, to 1e-4 and now and then 5e-4 for the few hundred values that bf16 has here.  What
      // falls short costs three to five times as much as the whole row, some hundred more to put in order 2 us.
      const double give = off + 5e-4;
      if (tid == 0) box.window[0] = box.window[1] = BINS;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int b       = tid * EACH + e;
        const double less = b == 0 ? -1.0 : upto;
        upto += mass[e];
        // the first bin that may hold the end, and the first that should lie behind it (one thread each); the
        // exact pass finds out whether that is so
        if (less < goal * (1 - give) && upto >= goal * (1 - give)) box.window[0] = b;
        if (less < goal * (1 + give) + 1 && upto >= goal * (1 + give) + 1) box.window[1] = b + 1;
      }
      __syncthreads();
      // bins before b0 are kept whole, b1 and later ones not at all
      const int b0 = box.window[0] > known ? box.window[0] : known, b1 = box.window[1];
      u32 in = 0;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int b = tid * EACH + e;
        if (b >= b0 && b < b1) in += count[e];
      }
      in = block_all<W>(in, AddF{}, reinterpret_cast<u32*>(box.ibox));
      // min_p may cut before the window: the nucleus then matters no more, if what min_p keeps has less mass
      if (set.min_p > 0.0f && fmaf(__builtin_amdgcn_logf(set.min_p), -(float)BINS / 48.0f, 2.0f) < (float)b0) nucleus = false;
      if (nucleus && in > (u32)CandidateBox<W>::kEntries) return false;
      if (tid == 0) {
        box.c.count = 0;
        box.last    = (u64)(goal * (1 - off));  // where the nucleus matters no more
      }
      above = least_in(bin, b0);
      low   = least_in(bin, b1);
    }
    __syncthreads();

    // the exact pass.  Every weight comes with the bits of 2^52, which are taken off a vector at a time.
    constexpr u64 kHead = 0x4330000000000000ull;
    u64 all = 0, sum_s = 0;
    int at_segment = -1;
    auto close     = [&]() {  // this wave's segment is complete
      if (at_segment < 0) return;
      const u64 w = wave_all(sum_s, AddF{});
      if (lane == 0) box.mass[at_segment] = w;
      sum_s = 0;
    };
    auto in_segment = [&](int s) {
      if (s == at_segment) return;
      close();
      at_segment = s;
    };
    if (nucleus) {
      segments_of_wave([&](int s, int at, const float(&x)[VEC]) {
        in_segment(s);
        u64 part = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const u64 w     = weight.raw(x[j]);
          const bool kept = x[j] >= above;
          all += w;
          part += kept ? w : kHead;
        }
        all -= VEC * kHead;
        sum_s += part - VEC * kHead;
        asm volatile("" : "+v"(sum_s), "+v"(all));  // the sums are formed here, not after the branches
        // where the values between lie, put down by the wave as a whole: one place is asked for
        u64 lanes[VEC];
        int hits = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          lanes[j] = __ballot(x[j] >= low && !(x[j] >= above));
          hits += __builtin_popcountll(lanes[j]);
        }
        if (hits == 0) return;
        int place = 0;
        if (lane == 0) place = atomicAdd(&box.c.count, hits);
        place = __builtin_amdgcn_readfirstlane(place);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (lanes[j] == 0) continue;
          const int to = __builtin_amdgcn_mbcnt_hi((u32)(lanes[j] >> 32), __builtin_amdgcn_mbcnt_lo((u32)lanes[j], place));
          if ((lanes[j] >> lane) & 1) box.c.entries[to] = (u64)(u32)(at + j);
          place += __builtin_popcountll(lanes[j]);
        }
      });
    } else if (least > 0) {
      segments_of_wave([&](int s, int, const float(&x)[VEC]) {
        in_segment(s);
        u64 part = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const u64 w = weight.raw(x[j]);
          part += w >= least + kHead ? w : kHead;
        }
        sum_s += part - VEC * kHead;
      });
    } else {
      segments_of_wave([&](int s, int, const float(&x)[VEC]) {
        in_segment(s);
        u64 part = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) part += weight.raw(x[j]);
        sum_s += part - VEC * kHead;
      });
    }
    close();
    __syncthreads();
    u64 total = block_all<W>(tid < segments ? box.mass[tid] : (u64)0, AddF{}, box.box);
    u64 last  = 0;  // the last entry kept of those between b0 and b1
    if (!nucleus && set.top_p < 1.0f && total >= box.last) return false;
    if (nucleus) {
      all            = block_all<W>(all, AddF{}, box.box);
      const u64 goal = set.nucleus(all);
      const int in   = box.c.count;
      u64* entries   = box.c.entries;
      auto entry_at  = [&](int i) {
        const u32 where = (u32)entries[i];
        return entry_of(key32(widen(row + where)), where);
      };
      int size = 64;
      while (size < in) size <<= 1;
      if (size <= THREADS) {
        const u64 own = sort_one_each<THREADS>(tid < in ? entry_at(tid) : 0, size, box.sorted);
        if (tid < in) entries[tid] = own;
        __syncthreads();
      } else {
        for (int i = tid; i < size; i += THREADS) entries[i] = i < in ? entry_at(i) : 0;
        sort_entries<THREADS>(entries, size);
      }
      constexpr int EACH = CandidateBox<W>::kEntries / THREADS;  // consecutive ones
      u64 w[EACH], mine = 0;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int i = tid * EACH + e;
        w[e]        = i < in ? weight(value_of<float>(entry_key(entries[i]))) : 0;
        mine += w[e];
      }
      u64 inside;
      u64 before = total + block_before<W>(mine, box.box, inside);
      // the nucleus ends where the counts said, or they were too coarse
      if (!(total < goal && total + inside >= goal)) return false;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int i = tid * EACH + e;
        if (i < in && before < goal) {
          atomicAdd((unsigned long long*)&box.mass[entry_index(entries[i]) / kSegment], (unsigned long long)w[e]);
          if (before + w[e] >= goal) {  // one thread
            box.last     = entries[i];
            box.found[0] = before + w[e];
            box.found[1] = w[e];
          }
        }
        before += w[e];
      }
      __syncthreads();
      last  = box.last;
      total = box.found[0];
      // min_p may cut deeper: that is left to the general way
      if (set.min_p > 0.0f && box.found[1] < least) return false;
    }
    // the segment, and in it the element, at which the mass passes the goal
    const u64 goal = set.goal(total);
    const u64 own  = tid < segments ? box.mass[tid] : 0;
    u64 t2;
    const u64 before = block_before<W>(own, box.box, t2);
    __syncthreads();
    if (before <= goal && before + own > goal) {
      box.found[0]  = before;
      box.window[0] = tid;
    }
    __syncthreads();
    const int s   = box.window[0];
    u64 upto      = box.found[0];
    constexpr int EACH = (kSegment + THREADS - 1) / THREADS;
    u64 w[EACH], mine = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int in = tid * EACH + e;
      const int i  = s * kSegment + in;
      w[e]         = 0;
      if (in < kSegment && i < n) {
        const float x = widen(row + i);
        if (eligible(x, i)) {
          w[e] = weight(x);
          if (nucleus) {
            if (!(x >= above) && !(x >= low && entry_of(key32(x), (u32)i) >= last)) w[e] = 0;
          } else if (w[e] < least) {
            w[e] = 0;
          }
        }
      }
      mine += w[e];
    }
    upto += block_before<W>(mine, box.box, t2);
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      if (upto <= goal && upto + w[e] > goal) answer(s * kSegment + tid * EACH + e, w[e], total);
      upto += w[e];
    }
    return true;
  }

  // Whatever the settings and the row are: sweeps for the cut by count and by mass (8 bits of the key
  // each), one for the total, and one in index order that ends at the token.
  __device__ __forceinline__ void in_general(u64 count) const
  {
    u64* bins = box.c.entries;
    // the cut in rank order: every element with a key above `key`, and with it up to index `last`
    u32 key       = 0;
    int last      = n;
    u64 take      = ~(u64)0;  // elements with the key itself
    u64 with      = 0;        // how many there are
    const u32 top = key_of<T>(max);
    if (set.top_k > 0 && (u64)set.top_k < count) {
      const Cut c = find_cut<T, THREADS, true>(
        row, n, top, (u64)set.top_k, [&](float x, int i) { return (u64)(eligible(x, i) ? 1 : 0); }, bins);
      key  = c.key;
      take = (u64)set.top_k - c.above;
      with = c.with;
    }
    if (set.top_p < 1.0f) {
      u64 all = 0;
      narrow_sweep<T, THREADS>(row, n, [&](float x, int i) {
        if (!eligible(x, i)) return;
        const u32 k = key_of<T>(x);
        if (k > key || (k == key && take == ~(u64)0)) all += weight(x);
      });
      all = block_all<W>(all, AddF{}, box.box);
      if (take != ~(u64)0) all += take * weight(value_of<T>(key));
      const u64 goal = set.nucleus(all);
      if (goal < all) {
        const Cut c = find_cut<T, THREADS, true>(
          row, n, top, goal, [&](float x, int i) { return eligible(x, i) ? weight(x) : (u64)0; }, bins);
        const u64 each = weight(value_of<T>(c.key));
        key            = c.key;
        take           = (goal - c.above + each - 1) / each;
        with           = c.with / each;
      }
    }
    if (take < with) {  // where the last of the equal elements is that is kept
      u64 seen = 0;
      ordered_sweep<T, THREADS, 2>(row, n, [&](int at, const float(&x)[2], int cnt) {
        u64 ties = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (j < cnt && key_of<T>(x[j]) == key && eligible(x[j], at + j)) ++ties;
        u64 all;
        u64 rank = seen + block_before<W>(ties, box.box, all);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (j < cnt && key_of<T>(x[j]) == key && eligible(x[j], at + j) && ++rank == take) box.found[0] = (u64)(at + j);
        seen += all;
        return seen < take;
      });
      __syncthreads();
      last = (int)box.found[0];
    }
    auto kept = [&](float x, int i) -> u64 {
      if (!eligible(x, i)) return 0;
      const u32 k = key_of<T>(x);
      if (k < key || (k == key && i > last)) return 0;
      const u64 w = weight(x);
      return w >= least ? w : 0;
    };
    u64 all = 0;
    narrow_sweep<T, THREADS>(row, n, [&](float x, int i) { all += kept(x, i); });
    all            = block_all<W>(all, AddF{}, box.box);
    const u64 goal = set.goal(all);
    u64 seen       = 0;
    ordered_sweep<T, THREADS, 2>(row, n, [&](int at, const float(&x)[2], int cnt) {
      u64 own[2], sum = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) sum += own[j] = j < cnt ? kept(x[j], at + j) : 0;
      u64 tile;
      u64 upto = seen + block_before<W>(sum, box.box, tile);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (upto <= goal && upto + own[j] > goal) answer(at + j, own[j], all);
        upto += own[j];
      }
      seen += tile;
      return seen <= goal;
    });
  }
};

template <class T, int W, int W_REST, bool MASKED>
__device__ __forceinline__ Row<T, W, W_REST, MASKED> row_of(const SampleArgs& a, int64_t r, SampleBox<W>& box,
                                                            const Settings& set, float max)
{
  Weights weight;
  weight.table    = box.table;
  weight.m        = (double)max;
  weight.c        = kLog2e / (double)set.temperature;
  weight.bits     = a.bits;
  weight.infinite = max == kInf;
  const u64 least = (u64)ceil((double)set.min_p * (double)((u64)1 << a.bits));
  return Row<T, W, W_REST, MASKED>{a, static_cast<const T*>(a.logits) + r * a.ld,
                                   MASKED ? a.allowed + r * a.ld_allowed : nullptr, box, set, weight, a.n_cols, max, least, r};
}

// A row that its candidates did not decide.
template <class T, int W, bool MASKED>
__device__ __forceinline__ void rest_of_row(const SampleArgs& a, const Settings& set, const Row<T, W, W, MASKED>& it,
                                            SampleBox<W>& box, const Undecided& rest)
{
  if (set.top_k <= 0 || set.top_k >= a.n_cols)
    if (it.from_segments(rest.mass, rest.off, rest.base, rest.known)) return;
  // the general way starts from the number of elements that count
  __syncthreads();
  u64 count = 0;
  narrow_sweep<T, 64 * W>(it.row, a.n_cols, [&](float x, int i) { count += it.eligible(x, i) ? 1 : 0; });
  count = block_all<W>(count, AddF{}, box.box);
  it.in_general(count);
}

// One workgroup per row.  One pass finds the maximum, the elements that rank first and, where a nucleus is
// asked for, the mass in fp32; that is enough wherever what is kept lies among some hundred elements.  With SPLIT a row
// that it does not decide is left to the second kernel, so that rows of 20 us and of 100 us do not take turns on the
// same CUs, and the pass that is bound by memory holds a third fewer registers.
template <class T, int W, int NV, int W_REST, bool MASKED, bool SPLIT>
__global__ __launch_bounds__(64 * W, MASKED && W == 4 ? 3 : 4) void sample_kernel(SampleArgs a)
{
  constexpr int THREADS = 64 * W;
  __shared__ SampleBox<W> box;
  maxima_ignore_nan();
  const int64_t r = block_of_grid();
  if (r >= a.n_rows) return;
  const int tid = (int)threadIdx.x;
  const int n   = a.n_cols;
  const Settings set(a, r);
  for (int i = tid; i < kTable; i += THREADS) box.table[i] = exp2(a.bits + (double)i / kTable);

  const bool sharp  = set.top_k > 0 && set.top_k <= 64 * W;
  const bool some   = set.top_p < 1.0f || set.min_p > 0.0f;
  const bool sum    = !sharp && set.top_p < 1.0f;
  const bool ranked = sharp || (some && set.top_k <= 0);
  const int target  = sharp ? set.top_k : (ranked ? Row<T, W, W_REST, MASKED>::kNucleus : 1);
  const float c     = (float)(kLog2e / (double)set.temperature);
  Running run;
  const Found f = stream_candidates<T, W, NV, MASKED ? Look::kMasked : Look::kReal, true>(
    static_cast<const T*>(a.logits) + r * a.ld, n, target, MASKED ? a.allowed + r * a.ld_allowed : nullptr, c, box.c, run, sum);
  if (!(f.max > -kInf)) {  // nothing to choose from
    if (tid == 0) {
      if (SPLIT) a.todo[r] = 0;
      a.token[r] = -1;
      if (a.logprob != nullptr) a.logprob[r] = -kInf;
    }
    return;
  }
  const auto it = row_of<T, W, W_REST, MASKED>(a, r, box, set, f.max);
  // The mass in fp32, and how far it may be off: n / THREADS additions in order and some 64 roundings of a term,
  // as for a log-sum-exp, and the rounding of the reference that the terms are taken against; doubled.
  Undecided rest{0, 0.0, 0.0, f.max, 0};
  if (sum) {
    rest.mass = block_all<W>(run.against(f.max, c), AddF{}, reinterpret_cast<double*>(box.box)) * (double)((u64)1 << a.bits);
    rest.off  = ((double)n / THREADS + 256.0 + fabs(it.weight.m * it.weight.c)) * 0x1p-23;
  }
  const bool done = ranked && it.from_candidates(f, rest.mass, rest.off, rest.base, rest.known);
  if constexpr (SPLIT) {
    if (tid != 0) return;
    a.todo[r] = done ? 0 : 1;
    if (!done) a.rest[r] = rest;
  } else {
    if (done) return;
    __syncthreads();
    rest_of_row<T, W, MASKED>(a, set, it, box, rest);
  }
}

// The rows that are left: workgroup b takes the b-th of them, which it counts out itself.  Workgroups are dealt to
// the CUs in order, so by their own numbers the rows that are left would meet on some CUs while others had none (1024 x
// 131072 f16, 237 rows left: 139 us, counted out 80, and 74 now).  Without COUNTED, which is for so many rows that they even out,
// it takes its own row.
template <class T, int W, bool MASKED, bool COUNTED>
__global__ __launch_bounds__(64 * W, 4) void sample_rest_kernel(SampleArgs a)
{
  constexpr int THREADS = 64 * W;
  __shared__ SampleBox<W> box;
  const int tid = (int)threadIdx.x;
  int64_t r     = block_of_grid();
  if constexpr (COUNTED) {
    int skip = (int)r;  // rows left that come before the one wanted
    int base = 0, all = 0, before = 0, left = 0;
    for (; base < a.n_rows; base += THREADS) {
      left   = base + tid < a.n_rows ? (a.todo[base + tid] != 0 ? 1 : 0) : 0;
      before = block_before<W>(left, box.ibox, all);
      if (all > skip) break;  // the same in every thread
      skip -= all;
    }
    if (base >= a.n_rows) return;
    if (left != 0 && before == skip) box.window[2] = base + tid;
    __syncthreads();
    r = box.window[2];
  } else {
    if (r >= a.n_rows || a.todo[r] == 0) return;
  }
  for (int i = tid; i < kTable; i += THREADS) box.table[i] = exp2(a.bits + (double)i / kTable);
  __syncthreads();
  const Undecided rest = a.rest[r];
  const Settings set(a, r);
  rest_of_row<T, W, MASKED>(a, set, row_of<T, W, W, MASKED>(a, r, box, set, rest.max), box, rest);
}

constexpr int kCounted = 8192;

template <class T, bool MASKED>
void launch_as(const SampleArgs& a, hipStream_t st)
{
  const dim3 grid = grid_of(a.n_rows);
  if ((int64_t)a.n_cols / In<T>::VEC <= 1024) {
    hipLaunchKernelGGL((sample_kernel<T, 4, 4, 4, MASKED, false>), grid, dim3(256), 0, st, a);
  } else if (a.n_rows <= cu_count()) {
    // every row has a CU: it wants all the loads that a CU can have in flight, and a second kernel would only wait
    // for the slowest row of the first (256 x 131072 bf16, every kind of row: in two kernels 12 us more)
    hipLaunchKernelGGL((sample_kernel<T, 16, 4, 16, MASKED, false>), grid, dim3(1024), 0, st, a);
  } else {
    // Two rows at a time on a CU hide each other's steps, and the few that their candidates do not decide, which
    // take many times as long, are dealt out anew (1024 x 131072 f16, nucleus, as first built: 153 us, in one kernel
    // 199; now 146).
    hipLaunchKernelGGL((sample_kernel<T, 8, 4, 16, MASKED, true>), grid, dim3(512), 0, st, a);
    if (a.n_rows <= kCounted)
      hipLaunchKernelGGL((sample_rest_kernel<T, 16, MASKED, true>), grid, dim3(1024), 0, st, a);
    else
      hipLaunchKernelGGL((sample_rest_kernel<T, 16, MASKED, false>), grid, dim3(1024), 0, st, a);
  }
}

template <class T>
int launch(const SampleArgs& a, hipStream_t st)
{
  if (a.allowed != nullptr)
    launch_as<T, true>(a, st);
  else
    launch_as<T, false>(a, st);
  return hipGetLastError() == hipSuccess ? RMI_OK : RMI_ERR_LAUNCH;
}

}  // namespace
}  // namespace logits
}  // namespace rmi

extern "C" {

size_t rmi_sample_workspace_bytes(int dtype, int64_t n_rows, int64_t n_cols)
{
  using namespace rmi::logits;
  if (!is_logits_dtype(dtype) || check_shape(n_rows, n_cols, n_cols) != RMI_OK || n_rows == 0) return 0;
  return RMI_WORKSPACE_TICKET_BYTES + (size_t)n_rows * (sizeof(Undecided) + sizeof(int32_t));
}

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
               void* workspace,
               size_t workspace_bytes,
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
  if (workspace == nullptr || workspace_bytes < rmi_sample_workspace_bytes(dtype, n_rows, n_cols) ||
      !rmi::logits::aligned(workspace, 16))
    return RMI_ERR_WORKSPACE;
  SampleArgs a{};
  a.rest        = reinterpret_cast<Undecided*>(static_cast<char*>(workspace) + RMI_WORKSPACE_TICKET_BYTES);
  a.logits      = logits;
  a.allowed     = allowed;
  a.todo        = reinterpret_cast<int32_t*>(a.rest + n_rows);
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
