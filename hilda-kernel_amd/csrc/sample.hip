// Token sampling with temperature, top-k, top-p and min-p from given uniform
// numbers, and the sampled token's log-probability, for gfx950.
//
// Per row of V logits x, with z = x / T and p = e^(z - max z):
//   order    x descending, the lower index first among equal x
//   top-k    the first k of that order
//   top-p    of those the shortest prefix whose mass is >= top_p times theirs
//   min-p    of those the ones with p >= min_p
//   id       the first kept index i, in index order, with
//            sum_{kept j <= i} p_j > u * sum_{kept j} p_j
//   logp     z_id - log sum_j e^(z_j) over ALL tokens (the policy's
//            log-probability, as selective log-softmax gives it)
//
// Nothing is sorted. The kept set is a threshold x* and a number of ties at
// x* that are kept (the first ones by index), found by selection:
//   pass 1  max and log-sum-exp (fp32, online)
//   pass 2  counts and masses of the logits in kBins bins, linear in max - x
//           (only with top-k or top-p); the bin that holds the cut
//   pass 3  the same over ranges of ordered keys inside that bin, 11 bits at a
//           time, down to one value: x* and how many of its ties are kept
//   pass 4  the kept mass of each wave's run of indices; the run that holds
//           u * total is walked by the whole block
// Later passes hit L2 / the Infinity Cache.
//
// Masses are fp64: with 32-bit ones the running sums of a flat row of 1e5
// tokens (steps of 1e-5 of the total) would be off by a percent of a step, and
// one draw in a hundred would go to a neighbour. In bins they are fixed point
// (63 - log2 V bits, at most 43), so that LDS atomics in any order give the
// same sums. e^d is a polynomial in fp64: fp64 FMAs run at the rate of plain
// fp32 ones on this part.
//
// A row without a distribution (a NaN, a +inf, nothing above -inf) or with
// parameters out of range gives id -1 and logp NaN.
#include "hk_common.h"
#include "../../include/hilda_kernel_amd.h"

#include <algorithm>
#include <type_traits>

namespace hk {
namespace {

typedef unsigned long long u64;

constexpr int kLanes = 1024;
constexpr int kWaves = kLanes / kWave;
constexpr int kBins = 2048;
// the linear bins cover max - x < kRange * T; beyond it is one bin
constexpr double kRange = 24;
constexpr double kTempMin = 0x1p-64, kTempMax = 0x1p64;

// A setting of every row, or one each.
struct Setting {
  const float* rows;
  double all;
};
struct SampleArgs {
  int64_t* ids;
  float* logp;
  const void* logits;
  const float* u;
  Setting temperature, top_p, min_p;
  const void* top_k_rows;  // int32 / int64 by top_k_wide
  int top_k_wide;
  int64_t top_k;
  int64_t ld;
  int cols;
  int seg;        // columns of a wave's run, a multiple of 64 vectors
  double magic;   // 2^(52 - b): e + magic holds e in b fixed-point bits
};

__device__ __forceinline__ double setting(const Setting& s, int64_t row) { return s.rows ? s.rows[row] : s.all; }

struct Series {
  double c[13];
  constexpr Series() : c() {  // (ln 2)^k / k!
    c[0] = 1.0;
    for (int k = 1; k < 13; ++k) c[k] = c[k - 1] * 0.693147180559945309417 / k;
  }
};
constexpr Series kExp2Series;

// 2^y, y <= 0 (0 below -1074), by Taylor's series of e^(r ln 2) for |r| <= 1/2
// to degree 12 (remainder (ln2 / 2)^13 / 13! = 1.7e-16)
__device__ __forceinline__ double exp2_f64(double y) {
  y = fmax(y, -1100.0);
  const double n = rint(y), r = y - n;
  double p = kExp2Series.c[12];
#pragma unroll
  for (int k = 11; k >= 0; --k) p = fma(r, p, kExp2Series.c[k]);
  return ldexp(p, (int)n);
}

// order-preserving key of a float that came from T, without T's unused bits; -0 equals 0
template <typename T> struct KeyShift;
template <> struct KeyShift<float> { static constexpr int v = 0; };
template <> struct KeyShift<_Float16> { static constexpr int v = 13; };
template <> struct KeyShift<__bf16> { static constexpr int v = 16; };
__device__ __forceinline__ uint32_t key32(float x) {
  uint32_t b = f32_bits(x);
  if (b == 0x80000000u) b = 0;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
template <typename T> __device__ __forceinline__ uint32_t key_of(float x) { return key32(x) >> KeyShift<T>::v; }
template <typename T> __device__ __forceinline__ float value_of(uint32_t key) {
  constexpr int S = KeyShift<T>::v;
  const uint32_t k = (uint32_t)((uint64_t)key << S);
  if (k & 0x80000000u) return bits_f32(k ^ 0x80000000u);
  return bits_f32(~(k | (uint32_t)((1ull << S) - 1)));
}

// VEC logits from column `col`; -inf past the row's end
template <typename T, int VEC>
__device__ __forceinline__ void load_vals(const T* row, int col, int cols, float (&v)[VEC]) {
  if (col + VEC <= cols) {
    unpack(load_pack_any<T, VEC>(row + col), v);
    return;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = col + i < cols ? to_f32<T>(row[col + i]) : -INFINITY;
}

template <typename X> __device__ __forceinline__ X wave_total(X v) {
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) v += __shfl_xor(v, o, kWave);
  return v;
}
template <typename X> __device__ __forceinline__ X wave_scan(X v) {  // inclusive
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) {
    const X t = __shfl_up(v, o, kWave);
    if (lane >= o) v += t;
  }
  return v;
}
// sum over the threads before this one; `tmp` holds kWaves values
template <typename X> __device__ __forceinline__ X block_before(X v, X* tmp) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const X incl = wave_scan(v);
  __syncthreads();
  if (lane == kWave - 1) tmp[wave] = incl;
  __syncthreads();
  X before = incl - v;
  for (int i = 0; i < wave; ++i) before += tmp[i];
  return before;
}

struct Hist {
  u64 mass[kBins];
  uint32_t count[kBins];
};
struct Shared {
  Hist linear, fine;
  double dtmp[kWaves];
  u64 ltmp[kWaves];
  uint32_t utmp[kWaves];
  float m[kWaves], z[kWaves];
  // the bin that holds a cut
  int bin;
  uint32_t cnt_before;
  u64 mass_before;
  int found, last;
};

__device__ __forceinline__ void clear(Hist& h) {
  for (int i = threadIdx.x; i < kBins; i += kLanes) h.mass[i] = 0, h.count[i] = 0;
}

// The bin whose running count passes `count_target` (by count), or whose running mass reaches `mass_target`; what lies
// before it goes to sh. Exactly one bin qualifies. Ends with a barrier.
__device__ __forceinline__ void find_bin(const Hist& h, Shared& sh, bool by_count, uint32_t count_target,
                                         u64 mass_target) {
  static_assert(kBins == 2 * kLanes, "two bins a thread");
  __syncthreads();
  if (threadIdx.x == 0) sh.bin = kBins - 1, sh.cnt_before = 0, sh.mass_before = 0;
  const int b = 2 * threadIdx.x;
  const uint32_t c0 = h.count[b], c1 = h.count[b + 1];
  const u64 m0 = h.mass[b], m1 = h.mass[b + 1];
  uint32_t cb = block_before<uint32_t>(c0 + c1, sh.utmp);
  u64 mb = block_before<u64>(m0 + m1, sh.ltmp);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t c = i ? c1 : c0;
    const u64 m = i ? m1 : m0;
    const bool here = by_count ? cb < count_target && count_target - cb <= c
                               : mb < mass_target && mass_target - mb <= m;
    if (here) sh.bin = b + i, sh.cnt_before = cb, sh.mass_before = mb;
    cb += c;
    mb += m;
  }
  __syncthreads();
}

// A cut: logits above x are kept, and the first `ties` of those equal to x
// (of `equal` in the row).
struct Cut {
  float x;
  uint32_t ties, equal;
  u64 mass;  // fixed-point mass of the kept ones (with masses only)
};

template <typename T>
struct Row {
  static constexpr int VEC = 16 / sizeof(T);
  const T* x;
  int cols, seg;
  float max;        // of the row
  double to_log2;   // log2(e) / T
  float bin_step;   // kBins / (kRange T)
  double magic;

  __device__ __forceinline__ double mass(float v) const { return exp2_f64(((double)v - (double)max) * to_log2); }
  __device__ __forceinline__ u64 fixed(double e) const {
    return __builtin_bit_cast(u64, e + magic) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ int bin_of(float v) const {
    const float d = (max - v) * bin_step;
    return d < (float)(kBins - 1) ? (int)d : kBins - 1;
  }
  // f(values, column) over this wave's run of columns
  template <typename F> __device__ __forceinline__ void walk(F&& f) const {
    const int lane = threadIdx.x % kWave;
    const int c0 = (int)(threadIdx.x / kWave) * seg, c1 = min(cols, c0 + seg);
    for (int c = c0 + lane * VEC; c < c1; c += kWave * VEC) {
      float v[VEC];
      load_vals<T, VEC>(x, c, cols, v);
      f(v, c);
    }
  }

  __device__ __forceinline__ void fill_linear(Shared& sh, bool masses) const {
    clear(sh.linear);
    __syncthreads();
    uint32_t low = 0;
    u64 low_mass = 0;
    walk([&](const float (&v)[VEC], int c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (c + i >= cols) continue;
        const int b = bin_of(v[i]);
        const u64 e = masses ? fixed(mass(v[i])) : 0;
        if (b < kBins - 1) {
          atomicAdd(&sh.linear.count[b], 1u);
          if (masses) atomicAdd(&sh.linear.mass[b], e);
        } else {
          ++low;
          low_mass += e;
        }
      }
    });
    low = wave_total(low);
    low_mass = wave_total(low_mass);
    if (threadIdx.x % kWave == 0) {
      atomicAdd(&sh.linear.count[kBins - 1], low);
      if (masses) atomicAdd(&sh.linear.mass[kBins - 1], low_mass);
    }
  }

  // The cut at `k` logits (by count) or at mass `tau` (fixed point), from the linear bins.
  __device__ __forceinline__ Cut find_cut(Shared& sh, bool by_count, uint32_t k, u64 tau, bool masses) const {
    find_bin(sh.linear, sh, by_count, k, tau);
    const int lin = sh.bin;
    uint32_t cnt = sh.cnt_before;
    u64 above = sh.mass_before;
    // keys that the bin can hold, with the roundings of bin_of to spare
    const double width = 1.0 / (double)bin_step, slack = 0x1p-21;
    const float hi = (float)((double)max - lin * width * (1 - slack));
    const float lo = (float)((double)max - (lin + 1) * width * (1 + slack));
    uint32_t khi = lin == 0 ? key_of<T>(max) : ::min(key_of<T>(max), key_of<T>(hi) + 1);
    const uint32_t kl = key_of<T>(lo);
    uint32_t klo = lin == kBins - 1 || kl == 0 ? 0 : kl - 1;
    Cut cut = {-INFINITY, 0xffffffffu, 0, 0};
    // 32 bits of key in turns of 11
    for (int turn = 0; turn < 3; ++turn) {
      int s = 0;
      while (((khi - klo) >> s) >= (uint32_t)kBins) ++s;
      __syncthreads();
      clear(sh.fine);
      __syncthreads();
      walk([&](const float (&v)[VEC], int c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          if (c + i >= cols || bin_of(v[i]) != lin) continue;
          const uint32_t key = key_of<T>(v[i]);
          if (key < klo || key > khi) continue;
          const uint32_t b = (khi - key) >> s;
          atomicAdd(&sh.fine.count[b], 1u);
          if (masses) atomicAdd(&sh.fine.mass[b], fixed(mass(v[i])));
        }
      });
      find_bin(sh.fine, sh, by_count, k - cnt, tau - above);
      const uint32_t b = (uint32_t)sh.bin;
      cnt += sh.cnt_before;
      above += sh.mass_before;
      khi -= b << s;
      if (s == 0) {
        cut.x = value_of<T>(khi);
        cut.equal = sh.fine.count[b];
        const u64 each = masses ? fixed(mass(cut.x)) : 0;
        // (by mass: the bin holds equal * each >= tau - above > 0)
        cut.ties = by_count ? k - cnt : (uint32_t)((tau - above + each - 1) / each);
        cut.mass = above + each * cut.ties;
        break;
      }
      klo = ::max(klo, khi - ((1u << s) - 1));
    }
    return cut;
  }
};

template <typename T>
__global__ __launch_bounds__(kLanes) void sample_kernel(SampleArgs g) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ Shared sh;
  const int64_t row = blockIdx.x;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const double temp = setting(g.temperature, row), top_p = setting(g.top_p, row), min_p = setting(g.min_p, row);
  const float u = g.u[row];
  int64_t top_k = g.top_k;
  if (g.top_k_rows)
    top_k = g.top_k_wide ? static_cast<const int64_t*>(g.top_k_rows)[row]
                         : static_cast<const int32_t*>(g.top_k_rows)[row];

  Row<T> r;
  r.x = static_cast<const T*>(g.logits) + row * g.ld;
  r.cols = g.cols;
  r.seg = g.seg;
  r.magic = g.magic;
  const float c = (float)(1.4426950408889634074 / temp);

  // pass 1: the maximum and the sum of e^(z - max), over all tokens
  float m = -INFINITY, z = 0.f;
  r.walk([&](const float (&v)[VEC], int) {
    float n = v[0];
#pragma unroll
    for (int i = 1; i < VEC; ++i) n = fmaxf(n, v[i]);
    n = fmaxf(m, n);
    const float ref = n == -INFINITY ? 0.f : n;
    z *= exp2_fast((m - ref) * c);
#pragma unroll
    for (int i = 0; i < VEC; ++i) z += exp2_fast((v[i] - ref) * c);
    m = n;
  });
  {
    const float wm = wave_max(m), ref = wm == -INFINITY ? 0.f : wm;
    const float wz = wave_sum(z * exp2_fast((m - ref) * c));
    if (lane == 0) sh.m[wave] = wm, sh.z[wave] = wz;
  }
  __syncthreads();
  m = -INFINITY;
  for (int i = 0; i < kWaves; ++i) m = fmaxf(m, sh.m[i]);
  z = 0.f;
  for (int i = 0; i < kWaves; ++i) z += sh.m[i] == -INFINITY ? sh.z[i] : sh.z[i] * exp2_fast((sh.m[i] - m) * c);
  // (a NaN, a +inf or nothing above -inf leaves z NaN or 0)
  const bool fine = z > 0.f && z < INFINITY && m < INFINITY && temp >= kTempMin && temp <= kTempMax && u >= 0.f &&
                    u <= 1.f && top_p == top_p && min_p == min_p;
  if (!fine) {
    if (threadIdx.x == 0) g.ids[row] = -1, g.logp[row] = __builtin_nanf("");
    return;
  }
  r.max = m;
  r.to_log2 = 1.4426950408889634074 / temp;
  r.bin_step = (float)(kBins / (kRange * temp));

  // passes 2 and 3: the cut of top-k and top-p
  Cut cut = {-INFINITY, 0xffffffffu, 0, 0};
  const bool by_k = top_k > 0 && top_k < g.cols, by_p = top_p < 1.0;
  if (by_k || by_p) {
    r.fill_linear(sh, by_p);
    if (by_k) cut = r.find_cut(sh, true, (uint32_t)top_k, 0, by_p);
    if (by_p) {
      u64 total = cut.mass;
      if (!by_k) {
        __syncthreads();
        u64 t = wave_total(sh.linear.mass[2 * threadIdx.x] + sh.linear.mass[2 * threadIdx.x + 1]);
        if (lane == 0) sh.ltmp[wave] = t;
        __syncthreads();
        total = 0;
        for (int i = 0; i < kWaves; ++i) total += sh.ltmp[i];
        __syncthreads();
      }
      const u64 tau = min(total, max((u64)1, (u64)ceil(fmax(top_p, 0.0) * (double)total)));
      const Cut p = r.find_cut(sh, false, 0, tau, true);
      if (!by_k || p.x > cut.x) cut = p;
      else if (p.x == cut.x && p.ties < cut.ties) cut.ties = p.ties;
    }
  }
  if (min_p > 0.0) {
    // e^((x - max) / T) >= min_p, as the smallest float that satisfies it
    const double least = (double)m + temp * log(fmin(min_p, 1.0));
    float f = (float)least;
    if ((double)f < least) f = nextafterf(f, INFINITY);
    if (f > cut.x) cut = {f, 0xffffffffu, 0, 0};
  }
  const bool all_ties = cut.ties >= cut.equal;  // no count: every logit >= x is kept

  // pass 4: the kept mass of each wave's run
  double mass = 0.0;
  uint32_t ties = 0;
  r.walk([&](const float (&v)[VEC], int) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (all_ties ? v[i] >= cut.x : v[i] > cut.x) mass += r.mass(v[i]);
      else if (v[i] == cut.x) ++ties;
    }
  });
  mass = wave_total(mass);
  ties = wave_total(ties);
  __syncthreads();
  if (lane == 0) sh.dtmp[wave] = mass, sh.utmp[wave] = ties;
  if (threadIdx.x == 0) sh.found = kLanes, sh.last = -1;
  __syncthreads();
  const double each = all_ties ? 0.0 : r.mass(cut.x);
  double total = 0.0;
  uint32_t seen = 0;
  double runs[kWaves];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const uint32_t t = sh.utmp[w], left = cut.ties - min(cut.ties, seen);
    seen += t;
    runs[w] = sh.dtmp[w] + each * (double)min(left, t);
    total += runs[w];
  }
  const double target = (double)u * total;
  int run = -1;
  double base = 0.0, cum = 0.0;
  uint32_t base_ties = 0;
  seen = 0;
  bool hit = false;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (!hit && runs[w] > 0.0) run = w, base = cum, base_ties = seen;  // (the last one with any mass, if none passes)
    cum += runs[w];
    hit = hit || cum > target;
    seen += sh.utmp[w];
  }
  __syncthreads();

  // the run that holds the target: a stretch of columns a thread
  const int c0 = run * g.seg, c1 = min(g.cols, c0 + g.seg);
  const int per = (g.seg + kLanes - 1) / kLanes;
  const int t0 = c0 + (int)threadIdx.x * per, t1 = min(c1, t0 + per);
  ties = 0;
  if (!all_ties)
    for (int i = t0; i < t1; ++i) ties += to_f32<T>(r.x[i]) == cut.x ? 1 : 0;
  const uint32_t ties_before = base_ties + (all_ties ? 0 : block_before<uint32_t>(ties, sh.utmp));
  auto kept = [&](float v, uint32_t& rank) {
    if (all_ties) return v >= cut.x;
    if (v == cut.x) return rank++ < cut.ties;
    return v > cut.x;
  };
  mass = 0.0;
  uint32_t rank = ties_before;
  for (int i = t0; i < t1; ++i) {
    const float v = to_f32<T>(r.x[i]);
    if (kept(v, rank)) mass += r.mass(v);
  }
  const double before = base + block_before<double>(mass, sh.dtmp);
  if (before + mass > target && mass > 0.0) atomicMin(&sh.found, (int)threadIdx.x);
  if (mass > 0.0) atomicMax(&sh.last, (int)threadIdx.x);
  __syncthreads();
  const int who = sh.found < kLanes ? sh.found : sh.last;
  if ((int)threadIdx.x == who) {
    double s = before;
    int id = -1;
    rank = ties_before;
    for (int i = t0; i < t1; ++i) {
      const float v = to_f32<T>(r.x[i]);
      if (!kept(v, rank)) continue;
      const double e = r.mass(v);
      if (e > 0.0) id = i;
      s += e;
      if (id == i && s > target) break;
    }
    g.ids[row] = id;
    g.logp[row] = (float)(((double)to_f32<T>(r.x[id]) - (double)m) / temp) - log_fast(z);
  }
}

}  // namespace
}  // namespace hk

using namespace hk;

extern "C" {

int hk_sample(int64_t* ids, float* logp, const void* logits, const float* u, int64_t rows, int64_t cols, int64_t ld,
              const float* temperature_rows, double temperature, const void* top_k_rows, int top_k_type, int64_t top_k,
              const float* top_p_rows, double top_p, const float* min_p_rows, double min_p, int dtype,
              hk_stream_t stream) {
  HK_REQUIRE(dtype == kF32 || dtype == kF16 || dtype == kBF16, "invalid dtype code %d", dtype);
  HK_REQUIRE(rows >= 0 && cols > 0, "invalid shape rows=%lld cols=%lld", (long long)rows, (long long)cols);
  HK_REQUIRE(cols <= (1 << 30) && rows < (1LL << 31), "rows=%lld cols=%lld too large", (long long)rows,
             (long long)cols);
  HK_REQUIRE(ld >= cols, "row stride smaller than cols");
  HK_REQUIRE(temperature_rows || (temperature >= kTempMin && temperature <= kTempMax),
             "temperature %g is not in [2^-64, 2^64]", temperature);
  HK_REQUIRE(top_p_rows || (top_p >= 0 && top_p <= 1), "top_p %g is not in [0, 1]", top_p);
  HK_REQUIRE(min_p_rows || (min_p >= 0 && min_p <= 1), "min_p %g is not in [0, 1]", min_p);
  HK_REQUIRE(!top_k_rows || top_k_type == HK_I32 || top_k_type == HK_I64, "top_k must be int32 or int64, got code %d",
             top_k_type);
  if (rows == 0) return HK_OK;
  HK_REQUIRE(ids && logp && logits && u, "null pointer argument");
  SampleArgs g = {};
  g.ids = ids;
  g.logp = logp;
  g.logits = logits;
  g.u = u;
  g.temperature = {temperature_rows, temperature};
  g.top_p = {top_p_rows, top_p};
  g.min_p = {min_p_rows, min_p};
  g.top_k_rows = top_k_rows;
  g.top_k_wide = top_k_type == HK_I64;
  g.top_k = top_k;
  g.ld = ld;
  g.cols = (int)cols;
  int log2_cols = 0;
  while ((1LL << log2_cols) < cols) ++log2_cols;
  g.magic = (double)(1ULL << (52 - std::min(43, 63 - log2_cols)));
  auto launch = [&](auto tag) {
    using T = decltype(tag);
    const int64_t step = (int64_t)kWave * (16 / sizeof(T));
    g.seg = (int)(cdiv(cdiv(cols, (int64_t)kWaves), step) * step);
    hipLaunchKernelGGL((sample_kernel<T>), dim3((unsigned)rows), dim3(kLanes), 0, (hipStream_t)stream, g);
    return check_launch("sample_kernel");
  };
  if (dtype == kF32) return launch(float{});
  if (dtype == kF16) return launch(_Float16{});
  return launch(__bf16{});
}

}  // extern "C"
