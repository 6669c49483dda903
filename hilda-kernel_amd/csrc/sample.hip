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
// x* that are kept (the first ones by index), found by selection. A row is cut
// into runs of 2048 columns, its runs are dealt to the waves of a few blocks,
// and up to five launches follow each other (the later ones read the row from
// the Infinity Cache):
//   scan  max and log-sum-exp (fp32); for a row without filters the fp64 mass
//         of each run instead
//   hist  counts, and for top-p masses, in kBins bins linear in max - x
//   cut   the bins of a row's blocks together; the bin that holds the cut; if
//         several values may lie in it, the same over ranges of ordered keys,
//         11 bits at a time, until one is left: x* and how many ties are kept
//   mass  the kept mass of each run
//   pick  the run that u * total falls into, and the token inside it
// A call whose settings are numbers launches those it needs: scan and pick
// without filters, scan, mass and pick with min-p alone.
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

constexpr int kRun = 2048;            // columns of a run: 32 a lane
constexpr int kLaneCols = kRun / kWave;
constexpr int kLanes = 512;           // threads of a block (pick: kPickLanes)
constexpr int kWaves = kLanes / kWave;
constexpr int kPickLanes = 256;
constexpr int kMaxSplit = 16;         // blocks a row
constexpr int kBins = 2048;
// the linear bins cover max - x < kRange * T; beyond it is one bin
constexpr double kRange = 24;
constexpr double kTempMin = 0x1p-64, kTempMax = 0x1p64;
constexpr int kMaxQuarters = 1024;    // quarter maxima that a bound on the k-th logit is taken from

// A setting of every row, or one each.
struct Setting {
  const float* rows;
  double all;
};
struct Hist {
  u64 mass[kBins];
  uint32_t count[kBins];
};
// A cut: logits above x are kept, and the first `ties` of those equal to x
// (of `equal` in the row; all of them if ties >= equal).
struct Cut {
  float x;
  uint32_t ties, equal;
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
  int cols, runs;  // runs of a row
  int split;       // blocks of a row
  double magic;    // 2^(52 - b): e + magic holds e in b fixed-point bits
  // workspace
  float *part_max, *part_sum;  // [rows][split]
  float* quarters;             // [rows][4 runs] maxima of 512 columns
  double* run_mass;            // [rows][runs]
  uint32_t* run_ties;
  float* run_max;
  Hist* hist;                  // [rows][split], split > 1
  Cut* cuts;                   // [rows]
};

__device__ __forceinline__ double setting(const Setting& s, int64_t row) { return s.rows ? s.rows[row] : s.all; }

// What a row asks for.
struct Asked {
  double temp, top_p, min_p;
  int64_t top_k;
  bool by_k, by_p, open;  // open: no filter at all
  bool in_range;
};
__device__ __forceinline__ Asked asked(const SampleArgs& g, int64_t row) {
  Asked a;
  a.temp = setting(g.temperature, row);
  a.top_p = setting(g.top_p, row);
  a.min_p = setting(g.min_p, row);
  a.top_k = g.top_k;
  if (g.top_k_rows)
    a.top_k = g.top_k_wide ? static_cast<const int64_t*>(g.top_k_rows)[row]
                           : static_cast<const int32_t*>(g.top_k_rows)[row];
  a.by_k = a.top_k > 0 && a.top_k < g.cols;
  a.by_p = a.top_p < 1.0;
  a.open = !a.by_k && !a.by_p && !(a.min_p > 0.0);
  const float u = g.u[row];
  a.in_range = a.temp >= kTempMin && a.temp <= kTempMax && u >= 0.f && u <= 1.f && a.top_p == a.top_p &&
               a.min_p == a.min_p;
  return a;
}

// 2^y for y <= 0: y = n + r, |r| <= 1/2 (n from the low bits of y + 1.5 * 2^52), and for 2^r the polynomial of degree
// 10 that interpolates it at the Chebyshev nodes of [-1/2, 1/2] (relative error 3.2e-16). y = d * k with one rounding.
// 0 below y = -1080; NaN stays NaN.
__device__ __forceinline__ double exp2_product(double d, double k) {
  constexpr double kShift = 6755399441055744.0;
  constexpr double c[11] = {1.0,
                            0.69314718055995,
                            0.24022650695910097,
                            0.05550410866444772,
                            0.009618129107606888,
                            0.0013333558230164974,
                            0.0001540353044173605,
                            1.5252657260200837e-05,
                            1.321544258792169e-06,
                            1.0208690299958306e-07,
                            7.072585949269223e-09};
  const double t = fma(d, k, kShift);
  const double r = fma(d, k, -(t - kShift));
  double p = c[10];
#pragma unroll
  for (int i = 9; i >= 0; --i) p = fma(p, r, c[i]);
  const double e = __builtin_amdgcn_ldexp(p, (int)__builtin_bit_cast(u64, t));
  return t < kShift - 1080.0 ? 0.0 : e;
}

// order-preserving key of a float that came from T, without T's unused bits; -0 equals 0
template <typename T> struct KeyShift;
template <> struct KeyShift<float> { static constexpr int v = 0; };
template <> struct KeyShift<_Float16> { static constexpr int v = 13; };
template <> struct KeyShift<__bf16> { static constexpr int v = 16; };
template <typename T> __device__ __forceinline__ uint32_t key_of(float x) {
  uint32_t b = f32_bits(x);
  if (b == 0x80000000u) b = 0;
  return ((b & 0x80000000u) ? ~b : b | 0x80000000u) >> KeyShift<T>::v;
}
template <typename T> __device__ __forceinline__ float value_of(uint32_t key) {
  constexpr int S = KeyShift<T>::v;
  const uint32_t k = (uint32_t)((u64)key << S);
  if (k & 0x80000000u) return bits_f32(k ^ 0x80000000u);
  return bits_f32(~(k | (uint32_t)((1ull << S) - 1)));
}

// This lane's 32 logits of a run; column of v[i]: run * kRun + col_of(i). -inf past the row's end (no filter and no sum
// tells those from masked tokens).
template <typename T>
struct Run {
  static constexpr int VEC = 16 / sizeof(T);
  float v[kLaneCols];
  __device__ __forceinline__ void load(const T* row, int run, int cols) {
    const int lane = threadIdx.x % kWave;
    const int c0 = run * kRun + lane * VEC;
    if ((run + 1) * kRun <= cols) {  // (the same for the whole wave)
      Pack<T, VEC> p[kLaneCols / VEC];
#pragma unroll
      for (int j = 0; j < kLaneCols / VEC; ++j) p[j] = load_pack_any<T, VEC>(row + c0 + j * kWave * VEC);
#pragma unroll
      for (int j = 0; j < kLaneCols / VEC; ++j) {
        float f[VEC];
        unpack(p[j], f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j * VEC + i] = f[i];
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < kLaneCols / VEC; ++j) {
      const int c = c0 + j * kWave * VEC;
      float f[VEC];
      if (c + VEC <= cols) {
        unpack(load_pack_any<T, VEC>(row + c), f);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = c + i < cols ? to_f32<T>(row[c + i]) : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j * VEC + i] = f[i];
    }
  }
  __device__ __forceinline__ float lane_max() const {
    float m = v[0];
#pragma unroll
    for (int i = 1; i < kLaneCols; ++i) m = fmaxf(m, v[i]);
    return m;
  }
};

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
// sum over the threads before this one; `tmp` holds one value a wave
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

// A row's maximum and sum of e^(z - max) from its blocks' parts (split <= 64); false if it has no distribution. Every
// wave computes it for itself.
__device__ __forceinline__ bool row_state(const SampleArgs& g, int64_t row, const Asked& a, float* max, float* sum) {
  const int lane = threadIdx.x % kWave;
  const float m = lane < g.split ? g.part_max[row * g.split + lane] : -INFINITY;
  const float s = lane < g.split ? g.part_sum[row * g.split + lane] : 0.f;
  const float c = (float)(1.4426950408889634074 / a.temp);
  *max = wave_max(m);
  *sum = wave_sum(m == -INFINITY ? s : s * exp2_fast((m - *max) * c));
  // (a NaN, a +inf or nothing above -inf leaves the sum NaN or 0)
  return a.in_range && *sum > 0.f && *sum < INFINITY && *max < INFINITY;
}

// ---- scan -------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kLanes) void sample_scan_kernel(SampleArgs g) {
  __shared__ float sm[kWaves], sz[kWaves];
  const int64_t row = blockIdx.x / g.split;
  const int part = blockIdx.x % g.split;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const Asked a = asked(g, row);
  const T* x = static_cast<const T*>(g.logits) + row * g.ld;
  const double k = 1.4426950408889634074 / a.temp;
  const float c = (float)k;
  float m = -INFINITY, z = 0.f;
  for (int run = part * kWaves + wave; run < g.runs; run += g.split * kWaves) {
    Run<T> r;
    r.load(x, run, g.cols);
    float q = r.lane_max();
    q = fmaxf(q, dpp_move<dpp::kXor1>(q, q));
    q = fmaxf(q, dpp_move<dpp::kXor2>(q, q));
    q = fmaxf(q, dpp_move<dpp::kHalfMirror>(q, q));
    q = fmaxf(q, dpp_move<dpp::kMirror>(q, q));
    if (a.by_k && lane % 16 == 0) g.quarters[(row * g.runs + run) * 4 + lane / 16] = q;
    q = fmaxf(q, dpp_move<dpp::kBcast15, 0xa>(q, q));
    q = fmaxf(q, dpp_move<dpp::kBcast31, 0xc>(q, q));
    const float rm = lane63(q);
    if (a.open) {
      const double ref = rm == -INFINITY ? 0.0 : (double)rm;
      double mass = 0.0;
#pragma unroll
      for (int i = 0; i < kLaneCols; ++i) mass += exp2_product((double)r.v[i] - ref, k);
      mass = wave_total(mass);
      if (lane == 0) g.run_mass[row * g.runs + run] = mass, g.run_max[row * g.runs + run] = rm;
    } else {
      const float n = fmaxf(m, rm), ref = n == -INFINITY ? 0.f : n;
      z *= exp2_fast((m - ref) * c);
#pragma unroll
      for (int i = 0; i < kLaneCols; ++i) z += exp2_fast((r.v[i] - ref) * c);
      m = n;
    }
  }
  if (a.open) return;
  z = wave_sum(z);
  if (lane == 0) sm[wave] = m, sz[wave] = z;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kWaves; ++i) m = fmaxf(m, sm[i]);
    z = 0.f;
    for (int i = 0; i < kWaves; ++i) z += sm[i] == -INFINITY ? sz[i] : sz[i] * exp2_fast((sm[i] - m) * c);
    g.part_max[blockIdx.x] = m;
    g.part_sum[blockIdx.x] = z;
  }
}

// ---- hist and cut -----------------------------------------------------------
struct Fine {
  u64 mass[kBins];
  uint32_t count[kBins], key[kBins];
};
// What the bins of a block's columns need, and what finding a cut needs beside.
struct HistShared {
  Hist linear;
  float quarters[kMaxQuarters];
  float bound;
};
struct CutShared : HistShared {
  Fine fine;
  u64 ltmp[kWaves];
  uint32_t utmp[kWaves];
  // the bin that holds a cut
  int bin;
  uint32_t cnt_before;
  u64 mass_before;
};

// The bin whose running count passes `count_target` (by count), or whose running mass reaches `mass_target`; what lies
// before it goes to sh. Exactly one bin qualifies. Begins and ends with a barrier.
__device__ __forceinline__ void find_bin(const u64* mass, const uint32_t* count, CutShared& sh, bool by_count,
                                         uint32_t count_target, u64 mass_target) {
  constexpr int kEach = kBins / kLanes;
  __syncthreads();
  if (threadIdx.x == 0) sh.bin = kBins - 1, sh.cnt_before = 0, sh.mass_before = 0;
  const int b = kEach * threadIdx.x;
  uint32_t c[kEach], cs = 0;
  u64 m[kEach], ms = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) c[i] = count[b + i], m[i] = mass[b + i], cs += c[i], ms += m[i];
  uint32_t cb = block_before<uint32_t>(cs, sh.utmp);
  u64 mb = block_before<u64>(ms, sh.ltmp);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const bool here = by_count ? cb < count_target && count_target - cb <= c[i]
                               : mb < mass_target && mass_target - mb <= m[i];
    if (here) sh.bin = b + i, sh.cnt_before = cb, sh.mass_before = mb;
    cb += c[i];
    mb += m[i];
  }
  __syncthreads();
}

template <typename T>
struct Row {
  const T* x;
  int cols, runs;
  float max;        // of the row
  double to_log2;   // log2(e) / T
  float bin_step;   // kBins / (kRange T)
  double magic;

  __device__ __forceinline__ double mass(float v) const { return exp2_product((double)v - (double)max, to_log2); }
  __device__ __forceinline__ u64 fixed(double e) const {
    return __builtin_bit_cast(u64, e + magic) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ int bin_of(float v) const {
    const float d = (max - v) * bin_step;
    return d < (float)(kBins - 1) ? (int)d : kBins - 1;
  }

  // Adds the runs of one block (part of split) to sh.linear; logits below `least` are left out.
  __device__ __forceinline__ void fill_linear(HistShared& sh, int part, int split, float least, bool masses) const {
    for (int i = threadIdx.x; i < kBins; i += kLanes) sh.linear.mass[i] = 0, sh.linear.count[i] = 0;
    __syncthreads();
    uint32_t low = 0;
    u64 low_mass = 0;
    for (int run = part * kWaves + (int)threadIdx.x / kWave; run < runs; run += split * kWaves) {
      Run<T> r;
      r.load(x, run, cols);
#pragma unroll
      for (int i = 0; i < kLaneCols; ++i) {
        if (r.v[i] >= least) {
          const int b = bin_of(r.v[i]);
          const u64 e = masses ? fixed(mass(r.v[i])) : 0;
          if (b < kBins - 1) {
            atomicAdd(&sh.linear.count[b], 1u);
            if (masses) atomicAdd(&sh.linear.mass[b], e);
          } else {
            ++low;
            low_mass += e;
          }
        }
      }
    }
    low = wave_total(low);
    low_mass = wave_total(low_mass);
    if (threadIdx.x % kWave == 0) {
      atomicAdd(&sh.linear.count[kBins - 1], low);
      if (masses) atomicAdd(&sh.linear.mass[kBins - 1], low_mass);
    }
  }

  // The cut after `k` logits (by count) or at mass `tau` (fixed point), and the mass that it keeps.
  __device__ __forceinline__ Cut find_cut(CutShared& sh, bool by_count, uint32_t k, u64 tau, bool masses,
                                          u64* kept) const {
    find_bin(sh.linear.mass, sh.linear.count, sh, by_count, k, tau);
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
    float value = max;
    uint32_t equal = 0;
    // one value of T in the bin (16-bit logits away from 0): nothing to look at
    int values = 0;
    if (khi - klo < 16) {
      for (uint32_t key = klo; key <= khi; ++key) {
        const float v = value_of<T>(key);
        if (bin_of(v) == lin) ++values, value = v;
      }
    }
    if (values == 1) {
      equal = sh.linear.count[lin];
    } else {
      // 32 bits of key in turns of 11
      for (int turn = 0; turn < 3; ++turn) {
        int s = 0;
        while (((khi - klo) >> s) >= (uint32_t)kBins) ++s;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kLanes) sh.fine.mass[i] = 0, sh.fine.count[i] = 0, sh.fine.key[i] = 0;
        __syncthreads();
        for (int run = threadIdx.x / kWave; run < runs; run += kWaves) {
          Run<T> r;
          r.load(x, run, cols);
#pragma unroll
          for (int i = 0; i < kLaneCols; ++i) {
            if (bin_of(r.v[i]) == lin) {
              const uint32_t key = key_of<T>(r.v[i]);
              if (key >= klo && key <= khi) {
                const uint32_t b = (khi - key) >> s;
                atomicAdd(&sh.fine.count[b], 1u);
                atomicMax(&sh.fine.key[b], key);
                if (masses) atomicAdd(&sh.fine.mass[b], fixed(mass(r.v[i])));
              }
            }
          }
        }
        find_bin(sh.fine.mass, sh.fine.count, sh, by_count, k - cnt, tau - above);
        const uint32_t b = (uint32_t)sh.bin;
        cnt += sh.cnt_before;
        above += sh.mass_before;
        khi -= b << s;
        equal = sh.fine.count[b];
        value = value_of<T>(sh.fine.key[b]);
        if (s == 0 || equal == 1) break;
        klo = ::max(klo, khi - ((1u << s) - 1));
      }
    }
    Cut cut;
    cut.x = value;
    cut.equal = equal;
    const u64 each = masses ? fixed(mass(value)) : 0;
    // (by mass: the bin holds equal * each >= tau - above > 0)
    cut.ties = by_count ? k - cnt : (uint32_t)((tau - above + each - 1) / each);
    *kept = above + each * cut.ties;
    return cut;
  }

  // The row's cut by top-k and top-p, from sh.linear.
  __device__ __forceinline__ Cut find(CutShared& sh, const Asked& a) const {
    Cut cut = {-INFINITY, 0xffffffffu, 0};
    u64 total = 0;
    if (a.by_k) cut = find_cut(sh, true, (uint32_t)a.top_k, 0, a.by_p, &total);
    if (a.by_p) {
      if (!a.by_k) {
        __syncthreads();
        u64 t = 0;
        for (int i = threadIdx.x; i < kBins; i += kLanes) t += sh.linear.mass[i];
        t = wave_total(t);
        if (threadIdx.x % kWave == 0) sh.ltmp[threadIdx.x / kWave] = t;
        __syncthreads();
        for (int i = 0; i < kWaves; ++i) total += sh.ltmp[i];
      }
      const u64 tau = ::min(total, ::max((u64)1, (u64)ceil(fmax(a.top_p, 0.0) * (double)total)));
      u64 unused;
      const Cut p = find_cut(sh, false, 0, tau, true, &unused);
      if (!a.by_k || p.x > cut.x) cut = p;
      else if (p.x == cut.x && p.ties < cut.ties) cut.ties = p.ties;
    }
    return cut;
  }
};

template <typename T>
__device__ __forceinline__ Row<T> row_of(const SampleArgs& g, int64_t row, const Asked& a, float max) {
  Row<T> r;
  r.x = static_cast<const T*>(g.logits) + row * g.ld;
  r.cols = g.cols;
  r.runs = g.runs;
  r.max = max;
  r.to_log2 = 1.4426950408889634074 / a.temp;
  r.bin_step = (float)(kBins / (kRange * a.temp));
  r.magic = g.magic;
  return r;
}

// A lower bound of the k-th largest logit: the k-th largest of the maxima of 512 columns (each of those k is a logit of
// its own), where there are enough of them.
__device__ __forceinline__ float least_of_top_k(const SampleArgs& g, int64_t row, const Asked& a, HistShared& sh) {
  const int n = 4 * g.runs;
  if (!a.by_k || a.top_k > n || n > kMaxQuarters) return -INFINITY;
  for (int i = threadIdx.x; i < n; i += kLanes) sh.quarters[i] = g.quarters[row * n + i];
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kLanes) {
    const float v = sh.quarters[i];
    int before = 0;
    for (int j = 0; j < n; ++j) before += sh.quarters[j] > v || (sh.quarters[j] == v && j < i);
    if (before == (int)a.top_k - 1) sh.bound = v;
  }
  __syncthreads();
  return sh.bound;
}

// WHOLE: one block has the whole row (split 1) and goes on to the cut.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kLanes) void sample_hist_kernel(SampleArgs g) {
  __shared__ typename std::conditional<WHOLE, CutShared, HistShared>::type sh;
  const int64_t row = blockIdx.x / g.split;
  const Asked a = asked(g, row);
  if (!a.by_k && !a.by_p) return;
  float max, sum;
  if (!row_state(g, row, a, &max, &sum)) return;
  const Row<T> r = row_of<T>(g, row, a, max);
  r.fill_linear(sh, (int)(blockIdx.x % g.split), g.split, least_of_top_k(g, row, a, sh), a.by_p);
  if constexpr (WHOLE) {
    const Cut cut = r.find(sh, a);
    if (threadIdx.x == 0) g.cuts[row] = cut;
  } else {
    __syncthreads();
    Hist& to = g.hist[blockIdx.x];
    for (int i = threadIdx.x; i < kBins; i += kLanes) {
      to.count[i] = sh.linear.count[i];
      if (a.by_p) to.mass[i] = sh.linear.mass[i];
    }
  }
}

// (split > 1)
template <typename T>
__global__ __launch_bounds__(kLanes) void sample_cut_kernel(SampleArgs g) {
  __shared__ CutShared sh;
  const int64_t row = blockIdx.x;
  const Asked a = asked(g, row);
  if (!a.by_k && !a.by_p) return;
  float max, sum;
  if (!row_state(g, row, a, &max, &sum)) return;
  const Row<T> r = row_of<T>(g, row, a, max);
  const Hist* from = g.hist + row * g.split;
  for (int i = threadIdx.x; i < kBins; i += kLanes) {
    uint32_t c = 0;
    u64 m = 0;
    for (int p = 0; p < g.split; ++p) {
      c += from[p].count[i];
      if (a.by_p) m += from[p].mass[i];
    }
    sh.linear.count[i] = c;
    sh.linear.mass[i] = m;
  }
  const Cut cut = r.find(sh, a);
  if (threadIdx.x == 0) g.cuts[row] = cut;
}

// The row's cut with min-p in it.
__device__ __forceinline__ Cut final_cut(const SampleArgs& g, int64_t row, const Asked& a, float max) {
  Cut cut = {-INFINITY, 0xffffffffu, 0};
  if (a.by_k || a.by_p) cut = g.cuts[row];
  if (a.min_p > 0.0) {
    // e^((x - max) / T) >= min_p, as the smallest float that satisfies it
    const double least = (double)max + a.temp * log(fmin(a.min_p, 1.0));
    float f = (float)least;
    if ((double)f < least) f = nextafterf(f, INFINITY);
    if (f > cut.x) cut = {f, 0xffffffffu, 0};
  }
  return cut;
}

// ---- mass -------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kLanes) void sample_mass_kernel(SampleArgs g) {
  const int64_t row = blockIdx.x / g.split;
  const int part = blockIdx.x % g.split;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const Asked a = asked(g, row);
  if (a.open) return;
  float max, sum;
  if (!row_state(g, row, a, &max, &sum)) return;
  const Cut cut = final_cut(g, row, a, max);
  const Row<T> r = row_of<T>(g, row, a, max);
  const bool all_ties = cut.ties >= cut.equal;
  for (int run = part * kWaves + wave; run < g.runs; run += g.split * kWaves) {
    Run<T> l;
    l.load(r.x, run, g.cols);
    double mass = 0.0;
    uint32_t ties = 0;
#pragma unroll
    for (int i = 0; i < kLaneCols; ++i) {
      const float v = l.v[i];
      if (v >= cut.x) {
        if (all_ties || v > cut.x) mass += r.mass(v);
        else ++ties;
      }
    }
    mass = wave_total(mass);
    ties = wave_total(ties);
    if (lane == 0) g.run_mass[row * g.runs + run] = mass, g.run_ties[row * g.runs + run] = ties;
  }
}

// ---- pick -------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kPickLanes) void sample_pick_kernel(SampleArgs g) {
  constexpr int kPickWaves = kPickLanes / kWave;
  constexpr int kCols = kRun / kPickLanes;  // columns a thread, in order
  __shared__ double dtmp[kPickWaves];
  __shared__ uint32_t utmp[kPickWaves];
  __shared__ float ftmp[kPickWaves];
  __shared__ int found, last, sh_run;
  __shared__ double sh_base;
  __shared__ uint32_t sh_ties;
  const int64_t row = blockIdx.x;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const Asked a = asked(g, row);
  const double* run_mass = g.run_mass + row * g.runs;
  const uint32_t* run_ties = g.run_ties + row * g.runs;
  const float* run_max = g.run_max + row * g.runs;
  const int per = (g.runs + kPickLanes - 1) / kPickLanes;  // runs a thread, in order
  const int r0 = min(g.runs, (int)threadIdx.x * per), r1 = min(g.runs, r0 + per);

  float max, sum = 0.f;
  bool fine = a.in_range;
  if (a.open) {
    float m = -INFINITY;
    for (int i = r0; i < r1; ++i) m = fmaxf(m, run_max[i]);
    m = wave_max(m);
    if (lane == 0) ftmp[wave] = m;
    __syncthreads();
    max = ftmp[0];
    for (int i = 1; i < kPickWaves; ++i) max = fmaxf(max, ftmp[i]);
  } else {
    fine = row_state(g, row, a, &max, &sum);
  }
  if (!fine) {
    if (threadIdx.x == 0) g.ids[row] = -1, g.logp[row] = __builtin_nanf("");
    return;
  }
  const Row<T> r = row_of<T>(g, row, a, max);
  const Cut cut = a.open ? Cut{-INFINITY, 0xffffffffu, 0} : final_cut(g, row, a, max);
  const bool all_ties = cut.ties >= cut.equal;
  const double each = all_ties ? 0.0 : r.mass(cut.x);

  // the masses of the runs: an open row's are relative to the run's own maximum
  uint32_t ties = 0, seen = 0;
  if (!all_ties) {
    for (int i = r0; i < r1; ++i) ties += run_ties[i];
    seen = block_before<uint32_t>(ties, utmp);
  }
  auto mass_of = [&](int i, uint32_t& ties_before) {
    if (a.open) {
      const float m = run_max[i];
      return m == -INFINITY ? run_mass[i] : run_mass[i] * r.mass(m);
    }
    if (all_ties) return run_mass[i];
    const uint32_t t = run_ties[i], left = cut.ties - min(cut.ties, ties_before);
    ties_before += t;
    return run_mass[i] + each * (double)min(left, t);
  };
  double mass = 0.0;
  uint32_t rank = seen;
  for (int i = r0; i < r1; ++i) mass += mass_of(i, rank);
  const double before = block_before<double>(mass, dtmp);
  if (threadIdx.x == 0) found = kPickLanes, last = -1;
  __syncthreads();
  double total = 0.0;
  for (int i = 0; i < kPickWaves; ++i) total += dtmp[i];
  if (!(total > 0.0 && total < INFINITY && max < INFINITY)) {  // (only an open row's can be)
    if (threadIdx.x == 0) g.ids[row] = -1, g.logp[row] = __builtin_nanf("");
    return;
  }
  const double target = (double)g.u[row] * total;
  // the first thread that passes the target; if none does, the last one with any mass
  if (mass > 0.0) {
    if (before + mass > target) atomicMin(&found, (int)threadIdx.x);
    atomicMax(&last, (int)threadIdx.x);
  }
  __syncthreads();
  if ((int)threadIdx.x == (found < kPickLanes ? found : last)) {
    double s = before;
    int run = r0;
    rank = seen;
    for (int i = r0; i < r1; ++i) {
      const uint32_t rank_before = rank;
      const double m = mass_of(i, rank);
      if (m > 0.0) run = i, sh_base = s, sh_ties = rank_before;
      s += m;
      if (m > 0.0 && s > target) break;
    }
    sh_run = run;
  }
  __syncthreads();
  const int c0 = sh_run * kRun + (int)threadIdx.x * kCols;
  float v[kCols];
#pragma unroll
  for (int i = 0; i < kCols; ++i) v[i] = c0 + i < g.cols ? to_f32<T>(r.x[c0 + i]) : -INFINITY;
  rank = sh_ties;
  const double base = sh_base;
  if (!all_ties) {
    ties = 0;
#pragma unroll
    for (int i = 0; i < kCols; ++i) ties += v[i] == cut.x ? 1 : 0;
    rank += block_before<uint32_t>(ties, utmp);
  }
  double e[kCols];
  mass = 0.0;
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    bool keep = v[i] >= cut.x;
    if (!all_ties && v[i] == cut.x) keep = rank++ < cut.ties;
    e[i] = keep ? r.mass(v[i]) : 0.0;
    mass += e[i];
  }
  double s = base + block_before<double>(mass, dtmp);
  if (threadIdx.x == 0) found = kPickLanes, last = -1;
  __syncthreads();
  if (mass > 0.0) {
    if (s + mass > target) atomicMin(&found, (int)threadIdx.x);
    atomicMax(&last, (int)threadIdx.x);
  }
  __syncthreads();
  if ((int)threadIdx.x != (found < kPickLanes ? found : last)) return;
  int id = -1;
  float at = 0.f;
  bool done = false;
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    if (!done && e[i] > 0.0) id = c0 + i, at = v[i];
    s += e[i];
    done = done || (e[i] > 0.0 && s > target);
  }
  g.ids[row] = id;
  g.logp[row] = (float)(((double)at - (double)max) / a.temp) - log_fast(a.open ? (float)total : sum);
}

// Blocks a row: enough for three blocks a CU, each with a run a wave at least.
int split_of(int64_t rows, int64_t runs, int64_t cus) {
  const int64_t want = cdiv(3 * cus, std::max<int64_t>(rows, 1));
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, (int64_t)kMaxSplit, cdiv(runs, (int64_t)kWaves)}));
}

struct Layout {
  size_t part_max, part_sum, quarters, run_mass, run_ties, run_max, hist, cuts, total;
};
Layout layout_of(int64_t rows, int64_t runs, int64_t split, bool cuts) {
  Layout l = {};
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t here = at;
    at += (n + 255) / 256 * 256;
    return here;
  };
  l.run_mass = take((size_t)(rows * runs) * sizeof(double));
  l.run_ties = take((size_t)(rows * runs) * sizeof(uint32_t));
  l.run_max = take((size_t)(rows * runs) * sizeof(float));
  l.part_max = take((size_t)(rows * split) * sizeof(float));
  l.part_sum = take((size_t)(rows * split) * sizeof(float));
  if (cuts) {
    l.quarters = take((size_t)(rows * runs) * 4 * sizeof(float));
    l.cuts = take((size_t)rows * sizeof(Cut));
    if (split > 1) l.hist = take((size_t)(rows * split) * sizeof(Hist));
  }
  l.total = at;
  return l;
}

}  // namespace
}  // namespace hk

using namespace hk;

extern "C" {

size_t hk_sample_workspace_size(int64_t rows, int64_t cols, int cuts, int device) {
  if (rows < 0 || rows >= (1LL << 31) || cols <= 0 || cols > (1 << 30)) return 0;
  const int cus = cu_count(device);
  const int64_t runs = cdiv(cols, (int64_t)kRun);
  return std::max<size_t>(256, layout_of(rows, runs, split_of(rows, runs, cus > 0 ? cus : 256), cuts != 0).total);
}

int hk_sample(int64_t* ids, float* logp, const void* logits, const float* u, int64_t rows, int64_t cols, int64_t ld,
              const float* temperature_rows, double temperature, const void* top_k_rows, int top_k_type, int64_t top_k,
              const float* top_p_rows, double top_p, const float* min_p_rows, double min_p, int dtype,
              void* workspace, size_t workspace_bytes, hk_stream_t stream) {
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
  HK_REQUIRE(workspace != nullptr && aligned_to(workspace, 16), "the workspace must be 16-byte aligned");
  const int dev = current_device();
  if (dev < 0) return (int)hipErrorNoDevice;
  const int cus = cu_count(dev);
  const int64_t runs = cdiv(cols, (int64_t)kRun);
  const int split = split_of(rows, runs, cus > 0 ? cus : 256);
  HK_REQUIRE(rows * split < (1LL << 31), "rows=%lld too large", (long long)rows);
  const bool cuts = top_k_rows || (top_k > 0 && top_k < cols) || top_p_rows || top_p < 1;
  const bool masses = cuts || min_p_rows || min_p > 0;
  const Layout l = layout_of(rows, runs, split, cuts);
  HK_REQUIRE(workspace_bytes >= l.total, "workspace too small: need %zu bytes, got %zu", l.total, workspace_bytes);
  char* ws = (char*)workspace;
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
  g.runs = (int)runs;
  g.split = split;
  int log2_cols = 0;
  while ((1LL << log2_cols) < cols + kRun) ++log2_cols;
  g.magic = (double)(1ULL << (52 - std::min(43, 63 - log2_cols)));
  g.part_max = (float*)(ws + l.part_max);
  g.part_sum = (float*)(ws + l.part_sum);
  g.quarters = (float*)(ws + l.quarters);
  g.run_mass = (double*)(ws + l.run_mass);
  g.run_ties = (uint32_t*)(ws + l.run_ties);
  g.run_max = (float*)(ws + l.run_max);
  g.hist = (Hist*)(ws + l.hist);
  g.cuts = (Cut*)(ws + l.cuts);
  auto launch = [&](auto tag) {
    using T = decltype(tag);
    const hipStream_t st = (hipStream_t)stream;
    const dim3 parts((unsigned)(rows * split)), each((unsigned)rows);
    hipLaunchKernelGGL((sample_scan_kernel<T>), parts, dim3(kLanes), 0, st, g);
    if (const int rc = check_launch("sample_scan_kernel")) return rc;
    if (cuts) {
      if (split == 1) hipLaunchKernelGGL((sample_hist_kernel<T, true>), parts, dim3(kLanes), 0, st, g);
      else hipLaunchKernelGGL((sample_hist_kernel<T, false>), parts, dim3(kLanes), 0, st, g);
      if (const int rc = check_launch("sample_hist_kernel")) return rc;
      if (split > 1) {
        hipLaunchKernelGGL((sample_cut_kernel<T>), each, dim3(kLanes), 0, st, g);
        if (const int rc = check_launch("sample_cut_kernel")) return rc;
      }
    }
    if (masses) {
      hipLaunchKernelGGL((sample_mass_kernel<T>), parts, dim3(kLanes), 0, st, g);
      if (const int rc = check_launch("sample_mass_kernel")) return rc;
    }
    hipLaunchKernelGGL((sample_pick_kernel<T>), each, dim3(kPickLanes), 0, st, g);
    return check_launch("sample_pick_kernel");
  };
  if (dtype == kF32) return launch(float{});
  if (dtype == kF16) return launch(_Float16{});
  return launch(__bf16{});
}

}  // extern "C"
