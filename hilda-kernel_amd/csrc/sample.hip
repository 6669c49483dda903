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
// into runs of 512 to 2048 columns, its runs are dealt to the waves of a few
// blocks, and a few launches follow each other (the first reads the row from
// HBM, the later ones from the Infinity Cache):
//   no filter       open, pick
//   min-p alone     scan, mass, pick
//   a small top-k   scan, list, draw
//   top-k or top-p  bf16: count, cut, mass, pick
//                   fp16, fp32: scan, hist, cut, mass, pick
// (a setting that comes row by row may be any of its values; fp16's and
// fp32's rows of a small top-k of their own go by a list between the others)
//   open   the fp64 mass and the maximum of each run
//   scan   max and log-sum-exp (fp32)
//   list   the few logits at or above a bound on the k-th, taken from the scan's
//          maxima, and (draw) the token from them, ordered. One reading of the
//          row and two launches less than bins: 256 rows of 151936 fp32 logits
//          with k = 50 take 65 us, with k = 209 by bins 99; one bf16 row of 128256
//          20 and 31.
//   hist   counts, and for top-p masses, in bins linear in max - x
//   count  counts in bins of one bf16 value each, which give the maximum, the
//          sum and every mass
//   cut    the bins of a row's blocks together; the bin that holds the cut; if
//          several values may lie in it, the same over ranges of ordered keys,
//          11 bits at a time, until one is left: x* and how many ties are kept.
//          With one block a row this ends the launch before. If the bin has 768
//          logits or less and there is one filter, mass lists them and pick finds
//          the cut in their order instead: a block takes 25 to 45 us to read a
//          row of 151936 fp32 logits, mass reads them anyway, and pick takes 10 us
//          more (256 such rows with top-p: 174 us, 193 before).
//          Of bf16 rows in few long parts it also tells the part that the
//          token lies in, by the parts' counts.
//   mass   the kept mass of each run (of that part)
//   pick   the run that u * total falls into, and the token inside it
//
// What bounds it: the first pass of 256 rows of 151936 bf16 logits (78 MB) runs
// at HBM's rate (scan 15 us); the bins' LDS atomics (count 23 us) and the mass
// table's LDS gathers (mass 21 us, 33 cycles a wave's) are LDS-bound, cut, draw
// and pick (17, 7 and 8 us) chains of latencies. 69 us in all with top-p, 33
// without filters; few rows are bound by those chains, 4 to 14 us a launch. fp32
// and fp16 pay for e^(z - max) in fp64 in hist and mass (50 and 57 us with top-p).
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

constexpr int kLanes = 1024;          // threads of a block
constexpr int kWaves = kLanes / kWave;
constexpr int kMaxSplit = 16;         // blocks a row at most
constexpr int kFineBins = 2048;
// the linear bins cover max - x < kRange * T; beyond it is one bin
constexpr double kRange = 24;
constexpr double kTempMin = 0x1p-64, kTempMax = 0x1p64;
constexpr double kLog2eD = 1.4426950408889634074, kLn2D = 0.69314718055994530942;
constexpr int kGroups = 256;          // maxima that a bound on the k-th logit is taken from
// Columns of a part at least for a choice of the part (choose_part takes 4 to 6 us; bf16, top-p 0.95 and top-k 5000, with
// and without: 128 rows in parts of 76000 52 and 55, 46 and 45 us; 100 of 50000 45 and 45, 42 and 39; 64 of 38000 43 and
// 43, 42 and 38).
constexpr int64_t kChooseCols = 64 << 10;
// Rows of few kept logits go by a list of those at or above that bound: for k = 208 of 256 groups it has about
// 256 ln(256 / 48) = 430 of them, for k = 50 some 56. (64 x 151936 bf16: k = 20 23 us, 208 38; by bins k = 209 39.
// 256 x 151936 fp32: 66, 81; 97.)
constexpr int kListMost = 208;        // k of such a row at most
// (430 has a deviation of 26; a list short of room costs three more readings of the row.)
constexpr int kPartList = 768, kList = 768;  // room for a block's, and a row's
// columns at least: the lists then have three quarters of the logits' bytes at most. 512 rows of 8192 with k = 50 take 26
// us, by bins 44.
constexpr int kListCols = 8192;
__host__ __device__ constexpr int list_most(int runs) { return 4 * runs < kListMost ? 4 * runs : kListMost; }

// A setting of every row, or one each.
struct Setting {
  const float* rows;
  double all;
};

// Bins of logits, in descending order. fp32 and fp16: linear in max - x, with counts and masses. bf16: one bin for each
// value of 2^-16 <= |x| < 2^8 (kSide of either sign), so a count is a mass, and three more that hold several: x >= 2^8,
// |x| < 2^-16 and x <= -2^8.
template <typename T> struct Bins {
  static constexpr int kCount = 2048, kMasses = kCount;
  static constexpr bool kExact = false;
};
template <> struct Bins<__bf16> {
  static constexpr int kSide = 24 * 128, kLowest = (127 - 16) << 7;  // kLowest: the bits of 2^-16
  static constexpr int kZero = kSide + 1, kUsed = 2 * kSide + 3;
  static constexpr int kCount = 7168, kMasses = 4;  // (whole turns of the block; masses of the three)
  static constexpr bool kExact = true;
  static __device__ __forceinline__ int of(float v) {
    const int b = (int)f32_bits(v), sign = b >> 31;
    const int i = ::min(::max(((b >> 16) & 0x7fff) - kLowest + 1, 0), kSide + 1);
    return kZero - (i ^ sign) + sign;
  }
  // of both bf16 values of a word, by packed 16-bit integers; `rank`: 0 for |x| < 2^-16, kSide + 1 for |x| >= 2^8
  typedef short Two __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ Two of_two(uint32_t w, Two* rank) {
    const Two sign = __builtin_bit_cast(Two, w) >> (short)15;
    const Two i = __builtin_elementwise_min(
        __builtin_elementwise_max((Two)(__builtin_bit_cast(Two, w & 0x7fff7fffu) - (short)(kLowest - 1)), (Two)((short)0)),
        (Two)((short)(kSide + 1)));
    *rank = i;
    return (short)kZero - (i ^ sign) + sign;
  }
  static __device__ __forceinline__ bool several(int bin) { return bin == 0 || bin == kZero || bin == kUsed - 1; }
  static __device__ __forceinline__ int slot(int bin) { return bin == 0 ? 0 : bin == kZero ? 1 : 2; }
  static __device__ __forceinline__ float value(int bin) {
    const int i = bin < kZero ? kZero - bin : bin - kZero;
    return bits_f32((uint32_t)(kLowest + i - 1) << 16 | (bin < kZero ? 0u : 0x80000000u));
  }
};
template <typename T> struct Hist {
  u64 mass[Bins<T>::kMasses];
  uint32_t count[Bins<T>::kCount];
};
// A cut: logits above x are kept, and the first `ties` of those equal to x
// (of `equal` in the row; all of them if ties >= equal). A cut inside the bin
// inside - 1 (0: none) is left to the pick: the logits of the bins before it
// are kept, and of its own, which are x or more, the first `target` in order,
// or as many as have that mass.
struct Cut {
  float x;
  uint32_t ties, equal;
  uint32_t count;  // logits kept
  u64 target;
  int inside;
};
struct Listed {
  float x;
  int col;
};
// The part of a row (of `split`, whose runs lie side by side) that u * total
// falls into, the kept mass and ties before it and the kept mass of the row;
// -1: not known.
struct Chosen {
  double before, total;
  uint32_t ties;
  int part;
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
  int cols, run_cols, runs;  // columns of a run (512, 1024 or 2048), runs of a row
  int split;       // blocks of a row
  int open;        // no row has a filter
  int has_cuts;    // cuts is written
  int lists;       // rows of few kept logits go by a list
  double magic;    // 2^(52 - b): e + magic holds e in b fixed-point bits
  // workspace
  float *part_max, *part_sum;  // [rows][split]
  float* quarters;             // [rows][4 runs] maxima of a quarter of a run's columns (those of 16 lanes)
  double* run_mass;            // [rows][runs]
  uint32_t* run_ties;
  float *run_max, *run_ref;    // of an open call: the run's maximum, and the logit whose mass its masses take as 1
  void* hist;                  // Hist<T> [rows][split], split > 1
  Cut* cuts;                   // [rows]
  Chosen* chosen;              // [rows], or null: no row has one
  Listed* list;                // [rows][split][kPartList]
  uint32_t* listed;            // [rows][split] how many (more than kPartList: not all are there)
};

__device__ __forceinline__ double setting(const Setting& s, int64_t row) { return s.rows ? s.rows[row] : s.all; }

// What a row asks for.
struct Asked {
  double temp, top_p, min_p;
  double k;  // log2(e) / T
  int64_t top_k;
  bool by_k, by_p, by_list;
  bool in_range;
};
__device__ __forceinline__ Asked asked(const SampleArgs& g, int64_t row) {
  Asked a;
  const float u = g.u[row];
  a.temp = setting(g.temperature, row);
  a.top_p = setting(g.top_p, row);
  a.min_p = setting(g.min_p, row);
  a.top_k = g.top_k;
  if (g.top_k_rows)
    a.top_k = g.top_k_wide ? static_cast<const int64_t*>(g.top_k_rows)[row]
                           : static_cast<const int32_t*>(g.top_k_rows)[row];
  a.k = kLog2eD / a.temp;
  a.by_k = a.top_k > 0 && a.top_k < g.cols;
  a.by_p = a.top_p < 1.0;
  a.by_list = g.lists && a.by_k && a.top_k <= list_most(g.runs);
  a.in_range = a.temp >= kTempMin && a.temp <= kTempMax && u >= 0.f && u <= 1.f && a.top_p == a.top_p &&
               a.min_p == a.min_p;
  return a;
}

// 2^y: y = n + r, |r| <= 1/2 (n from the low bits of y + 1.5 * 2^52), and for 2^r the polynomial of degree 10 that
// interpolates it at the Chebyshev nodes of [-1/2, 1/2] (relative error 3.2e-16). y = d * k with one rounding.
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

// VEC logits from column c; -inf past the row's end (no filter and no sum tells those from masked tokens)
template <typename T>
__device__ __forceinline__ Pack<T, 16 / sizeof(T)> load_cols(const T* row, int c, int cols) {
  constexpr int VEC = 16 / sizeof(T);
  if (c + VEC <= cols) return load_pack_any<T, VEC>(row + c);
  float f[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = -INFINITY;
  if (c < cols) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (c + i < cols) f[i] = to_f32<T>(row[c + i]);
  }
  return pack<T, VEC>(f);
}

// A row's runs first, first + waves, ...: look(pack, column) for each 16 bytes of a lane, done(run) after each run. A
// wave has two packs on their way. The loop stays rolled: unrolled over a run (32 logits a lane) these kernels have 25 to 80 KB
// of code, and fetching it, not the logits, set their time (hist of 64 x 151936: 33 us; 24 rolled).
template <typename T, typename L, typename D>
__device__ __forceinline__ void each_run(const T* row, int cols, int run_cols, int runs, int first, int waves, L&& look,
                                         D&& done) {
  constexpr int VEC = 16 / sizeof(T), kStep = kWave * VEC;
  first = __builtin_amdgcn_readfirstlane(first);  // (the wave's: the loop runs on the scalar unit)
  if (first >= runs) return;
  const int lane_col = (int)(threadIdx.x % kWave) * VEC;
  int run = first, at = 0, ahead = first, ahead_at = 0;
  auto load = [&] {
    const int c = ahead * run_cols + ahead_at;
    Pack<T, VEC> p;
    if (ahead < runs && c + kStep <= cols) p = load_pack_any<T, VEC>(row + c + lane_col);
    else p = load_cols(row, c + lane_col, ahead < runs ? cols : 0);
    ahead_at += kStep;
    if (ahead_at == run_cols) ahead_at = 0, ahead += waves;
    return p;
  };
  Pack<T, VEC> p0 = load(), p1 = load();
#pragma unroll 1
  while (run < runs) {
    const Pack<T, VEC> p = p0;
    p0 = p1;
    p1 = load();
    look(p, run * run_cols + at + lane_col);
    at += kStep;
    if (at == run_cols) {
      done(run);
      at = 0;
      run += waves;
    }
  }
}

// A value moved between lanes by the DPP pattern CTRL, word by word; lanes without a source, and rows outside ROW_MASK,
// get 0.
template <int CTRL, int ROW_MASK = 0xf, typename X>
__device__ __forceinline__ X moved(X v) {
  if constexpr (sizeof(X) == 4) {
    return __builtin_bit_cast(X, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROW_MASK, 0xf, false));
  } else {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(X, u32x2{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.x, CTRL, ROW_MASK, 0xf, false),
                                       (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.y, CTRL, ROW_MASK, 0xf, false)});
  }
}
template <typename X> __device__ __forceinline__ X of_lane63(X v) {
  if constexpr (sizeof(X) == 4) {
    return __builtin_bit_cast(X, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
  } else {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(X, u32x2{(uint32_t)__builtin_amdgcn_readlane((int)w.x, 63),
                                       (uint32_t)__builtin_amdgcn_readlane((int)w.y, 63)});
  }
}
// inclusive, over the wave: within rows of 16 lanes (row_shr 1, 2, 4, 8), then across them
template <typename X> __device__ __forceinline__ X wave_scan(X v) {
  v += moved<0x111>(v);
  v += moved<0x112>(v);
  v += moved<0x114>(v);
  v += moved<0x118>(v);
  v += moved<dpp::kBcast15, 0xa>(v);
  v += moved<dpp::kBcast31, 0xc>(v);
  return v;
}
template <typename X> __device__ __forceinline__ X wave_total(X v) {
  v += moved<dpp::kXor1>(v);
  v += moved<dpp::kXor2>(v);
  v += moved<dpp::kHalfMirror>(v);
  v += moved<dpp::kMirror>(v);
  v += moved<dpp::kBcast15, 0xa>(v);
  v += moved<dpp::kBcast31, 0xc>(v);
  return of_lane63(v);
}
template <typename X> __device__ __forceinline__ X of_lane(X v, int lane) {
  if constexpr (sizeof(X) == 4) {
    return __builtin_bit_cast(X, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  } else {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(X, u32x2{(uint32_t)__builtin_amdgcn_readlane((int)w.x, lane),
                                       (uint32_t)__builtin_amdgcn_readlane((int)w.y, lane)});
  }
}
// the sum over the threads before this one, and over all; `tmp` holds one value a wave
template <typename X> __device__ __forceinline__ X block_before(X v, X* tmp, X* total) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const X incl = wave_scan(v);
  __syncthreads();
  if (lane == kWave - 1) tmp[wave] = incl;
  __syncthreads();
  const X waves = wave_scan(lane < kWaves ? tmp[lane] : X(0));
  *total = of_lane63(waves);
  X before = incl - v;
  if (wave > 0) before += of_lane(waves, wave - 1);
  return before;
}

// The first thread of the block for which `passes`, or if there is none the last for which `some`; -1 without either.
// `tmp` holds two values a wave.
__device__ __forceinline__ int first_or_last(bool passes, bool some, int* tmp) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const u64 p = __ballot(passes), q = __ballot(some);
  __syncthreads();
  if (lane == 0) {
    tmp[wave] = p ? wave * kWave + __builtin_ctzll(p) : kLanes;
    tmp[kWaves + wave] = q ? wave * kWave + 63 - __builtin_clzll(q) : -1;
  }
  __syncthreads();
  int first = kLanes, last = -1;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) first = min(first, tmp[i]), last = max(last, tmp[kWaves + i]);
  return first < kLanes ? first : last;
}

// The smallest float x with e^((x - max) / T) >= min_p (-inf without min-p). log2 min_p: the instruction's, off by some
// 2^-22, and what is left of min_p after it (2^-100 of the largest probability is as good as none).
__device__ __forceinline__ float least_of_min_p(const Asked& a, float max) {
  if (!(a.min_p > 0.0)) return -INFINITY;
  if (a.min_p >= 1.0) return max;
  const double p = fmax(a.min_p, 0x1p-100);
  const double y = (double)log2_fast((float)p), rest = p * exp2_product(-y, 1.0) - 1.0;
  const double least = (double)max + a.temp * kLn2D * (y + kLog2eD * (rest - 0.5 * rest * rest));
  const float f = (float)least;
  return (double)f < least ? nextafterf(f, INFINITY) : f;
}

__device__ __forceinline__ void apply_min_p(Cut& cut, const Asked& a, float max) {
  const float f = least_of_min_p(a, max);
  if (f > cut.x) cut.x = f, cut.ties = 0xffffffffu, cut.equal = 0;
}
// The runs [begin, end) of a part of a row.
struct Runs {
  int begin, end;
};
__device__ __forceinline__ Runs runs_of(const SampleArgs& g, int part) {
  return {(int)((int64_t)g.runs * part / g.split), (int)((int64_t)g.runs * (part + 1) / g.split)};
}

// What the launches after the scan begin with, its loads in flight together: the row's settings, its maximum and sum of
// e^(z - max) from its blocks' parts (every wave puts them together for itself), and its cut. ok: it has a distribution.
struct Start {
  Asked a;
  float max, sum;
  bool ok;
  Cut cut;
  __device__ __forceinline__ Start(const SampleArgs& g, int64_t row, bool with_cut) {
    const int lane = threadIdx.x % kWave;
    const float m = lane < g.split ? g.part_max[row * g.split + lane] : -INFINITY;
    const float s = lane < g.split ? g.part_sum[row * g.split + lane] : 0.f;
    cut = {-INFINITY, 0xffffffffu, 0, 0xffffffffu};
    if (with_cut && g.has_cuts) cut = g.cuts[row];
    a = asked(g, row);
    if (!a.by_k && !a.by_p) cut = {-INFINITY, 0xffffffffu, 0, 0xffffffffu};
    max = wave_max(m);
    sum = wave_sum(m == -INFINITY ? s : s * exp2_fast((m - max) * (float)a.k));
    // (a NaN, a +inf or nothing above -inf leaves the sum NaN or 0)
    ok = a.in_range && sum > 0.f && sum < INFINITY && max < INFINITY;
    if (with_cut && ok) cut_min_p();
  }
  __device__ __forceinline__ void cut_min_p() {
    apply_min_p(cut, a, max);
  }
};

// The pack's logits one place down.
__device__ __forceinline__ void shift_down(Pack<__bf16, 8>& p) {
#pragma unroll
  for (int j = 0; j < 3; ++j) p.w[j] = __builtin_amdgcn_alignbit(p.w[j + 1], p.w[j], 16);
  p.w[3] >>= 16;
}
// f(logit) for those of a pack that are in a bin of several values and above -inf. Few are, so the loop stays rolled.
template <typename F>
__device__ __forceinline__ void each_several(Pack<__bf16, 8> p, F&& f) {
  typedef Bins<__bf16> B;
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const float v = bits_f32(p.w[0] << 16);
    if (B::several(B::of(v)) && v != -INFINITY) f(v);
    shift_down(p);
  }
}

// bf16: the masses of the bins that hold one value, and NaN for the bins of several up to `reach` (0 after it).
template <typename F>
__device__ __forceinline__ void fill_table(double* table, int reach, F&& mass) {
  typedef Bins<__bf16> B;
#pragma unroll 1
  for (int b = threadIdx.x; b < B::kUsed; b += kLanes)
    table[b] = b > reach ? 0.0 : B::several(b) ? (double)__builtin_nanf("") : mass(B::value(b));
  __syncthreads();
}
// The sum of the masses of a pack's logits: from the table, and by `mass` where that has NaN; 0 if no logit of the wave
// comes up to the bin `reach`.
template <typename F>
__device__ __forceinline__ double sum_table(const double* table, const Pack<__bf16, 8>& p, int reach, F&& mass) {
  typedef Bins<__bf16> B;
  B::Two bins[4], least = (B::Two)((short)B::kUsed), rank;
#pragma unroll
  for (int j = 0; j < 4; ++j) bins[j] = B::of_two(p.w[j], &rank), least = __builtin_elementwise_min(least, bins[j]);
  if (!__any(min(least.x, least.y) <= reach)) return 0.0;
  double s0 = 0.0, s1 = 0.0;
#pragma unroll
  for (int j = 0; j < 4; ++j) s0 += table[bins[j].x], s1 += table[bins[j].y];
  s0 += s1;
  if (s0 != s0) {  // few: the loop stays rolled, the pack moves down by one logit a turn
    Pack<__bf16, 8> q = p;
    s0 = 0.0;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const float v = bits_f32(q.w[0] << 16);
      const double e = table[B::of(v)];
      if (e == e) s0 += e;
      else if (v != -INFINITY) s0 += mass(v);
      shift_down(q);
    }
  }
  return s0;
}

// ---- scan -------------------------------------------------------------------
// The maximum and the sum of e^(z - max) of a block's runs, in its first wave; quarters: where the maxima of each run's
// quarters go, or null.
struct ScanShared {
  float m[kWaves], z[kWaves];
};
template <typename T>
__device__ __forceinline__ void scan_block(const T* x, const SampleArgs& g, int part, int split, float c, float* quarters,
                                           ScanShared& sh, float* max, float* sum) {
  constexpr int VEC = 16 / sizeof(T);
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  float m = -INFINITY, z = 0.f, rm = -INFINITY;  // rm: of the run
  each_run(
      x, g.cols, g.run_cols, g.runs, part * kWaves + wave, split * kWaves,
      [&](const Pack<T, VEC>& p, int) {
        float v[VEC];
        unpack(p, v);
        float q = v[0];
#pragma unroll
        for (int i = 1; i < VEC; ++i) q = fmaxf(q, v[i]);
        rm = fmaxf(rm, q);
        const float n = fmaxf(m, q), ref = n == -INFINITY ? 0.f : n;
        z *= exp2_fast((m - ref) * c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) z += exp2_fast((v[i] - ref) * c);
        m = n;
      },
      [&](int run) {
        if (!quarters) return;
        float q = rm;
        q = fmaxf(q, dpp_move<dpp::kXor1>(q, q));
        q = fmaxf(q, dpp_move<dpp::kXor2>(q, q));
        q = fmaxf(q, dpp_move<dpp::kHalfMirror>(q, q));
        q = fmaxf(q, dpp_move<dpp::kMirror>(q, q));
        if (lane % 16 == 0) quarters[run * 4 + lane / 16] = q;
        rm = -INFINITY;
      });
  {
    const float wm = wave_max(m), ref = wm == -INFINITY ? 0.f : wm;
    z = wave_sum(m == -INFINITY ? z : z * exp2_fast((m - ref) * c));
    m = wm;
  }
  if (lane == 0) sh.m[wave] = m, sh.z[wave] = z;
  __syncthreads();
  m = lane < kWaves ? sh.m[lane] : -INFINITY;
  z = lane < kWaves ? sh.z[lane] : 0.f;
  *max = wave_max(m);
  *sum = wave_sum(m == -INFINITY ? z : z * exp2_fast((m - *max) * c));
}

template <typename T>
__global__ __launch_bounds__(kLanes) void sample_scan_kernel(SampleArgs g) {
  __shared__ ScanShared sh;
  const int64_t row = blockIdx.x / g.split;
  const Asked a = asked(g, row);
  float max, sum;
  scan_block(static_cast<const T*>(g.logits) + row * g.ld, g, (int)(blockIdx.x % g.split), g.split, (float)a.k,
             a.by_list ? g.quarters + row * g.runs * 4 : nullptr, sh, &max, &sum);
  if (threadIdx.x == 0) g.part_max[blockIdx.x] = max, g.part_sum[blockIdx.x] = sum;
}

// A call without filters: the mass of each run, and its maximum.
template <typename T>
__global__ __launch_bounds__(kLanes) void sample_open_kernel(SampleArgs g) {
  constexpr int VEC = 16 / sizeof(T);
  // masses of bf16 logits below 2^8 in size: 2^(x k) itself from the table, within 2^+-739. Worth its making for two
  // runs a wave.
  constexpr bool kTable = Bins<T>::kExact;
  __shared__ double table[kTable ? Bins<__bf16>::kUsed : 1];
  const int64_t row = blockIdx.x / g.split;
  const int part = blockIdx.x % g.split;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const Asked a = asked(g, row);
  const T* x = static_cast<const T*>(g.logits) + row * g.ld;
  const int first = part * kWaves + wave, waves = g.split * kWaves;
  const bool use_table = kTable && a.temp >= 0.5 && g.runs * (g.run_cols / 512) > 8 * waves;
  if constexpr (kTable) {
    if (use_table) fill_table(table, Bins<T>::kUsed, [&](float v) { return exp2_product((double)v, a.k); });
  }
  // m: this lane's maximum in the run, and (without the table) the logit whose mass is 1
  float m = -INFINITY;
  double mass = 0.0;
  auto by_polynomial = [&](const Pack<T, VEC>& p, int) {
    float v[VEC], n = m;
    unpack(p, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) n = fmaxf(n, v[i]);
    const double ref = n == -INFINITY ? 0.0 : (double)n;
    if (__any(n > m) && mass > 0.0) mass *= exp2_product((double)m - ref, a.k);
    m = n;
#pragma unroll
    for (int i = 0; i < VEC; ++i) mass += exp2_product((double)v[i] - ref, a.k);
  };
  auto finish = [&](int run, bool table_done) {
    const float rm = wave_max(m);
    float ref = rm == -INFINITY ? 0.f : rm;
    if (table_done) ref = 0.f;
    else if (m != -INFINITY) mass *= exp2_product((double)m - (double)ref, a.k);
    mass = wave_total(mass);
    if (lane == 0) {
      g.run_mass[row * g.runs + run] = mass;
      g.run_max[row * g.runs + run] = rm;
      g.run_ref[row * g.runs + run] = ref;
    }
    m = -INFINITY;
    mass = 0.0;
  };
  if constexpr (kTable) {
    if (use_table) {
      each_run(
          x, g.cols, g.run_cols, g.runs, first, waves,
          [&](const Pack<T, VEC>& p, int) {
            float v[VEC];
            unpack(p, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) m = fmaxf(m, v[i]);
            // (a logit of 2^8 or more in size may take this sum out of range; the run is then done again)
            mass += sum_table(table, p, Bins<T>::kUsed, [&](float y) { return exp2_product((double)y, a.k); });
          },
          [&](int run) {
            const bool again = fabsf(wave_max(m)) >= 0x1p8f;
            if (again) {
              m = -INFINITY;
              mass = 0.0;
              each_run(x, g.cols, g.run_cols, run + 1, run, 1, by_polynomial, [](int) {});
            }
            finish(run, !again);
          });
      return;
    }
  }
  each_run(x, g.cols, g.run_cols, g.runs, first, waves, by_polynomial, [&](int run) { finish(run, false); });
}

// ---- hist and cut -----------------------------------------------------------
struct Fine {
  u64 mass[kFineBins];
  uint32_t count[kFineBins], key[kFineBins];
};
// What the bins of a block's columns need, and what finding a cut needs beside.
template <typename T> struct HistShared {
  Hist<T> hist;
};
struct BoundShared {
  float groups[kGroups], best[kGroups / kWave];
  int reach[kLanes];
};
template <typename T> struct CutShared : HistShared<T> {
  Fine fine;
  u64 ltmp[kWaves];
  uint32_t utmp[kWaves];
  // the bin that holds a cut
  int bin;
  uint32_t cnt_before;
  u64 mass_before;
};

// A thread's share of `BINS` bins: their counts and masses, and those of the bins before them.
template <int BINS>
struct Share {
  static constexpr int kEach = BINS / kLanes;
  static_assert(BINS % kLanes == 0, "whole turns");
  uint32_t count[kEach], total, before;
  u64 mass[kEach], mass_total, mass_before, all_mass;
  // (begins with a barrier)
  template <typename S, typename M>
  __device__ __forceinline__ Share(const uint32_t* counts, M&& mass_of, S& sh) : total(0), mass_total(0) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i) count[i] = counts[kEach * threadIdx.x + i], total += count[i];
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      mass[i] = count[i] ? mass_of(kEach * (int)threadIdx.x + i, count[i]) : 0, mass_total += mass[i];
    uint32_t all;
    before = block_before<uint32_t>(total, sh.utmp, &all);
    mass_before = block_before<u64>(mass_total, sh.ltmp, &all_mass);
  }
  // The bin whose running count reaches `count_target` (by count), or whose running mass reaches `mass_target`; what
  // lies before it goes to sh. Exactly one bin qualifies. Begins and ends with a barrier.
  template <typename S>
  __device__ __forceinline__ void find(S& sh, bool by_count, uint32_t count_target, u64 mass_target) const {
    __syncthreads();
    if (threadIdx.x == 0) sh.bin = BINS - 1, sh.cnt_before = 0, sh.mass_before = 0;
    __syncthreads();
    uint32_t cb = before;
    u64 mb = mass_before;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (by_count ? cb < count_target && count_target - cb <= count[i] : mb < mass_target && mass_target - mb <= mass[i])
        sh.bin = kEach * threadIdx.x + i, sh.cnt_before = cb, sh.mass_before = mb;
      cb += count[i];
      mb += mass[i];
    }
    __syncthreads();
  }
};

template <typename T>
struct Row {
  static constexpr int VEC = 16 / sizeof(T);
  typedef Bins<T> B;
  const T* x;
  int cols, run_cols, runs;
  float max;        // of the row
  double k;         // log2(e) / T
  float bin_step;   // linear bins: bins / (kRange T)
  double magic;

  __device__ __forceinline__ Row(const SampleArgs& g, int64_t row, const Asked& a, float max_)
      : x(static_cast<const T*>(g.logits) + row * g.ld),
        cols(g.cols),
        run_cols(g.run_cols),
        runs(g.runs),
        max(max_),
        k(a.k),
        bin_step((float)(B::kCount / kRange * kLn2D * a.k)),
        magic(g.magic) {}
  __device__ __forceinline__ double mass(float v) const { return exp2_product((double)v - (double)max, k); }
  __device__ __forceinline__ u64 fixed(double e) const {
    return __builtin_bit_cast(u64, e + magic) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ int bin_of(float v) const {
    if constexpr (B::kExact) {
      return B::of(v);
    } else {
      const float d = (max - v) * bin_step;
      return d < (float)(B::kCount - 1) ? (int)d : B::kCount - 1;
    }
  }
  __device__ __forceinline__ u64 mass_of_bin(const Hist<T>& h, int bin, uint32_t count) const {
    if constexpr (B::kExact) {
      if (B::several(bin)) return h.mass[B::slot(bin)];
      return count * fixed(mass(B::value(bin)));
    } else {
      return h.mass[bin];
    }
  }

  // Fills h with the runs of one block (part of split); bf16's masses are those of the bins of several.
  __device__ __forceinline__ void fill(Hist<T>& h, int part, int split, bool masses) const {
    for (int i = threadIdx.x; i < B::kCount; i += kLanes) h.count[i] = 0;
    for (int i = threadIdx.x; i < B::kMasses; i += kLanes) h.mass[i] = 0;
    __syncthreads();
    uint32_t low = 0;  // of the last bin, which masked tokens and most of a peaked row share
    u64 low_mass = 0;
    const int first = part * kWaves + (int)threadIdx.x / kWave, waves = split * kWaves;
    if constexpr (B::kExact) {
      constexpr int kLow = Bins<__bf16>::kUsed - 1;
      each_run(
          x, cols, run_cols, runs, first, waves,
          [&](const Pack<T, VEC>& p, int) {
            typename B::Two low2 = (typename B::Two)((short)B::kSide), high2 = (typename B::Two)((short)0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              typename B::Two rank;
              const typename B::Two b = B::of_two(p.w[j], &rank);
              low2 = __builtin_elementwise_min(low2, rank);
              high2 = __builtin_elementwise_max(high2, rank);
              if (b.x < kLow) atomicAdd(&h.count[b.x], 1u);
              else ++low;
              if (b.y < kLow) atomicAdd(&h.count[b.y], 1u);
              else ++low;
            }
            if (::min(low2.x, low2.y) == 0 || ::max(high2.x, high2.y) > B::kSide)
              each_several(p, [&](float v) { atomicAdd(&h.mass[B::slot(B::of(v))], fixed(mass(v))); });
          },
          [](int) {});
      low = wave_total(low);
      if (threadIdx.x % kWave == 0) atomicAdd(&h.count[kLow], low);
    } else {
      constexpr int kLow = B::kCount - 1;
      each_run(
          x, cols, run_cols, runs, first, waves,
          [&](const Pack<T, VEC>& p, int) {
            float v[VEC];
            unpack(p, v);
            u64 e[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) e[i] = 0;
            if (masses) {
#pragma unroll
              for (int i = 0; i < VEC; ++i) e[i] = fixed(mass(v[i]));
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const int b = bin_of(v[i]);
              if (b < kLow) {
                atomicAdd(&h.count[b], 1u);
                if (masses) atomicAdd(&h.mass[b], e[i]);
              } else {
                ++low;
                low_mass += e[i];
              }
            }
          },
          [](int) {});
      low = wave_total(low);
      low_mass = wave_total(low_mass);
      if (threadIdx.x % kWave == 0) {
        atomicAdd(&h.count[kLow], low);
        if (masses) atomicAdd(&h.mass[kLow], low_mass);
      }
    }
  }

  // The values that a bin can hold, as a range of keys; true (and the value) if there is one only.
  __device__ __forceinline__ bool one_value(int bin, uint32_t* klo, uint32_t* khi, float* value) const {
    if constexpr (B::kExact) {
      if (!B::several(bin)) {
        *value = B::value(bin);
        return true;
      }
      *khi = bin == 0 ? key_of<T>(max) : bin == B::kZero ? key_of<T>(0x1p-16f) : key_of<T>(-0x1p8f);
      *klo = bin == 0 ? key_of<T>(0x1p8f) : bin == B::kZero ? key_of<T>(-0x1p-16f) : 0;
      return false;
    } else {
      // with the roundings of bin_of to spare
      const double width = 1.0 / (double)bin_step, slack = 0x1p-21;
      const float hi = (float)((double)max - bin * width * (1 - slack));
      const float lo = (float)((double)max - (bin + 1) * width * (1 + slack));
      *khi = bin == 0 ? key_of<T>(max) : ::min(key_of<T>(max), key_of<T>(hi) + 1);
      const uint32_t kl = key_of<T>(lo);
      *klo = bin == B::kCount - 1 || kl == 0 ? 0 : kl - 1;
      int values = 0;
      if (*khi - *klo < 16) {
#pragma unroll 1
        for (uint32_t key = *klo; key <= *khi; ++key) {
          const float v = value_of<T>(key);
          if (bin_of(v) == bin) ++values, *value = v;
        }
      }
      return values == 1;
    }
  }

  // The cut after `count` logits (by count) or at mass `tau` (fixed point), and the mass that it keeps.
  // If the bin's logits fit into a list and `defer`, the cut stays inside the bin.
  __device__ __forceinline__ Cut find_cut(CutShared<T>& sh, const Share<B::kCount>& share, bool by_count, uint32_t count,
                                          u64 tau, bool masses, bool defer, u64* kept) const {
    share.find(sh, by_count, count, tau);
    const int bin = sh.bin;
    uint32_t cnt = sh.cnt_before;
    u64 above = sh.mass_before;
    uint32_t klo, khi;
    float value = max;
    uint32_t equal = 0;
    if (one_value(bin, &klo, &khi, &value)) {
      equal = sh.hist.count[bin];
    } else if (!B::kExact && defer && sh.hist.count[bin] <= (uint32_t)kPartList) {
      const float least = value_of<T>(klo);
      *kept = 0;
      return {least == least ? least : -INFINITY, 0xffffffffu, 0, cnt, by_count ? count - cnt : tau - above, bin + 1};
    } else {
      // 32 bits of key in turns of 11
#pragma unroll 1
      for (int turn = 0; turn < 3; ++turn) {
        int s = 0;
        while (((khi - klo) >> s) >= (uint32_t)kFineBins) ++s;
        __syncthreads();
        for (int i = threadIdx.x; i < kFineBins; i += kLanes) sh.fine.mass[i] = 0, sh.fine.count[i] = 0, sh.fine.key[i] = 0;
        __syncthreads();
        // one block reads the row: it needs many loads on their way, and finds few logits
        constexpr int kAhead = B::kExact ? 2 : 6, kStep = kLanes * VEC;
#pragma unroll 1
        for (int c0 = (int)threadIdx.x * VEC; c0 < cols; c0 += kAhead * kStep) {
          Pack<T, VEC> p[kAhead];
#pragma unroll
          for (int j = 0; j < kAhead; ++j)
            if (c0 + j * kStep + VEC <= cols) p[j] = load_pack_any<T, VEC>(x + c0 + j * kStep);
          uint32_t some = 0;
#pragma unroll
          for (int j = 0; j < kAhead; ++j) {
            float v[VEC];
            unpack(p[j], v);
            bool any = false;
#pragma unroll
            for (int i = 0; i < VEC; ++i) any = any || bin_of(v[i]) == bin;
            // (the columns of a vector that reaches past the row are looked at below)
            if (c0 + j * kStep + VEC <= cols ? any : c0 + j * kStep < cols) some |= 1u << j;
          }
#pragma unroll 1
          for (; some; some &= some - 1) {
            const int c = c0 + __builtin_ctz(some) * kStep;
#pragma unroll 1
            for (int i = c; i < ::min(c + VEC, cols); ++i) {
              const float y = to_f32<T>(x[i]);
              const uint32_t key = key_of<T>(y);
              if (bin_of(y) == bin && key >= klo && key <= khi) {
                const uint32_t b = (khi - key) >> s;
                atomicAdd(&sh.fine.count[b], 1u);
                atomicMax(&sh.fine.key[b], key);
                if (masses) atomicAdd(&sh.fine.mass[b], fixed(mass(y)));
              }
            }
          }
        }
        const Share<kFineBins> fine(sh.fine.count, [&](int b, uint32_t) { return sh.fine.mass[b]; }, sh);
        fine.find(sh, by_count, count - cnt, tau - above);
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
    Cut cut = {};
    cut.x = value;
    cut.equal = equal;
    const u64 each = masses ? fixed(mass(value)) : 0;
    // (by mass: the bin holds equal * each >= tau - above > 0)
    cut.ties = by_count ? count - cnt : (uint32_t)((tau - above + each - 1) / each);
    cut.count = cnt + cut.ties;
    *kept = above + each * cut.ties;
    return cut;
  }

  // The row's cut by top-k and top-p, from sh.hist.
  __device__ __forceinline__ Cut find(CutShared<T>& sh, const Asked& a, bool defer) const {
    const Share<B::kCount> share(
        sh.hist.count, [&](int b, uint32_t c) { return a.by_p ? mass_of_bin(sh.hist, b, c) : 0; }, sh);
    return find(sh, a, share, defer);
  }
  // (a top-p after a top-k needs the mass that this keeps)
  __device__ __forceinline__ Cut find(CutShared<T>& sh, const Asked& a, const Share<B::kCount>& share, bool defer) const {
    u64 total = share.all_mass;
    Cut cut = {INFINITY, 0, 0, 0};
    // by count, then by mass of what that kept
#pragma unroll 1
    for (int turn = a.by_k ? 0 : 1; turn < (a.by_p ? 2 : 1); ++turn) {
      const u64 tau = ::min(total, ::max((u64)1, (u64)ceil(fmax(a.top_p, 0.0) * (double)total)));
      u64 kept;
      const Cut c = find_cut(sh, share, turn == 0, (uint32_t)a.top_k, tau, a.by_p, defer && a.by_k != a.by_p, &kept);
      if (turn == 0 || !a.by_k || c.x > cut.x) cut = c;
      else if (c.x == cut.x && c.ties < cut.ties) cut.ties = c.ties, cut.count = c.count;
      total = kept;
    }
    return cut;
  }
};

// ---- lists --------------------------------------------------------------------
// A block's list: logits and their columns, in any order.
struct ListShared {
  uint32_t n;
  Listed list[kPartList];
  __device__ __forceinline__ void clear() {
    if (threadIdx.x == 0) n = 0;
    __syncthreads();
  }
  __device__ __forceinline__ void add(float x, int col) {
    const uint32_t at = atomicAdd(&n, 1u);
    if (at < (uint32_t)kPartList) list[at] = {x, col};
  }
  __device__ __forceinline__ void write(const SampleArgs& g, int64_t block) const {
    __syncthreads();
    for (int i = threadIdx.x; i < (int)min(n, (uint32_t)kPartList); i += kLanes) g.list[block * kPartList + i] = list[i];
    if (threadIdx.x == 0) g.listed[block] = n;
  }
};
// A row's lists in order, x descending and then by column; returns how many, -1 if a block's list or the row's has not
// room for all. Ends with a barrier.
struct OrderShared {
  u64 key[kList];  // larger x, then lower column, first
  uint32_t rank[kList];
  float x[kList];  // in order
  int col[kList];
};
__device__ __forceinline__ int order_listed(const SampleArgs& g, int64_t row, OrderShared& sh) {
  const int lane = threadIdx.x % kWave, t = threadIdx.x;
  const uint32_t in_part = lane < g.split ? g.listed[row * g.split + lane] : 0;
  const uint32_t incl = wave_scan(in_part);
  const int n = (int)of_lane63(incl);
  if (__any(in_part > (uint32_t)kPartList) || n > kList) return -1;
  int part = 0;
  uint32_t before_part = 0;
#pragma unroll 1
  for (int i = 0; i < g.split - 1; ++i) {
    const uint32_t upto = of_lane(incl, i);
    if ((uint32_t)t >= upto) part = i + 1, before_part = upto;
  }
  Listed mine = {0.f, 0};
  if (t < n) {
    mine = g.list[(row * g.split + part) * kPartList + (t - before_part)];
    sh.key[t] = (u64)key_of<float>(mine.x) << 32 | (uint32_t)~mine.col;
    sh.rank[t] = 0;
  }
  __syncthreads();
  // the rank of each, by comparison with all; the threads share them out
  int width = kWave;
  while (width < n) width *= 2;
  const int i = t & (width - 1), q = t / width, each = (n + kLanes / width - 1) / (kLanes / width);
  if (i < n) {
    const u64 key = sh.key[i];
    uint32_t rank = 0;
#pragma unroll 4
    for (int j = q * each; j < min(n, (q + 1) * each); ++j) rank += sh.key[j] > key ? 1 : 0;
    if (rank) atomicAdd(&sh.rank[i], rank);
  }
  __syncthreads();
  if (t < n) {
    const uint32_t r = sh.rank[t];
    sh.x[r] = mine.x;
    sh.col[r] = mine.col;
  }
  __syncthreads();
  return n;
}

// ---- mass -------------------------------------------------------------------
template <typename T> struct MassShared {
  ListShared list;  // of the bin that a cut is inside of
};
template <> struct MassShared<__bf16> {
  double table[Bins<__bf16>::kUsed];
};
// The kept masses of one block's share (part of split) of `runs`.
template <typename T>
__device__ __forceinline__ void mass_block(const SampleArgs& g, int64_t row, const Runs& runs, int part, int split,
                                           const Start& st, MassShared<T>& sh) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr bool kTable = Bins<T>::kExact;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const Row<T> r(g, row, st.a, st.max);
  const Cut cut = st.cut;
  const bool all_ties = cut.ties >= cut.equal;
  auto kept = [&](float v) { return all_ties ? v >= cut.x : v > cut.x; };
  double mass = 0.0;
  uint32_t ties = 0;  // (the wave's)
  const int first = runs.begin + part * kWaves + wave, waves = split * kWaves;
  auto count_ties = [&](const Pack<T, VEC>& p) {
    if (all_ties) return;
    float v[VEC];
    unpack(p, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) ties += __popcll(__ballot(v[i] == cut.x));
  };
  auto done = [&](int run) {
    mass = wave_total(mass);
    if (lane == 0) g.run_mass[row * g.runs + run] = mass, g.run_ties[row * g.runs + run] = ties;
    mass = 0.0;
    ties = 0;
  };
  if constexpr (kTable) {
    // The table is as many polynomials as it has bins: worth it for twice as many logits, of which more than a few are
    // kept.
    if (cut.count > (uint32_t)g.cols / 64 &&
        (int64_t)(runs.end - runs.begin) * g.run_cols > (int64_t)split * 2 * Bins<T>::kUsed) {
      const int reach = Bins<T>::of(cut.x);
      fill_table(sh.table, reach, [&](float v) { return v <= st.max && kept(v) ? r.mass(v) : 0.0; });
      each_run(
          r.x, g.cols, g.run_cols, runs.end, first, waves,
          [&](const Pack<T, VEC>& p, int) {
            mass += sum_table(sh.table, p, reach, [&](float y) { return kept(y) ? r.mass(y) : 0.0; });
            count_ties(p);
          },
          done);
      return;
    }
  }
  if constexpr (!kTable) {
    if (cut.inside) {
      const int inside = cut.inside - 1;
      sh.list.clear();
      each_run(
          r.x, g.cols, g.run_cols, runs.end, first, waves,
          [&](const Pack<T, VEC>& p, int c) {
            float v[VEC];
            unpack(p, v);
            float most = v[0];
#pragma unroll
            for (int i = 1; i < VEC; ++i) most = fmaxf(most, v[i]);
            if (!__any(most >= cut.x)) return;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const int bin = v[i] >= cut.x ? r.bin_of(v[i]) : inside + 1;
              mass += bin < inside ? r.mass(v[i]) : 0.0;
              if (bin == inside && c + i < g.cols) sh.list.add(v[i], c + i);
            }
          },
          done);
      sh.list.write(g, row * split + part);
      return;
    }
  }
  each_run(
      r.x, g.cols, g.run_cols, runs.end, first, waves,
      [&](const Pack<T, VEC>& p, int) {
        float v[VEC];
        unpack(p, v);
        float most = v[0];
#pragma unroll
        for (int i = 1; i < VEC; ++i) most = fmaxf(most, v[i]);
        if (__any(most >= cut.x)) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) mass += kept(v[i]) ? r.mass(v[i]) : 0.0;
          count_ties(p);
        }
      },
      done);
}

template <typename T>
__global__ __launch_bounds__(kLanes) void sample_mass_kernel(SampleArgs g) {
  __shared__ MassShared<T> sh;
  const int64_t row = blockIdx.x / g.split;
  const Start st(g, row, true);
  Runs runs = {0, g.runs};
  if (Bins<T>::kExact && g.chosen) {
    const int part = g.chosen[row].part;
    if (part >= 0) runs = runs_of(g, part);
  }
  if (st.ok && !st.a.by_list) mass_block<T>(g, row, runs, (int)(blockIdx.x % g.split), g.split, st, sh);
}

// ---- pick -------------------------------------------------------------------
struct PickShared {
  double dtmp[kWaves], base;
  uint32_t utmp[kWaves], ties;
  float ftmp[kWaves];
  int itmp[2 * kWaves], run;
};
// A cut inside a bin: orders the bin's list, adds the masses that are kept to their runs', and leaves the last kept logit
// and its column as the cut. The masses of a run are added in that order by one thread, so calls repeat.
struct InsideShared : OrderShared {
  double e[kPartList];
  int run[kPartList];
  u64 ltmp[kWaves];
  int last;
};
template <typename T>
__device__ __forceinline__ void cut_inside(const SampleArgs& g, int64_t row, Start& st, int* last_col, InsideShared& sh) {
  const Row<T> r(g, row, st.a, st.max);
  const int n = order_listed(g, row, sh), t = threadIdx.x;
  const float x = t < n ? sh.x[t] : -INFINITY;
  const int run = t < n ? sh.col[t] / g.run_cols : -1;
  const double e = t < n ? r.mass(x) : 0.0;
  u64 all;
  const u64 before = st.a.by_k ? (u64)t : block_before<u64>(t < n ? r.fixed(e) : 0, sh.ltmp, &all);
  const bool keep = t < n && before < st.cut.target;
  if (t == 0) sh.last = -1;
  __syncthreads();
  if (t < n) sh.e[t] = e, sh.run[t] = keep ? run : -1;
  const u64 kept_here = __ballot(keep);
  if (keep && t % kWave == 63 - __builtin_clzll(kept_here)) atomicMax(&sh.last, t);
  __syncthreads();
  const int last = sh.last;
  if (keep) {
    double sum = 0.0;
    bool first = true;
#pragma unroll 4
    for (int j = 0; j <= last; ++j) {
      const bool same = sh.run[j] == run;
      sum += same ? sh.e[j] : 0.0;
      first = first && !(same && j < t);
    }
    if (first) g.run_mass[row * g.runs + run] += sum;
  }
  // (none is listed if min-p cuts above the bin: x is its least then)
  if (last >= 0) st.cut.x = sh.x[last], *last_col = sh.col[last];
  __syncthreads();
}
// The row's token from the masses of its runs; `start` gives its Start.
template <typename T, typename S>
__device__ __forceinline__ void pick_row(const SampleArgs& g, int64_t row, S&& start, PickShared& sh,
                                         InsideShared* inside) {
  constexpr int kCols = 2;  // columns a thread, in order: runs of up to 2048
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const double* run_mass = g.run_mass + row * g.runs;
  const uint32_t* run_ties = g.run_ties + row * g.runs;
  const float *run_max = g.run_max + row * g.runs, *run_ref = g.run_ref + row * g.runs;
  Chosen from = {0.0, 0.0, 0, -1};
  if (Bins<T>::kExact && g.chosen) from = g.chosen[row];
  const Runs runs = from.part >= 0 ? runs_of(g, from.part) : Runs{0, g.runs};
  const int per = (runs.end - runs.begin + kLanes - 1) / kLanes;  // runs a thread, in order
  const int r0 = min(runs.end, runs.begin + (int)threadIdx.x * per), r1 = min(runs.end, r0 + per);
  // the first run's records, on the way while the row's start is put together (mostly there is no other)
  const int any_run = min(r0, g.runs - 1);
  double mass0 = run_mass[any_run];
  const uint32_t ties0 = run_ties[any_run];
  const float max0 = run_max[any_run], ref0 = run_ref[any_run];
  Start st = start();
  const Asked& a = st.a;
  const float u = g.u[row];

  bool fine = a.in_range;
  if (g.open) {
    float m = -INFINITY;
    for (int i = r0; i < r1; ++i) m = fmaxf(m, i == r0 ? max0 : run_max[i]);
    m = wave_max(m);
    if (lane == 0) sh.ftmp[wave] = m;
    __syncthreads();
    st.max = sh.ftmp[0];
    for (int i = 1; i < kWaves; ++i) st.max = fmaxf(st.max, sh.ftmp[i]);
  } else {
    fine = st.ok;
  }
  if (!fine) {
    if (threadIdx.x == 0) g.ids[row] = -1, g.logp[row] = __builtin_nanf("");
    return;
  }
  int last_col = g.cols;  // of the logits equal to the cut
  if constexpr (!Bins<T>::kExact) {
    if (inside && !g.open && st.cut.inside) {
      cut_inside<T>(g, row, st, &last_col, *inside);
      mass0 = run_mass[any_run];
    }
  }
  const float max = st.max;
  const Row<T> r(g, row, st.a, st.max);
  const Cut cut = g.open ? Cut{-INFINITY, 0xffffffffu, 0, 0} : st.cut;
  const bool all_ties = cut.ties >= cut.equal;
  const double each = all_ties ? 0.0 : r.mass(cut.x);

  // the masses of the runs (an open row's in terms of their own reference)
  uint32_t ties = 0, seen = 0;
  if (!all_ties) {
    for (int i = r0; i < r1; ++i) ties += i == r0 ? ties0 : run_ties[i];
    uint32_t all;
    seen = from.ties + block_before<uint32_t>(ties, sh.utmp, &all);
  }
  auto mass_of = [&](int i, uint32_t& ties_before) {
    const double m = i == r0 ? mass0 : run_mass[i];
    if (g.open) return m * exp2_product((double)(i == r0 ? ref0 : run_ref[i]) - (double)max, r.k);
    if (all_ties) return m;
    const uint32_t t = i == r0 ? ties0 : run_ties[i], left = cut.ties - min(cut.ties, ties_before);
    ties_before += t;
    return m + each * (double)min(left, t);
  };
  double mass = 0.0;
  uint32_t rank = seen;
#pragma unroll 1
  for (int i = r0; i < r1; ++i) mass += mass_of(i, rank);
  double total;
  const double before = from.before + block_before<double>(mass, sh.dtmp, &total);
  if (from.part >= 0) total = from.total;
  if (!(total > 0.0 && total < INFINITY && max < INFINITY)) {  // (only an open row's can be)
    if (threadIdx.x == 0) g.ids[row] = -1, g.logp[row] = __builtin_nanf("");
    return;
  }
  const double target = (double)u * total;
  // the first thread that passes the target; if none does, the last one with any mass
  if ((int)threadIdx.x == first_or_last(mass > 0.0 && before + mass > target, mass > 0.0, sh.itmp)) {
    double s = before;
    int run = r0;
    rank = seen;
#pragma unroll 1
    for (int i = r0; i < r1; ++i) {
      const uint32_t rank_before = rank;
      const double m = mass_of(i, rank);
      if (m > 0.0) run = i, sh.base = s, sh.ties = rank_before;
      s += m;
      if (m > 0.0 && s > target) break;
    }
    sh.run = run;
  }
  __syncthreads();
  const int c0 = sh.run * g.run_cols + (int)threadIdx.x * kCols, c1 = min(g.cols, (sh.run + 1) * g.run_cols);
  float v[kCols];
#pragma unroll
  for (int i = 0; i < kCols; ++i) v[i] = c0 + i < c1 ? to_f32<T>(r.x[c0 + i]) : -INFINITY;
  rank = sh.ties;
  const double base = sh.base;
  if (!all_ties) {
    ties = 0;
#pragma unroll
    for (int i = 0; i < kCols; ++i) ties += v[i] == cut.x ? 1 : 0;
    uint32_t all;
    rank += block_before<uint32_t>(ties, sh.utmp, &all);
  }
  double e[kCols];
  mass = 0.0;
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    bool keep = v[i] > cut.x || (v[i] == cut.x && c0 + i <= last_col);
    if (!all_ties && v[i] == cut.x) keep = rank++ < cut.ties;
    e[i] = keep ? r.mass(v[i]) : 0.0;
    mass += e[i];
  }
  double run_total;
  double s = base + block_before<double>(mass, sh.dtmp, &run_total);
  if ((int)threadIdx.x != first_or_last(mass > 0.0 && s + mass > target, mass > 0.0, sh.itmp)) return;
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
  g.logp[row] = (float)(((double)at - (double)max) * r.k * kLn2D) - log_fast(g.open ? (float)total : st.sum);
}

template <typename T>
__global__ __launch_bounds__(kLanes) void sample_pick_kernel(SampleArgs g) {
  __shared__ PickShared sh;
  const int64_t row = blockIdx.x;
  if (g.lists && asked(g, row).by_list) return;
  __shared__ InsideShared inside;  // (bf16 has no use for it, and no room is taken)
  pick_row<T>(g, row, [&] { return Start(g, row, true); }, sh, &inside);
}

// ---- list -------------------------------------------------------------------
// A lower bound of the k-th largest logit: the k-th largest of the maxima of kGroups disjoint sets of columns (each of
// those k is a logit of its own), put together from the scan's. Its value is the largest that k of them reach; four
// threads count for each.
__device__ __forceinline__ float least_of_top_k(const SampleArgs& g, int64_t row, const Asked& a, BoundShared& sh) {
  static_assert(kLanes == 4 * kGroups && kListMost <= kGroups, "four threads a group");
  const int n = 4 * g.runs, i = threadIdx.x % kGroups, part = threadIdx.x / kGroups;
  if (part == 0) {
    float m = -INFINITY;
#pragma unroll 1
    for (int j = i; j < n; j += kGroups) m = fmaxf(m, g.quarters[row * n + j]);
    sh.groups[i] = m;
  }
  __syncthreads();
  const float m = sh.groups[i];
  int reach = 0;
#pragma unroll 4
  for (int j = 0; j < kGroups / 4; ++j) reach += sh.groups[part * (kGroups / 4) + j] >= m ? 1 : 0;
  sh.reach[threadIdx.x] = reach;
  __syncthreads();
  if (part == 0) {
    for (int q = 1; q < 4; ++q) reach += sh.reach[q * kGroups + i];
    const float best = wave_max(reach >= (int)a.top_k ? m : -INFINITY);
    if (threadIdx.x % kWave == 0) sh.best[threadIdx.x / kWave] = best;
  }
  __syncthreads();
  float best = sh.best[0];
#pragma unroll
  for (int w = 1; w < kGroups / kWave; ++w) best = fmaxf(best, sh.best[w]);
  return best;
}

// Lists the logits of one block's runs that reach `least` (all finite ones if that is -inf), in any order.
template <typename T>
__device__ __forceinline__ void list_block(const T* x, const SampleArgs& g, int64_t row, int part, float least,
                                           ListShared& sh) {
  constexpr int VEC = 16 / sizeof(T);
  const float bound = fmaxf(least, -3.402823466e38f);
  sh.clear();
  each_run(
      x, g.cols, g.run_cols, g.runs, part * kWaves + (int)threadIdx.x / kWave, g.split * kWaves,
      [&](const Pack<T, VEC>& p, int c) {
        float v[VEC];
        unpack(p, v);
        float most = v[0];
#pragma unroll
        for (int i = 1; i < VEC; ++i) most = fmaxf(most, v[i]);
        if (!__any(most >= bound)) return;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          if (v[i] >= bound) sh.add(v[i], c + i);
        }
      },
      [](int) {});
  sh.write(g, row * g.split + part);
}

// Draws a row's token from its list; false if that has not room for all.
struct DrawShared : OrderShared {
  double e[kListMost];  // of the kept, by column
  int from[kListMost];
  double dtmp[kWaves];
  int itmp[2 * kWaves];
};
__device__ __forceinline__ bool draw_listed(const SampleArgs& g, int64_t row, const Start& st, DrawShared& sh) {
  const Asked& a = st.a;
  const int t = threadIdx.x;
  const float u = g.u[row];
  const int n = order_listed(g, row, sh);
  if (n < 0) return false;
  if (t < kListMost) sh.e[t] = 0.0;
  // the filters keep a prefix of that order
  const int k = min((int)a.top_k, n);
  const float x = t < k ? sh.x[t] : -INFINITY;
  const int col = t < k ? sh.col[t] : 0x7fffffff;
  const double e = exp2_product((double)x - (double)st.max, a.k);
  double total;
  const double above = block_before<double>(e, sh.dtmp, &total);
  const bool keep = t < k && (!a.by_p || t == 0 || above < a.top_p * total) && x >= least_of_min_p(a, st.max);
  __syncthreads();
  if (t < k) sh.col[t] = keep ? col : 0x7fffffff;
  __syncthreads();
  if (keep) {
    int at = 0;
#pragma unroll 4
    for (int j = 0; j < k; ++j) at += sh.col[j] < col ? 1 : 0;
    sh.e[at] = e;
    sh.from[at] = t;
  }
  __syncthreads();
  const double mass = t < kListMost ? sh.e[t] : 0.0;
  const double s = block_before<double>(mass, sh.dtmp, &total);
  if (t == first_or_last(mass > 0.0 && s + mass > (double)u * total, mass > 0.0, sh.itmp)) {
    const int r = sh.from[t];
    g.ids[row] = sh.col[r];
    g.logp[row] = (float)(((double)sh.x[r] - (double)st.max) * a.k * kLn2D) - log_fast(st.sum);
  }
  if (t == 0) g.cuts[row].count = 0;
  return true;
}

// What a row that goes by a list may need: the list is short of room if many logits equal the bound, and then one block
// goes the way of the others (cut, mass, pick) for the row (160 us for 64 rows of 151936 equal bf16 logits, 26 for
// random ones).
template <typename T>
union __align__(16) ListedShared {
  ListShared list;
  DrawShared draw;
  CutShared<T> cut;
  struct {
    MassShared<T> mass;
    PickShared pick;
  } rest;
  __device__ ListedShared() {}
};
template <typename T>
__device__ __forceinline__ void end_listed(const SampleArgs& g, int64_t row, Start& st, ListedShared<T>& sh) {
  if (draw_listed(g, row, st, sh.draw)) return;
  const Row<T> r(g, row, st.a, st.max);
  r.fill(sh.cut.hist, 0, 1, st.a.by_p);
  st.cut = r.find(sh.cut, st.a, false);
  st.cut_min_p();
  __syncthreads();
  mass_block<T>(g, row, {0, g.runs}, 0, 1, st, sh.rest.mass);
  __syncthreads();
  pick_row<T>(g, row, [&] { return st; }, sh.rest.pick, nullptr);
}

// A call whose rows all go by lists.
template <typename T>
__global__ __launch_bounds__(kLanes) void sample_list_kernel(SampleArgs g) {
  __shared__ BoundShared bound;
  __shared__ ListShared sh;
  const int64_t row = blockIdx.x / g.split;
  const Start st(g, row, false);
  if (!st.ok) return;
  list_block(static_cast<const T*>(g.logits) + row * g.ld, g, row, (int)(blockIdx.x % g.split),
             least_of_top_k(g, row, st.a, bound), sh);
}
template <typename T>
__global__ __launch_bounds__(kLanes) void sample_draw_kernel(SampleArgs g) {
  __shared__ ListedShared<T> sh;
  const int64_t row = blockIdx.x;
  Start st(g, row, false);
  if (st.ok) {
    end_listed(g, row, st, sh);
  } else if (threadIdx.x == 0) {
    g.ids[row] = -1;
    g.logp[row] = __builtin_nanf("");
  }
}

// ---- hist, cut ----------------------------------------------------------------
template <typename T, bool MIXED>
union __align__(16) RowShared {
  CutShared<T> cut;
  typename std::conditional<MIXED, ListedShared<T>, char>::type listed;
  __device__ RowShared() {}
};
template <typename T, bool MIXED>
union __align__(16) PartShared {
  HistShared<T> cut;
  typename std::conditional<MIXED, ListShared, char>::type listed;
  __device__ PartShared() {}
};
// WHOLE: one block has the whole row (split 1) and goes on to the cut. MIXED: rows may go by lists.
template <typename T, bool WHOLE, bool MIXED>
__global__ __launch_bounds__(kLanes) void sample_hist_kernel(SampleArgs g) {
  __shared__ typename std::conditional<WHOLE, RowShared<T, MIXED>, PartShared<T, MIXED>>::type sh;
  const int64_t row = blockIdx.x / g.split;
  const int part = (int)(blockIdx.x % g.split);
  Start st(g, row, false);
  if (MIXED && WHOLE && !st.ok && st.a.by_list && threadIdx.x == 0) g.ids[row] = -1, g.logp[row] = __builtin_nanf("");
  if (!st.ok || (!st.a.by_k && !st.a.by_p)) return;
  const Row<T> r(g, row, st.a, st.max);
  if constexpr (MIXED) {
    __shared__ BoundShared bound;
    if (st.a.by_list) {
      const float least = least_of_top_k(g, row, st.a, bound);
      if constexpr (WHOLE) {
        list_block(r.x, g, row, part, least, sh.listed.list);
        __syncthreads();
        end_listed(g, row, st, sh.listed);
      } else {
        list_block(r.x, g, row, part, least, sh.listed);
      }
      return;
    }
  }
  r.fill(sh.cut.hist, part, g.split, st.a.by_p);
  if constexpr (WHOLE) {
    const Cut cut = r.find(sh.cut, st.a, g.cols >= kListCols);
    if (threadIdx.x == 0) g.cuts[row] = cut;
  } else {
    __syncthreads();
    Hist<T>& to = static_cast<Hist<T>*>(g.hist)[blockIdx.x];
    static_assert(sizeof(Hist<T>) % 16 == 0 && Bins<T>::kMasses % 2 == 0, "whole vectors");
    // (masses first; they are not read without top-p)
    const int skip = st.a.by_p ? 0 : (int)(sizeof(u64) * Bins<T>::kMasses / 16);
    for (int i = skip + (int)threadIdx.x; i < (int)(sizeof(Hist<T>) / 16); i += kLanes)
      reinterpret_cast<u32x4*>(&to)[i] = reinterpret_cast<const u32x4*>(&sh.cut.hist)[i];
  }
}

// Element i of the `split` arrays that lie `stride` bytes apart, added up; the loads are in flight together.
template <typename V>
__device__ __forceinline__ V sum_parts(const char* p, size_t stride, int split) {
  V v[kMaxSplit], sum = {};
#pragma unroll
  for (int i = 0; i < kMaxSplit; ++i)
    if (i < split) v[i] = *reinterpret_cast<const V*>(p + i * stride);
#pragma unroll
  for (int i = 0; i < kMaxSplit; ++i)
    if (i < split) sum += v[i];
  return sum;
}

// (split > 1)
template <typename T, bool MIXED>
__global__ __launch_bounds__(kLanes) void sample_cut_kernel(SampleArgs g) {
  typedef u64 u64x2 __attribute__((ext_vector_type(2)));
  __shared__ RowShared<T, MIXED> all;
  const int64_t row = blockIdx.x;
  Start st(g, row, false);
  if (MIXED && !st.ok && st.a.by_list && threadIdx.x == 0) g.ids[row] = -1, g.logp[row] = __builtin_nanf("");
  if (!st.ok || (!st.a.by_k && !st.a.by_p)) return;
  if constexpr (MIXED) {
    if (st.a.by_list) {
      end_listed(g, row, st, all.listed);
      return;
    }
  }
  CutShared<T>& sh = all.cut;
  const Row<T> r(g, row, st.a, st.max);
  const Hist<T>* from = static_cast<const Hist<T>*>(g.hist) + row * g.split;
#pragma unroll 1
  for (int i = 4 * threadIdx.x; i < Bins<T>::kCount; i += 4 * kLanes)
    *reinterpret_cast<u32x4*>(&sh.hist.count[i]) = sum_parts<u32x4>((const char*)&from->count[i], sizeof(Hist<T>), g.split);
  if (st.a.by_p)
#pragma unroll 1
    for (int i = 2 * threadIdx.x; i < Bins<T>::kMasses; i += 2 * kLanes)
      *reinterpret_cast<u64x2*>(&sh.hist.mass[i]) =
          sum_parts<u64x2>((const char*)&from->mass[i], sizeof(Hist<T>), g.split);
  const Cut cut = r.find(sh, st.a, g.cols >= kListCols);
  if (threadIdx.x == 0) g.cuts[row] = cut;
}

// ---- count: bf16's scan, hist and cut -----------------------------------------
// bf16 bins do not depend on the maximum, so the row's first reading fills them; the maximum is the first bin with a
// count, and the sum of e^(z - max) that of the bins' masses. What the bins cannot tell (|x| >= 2^8, NaN, a maximum of
// |x| < 2^-16, or such x at a temperature that takes their masses far from 1) sets a flag, and the row's cut is made by
// scan and hist in one block.
constexpr double kTinyTemp = 0x1p-4;
constexpr int kFlag = 3;  // the place of h.mass that counts what was flagged
struct CountShared {
  ScanShared scan;
  int first[kWaves];
  // for choose_part
  float max;
  Cut cut;
  bool counted;  // the counts tell all kept masses
};

// Counts one block's runs into h. h.mass[1] sums 2^(x k) of |x| < 2^-16.
__device__ __forceinline__ void count_block(Hist<__bf16>& h, const SampleArgs& g, const __bf16* x, const Asked& a, int part) {
  typedef Bins<__bf16> B;
  for (int i = threadIdx.x; i < B::kCount; i += kLanes) h.count[i] = 0;
  if (threadIdx.x < B::kMasses) h.mass[threadIdx.x] = 0;
  __syncthreads();
  constexpr int kLow = B::kUsed - 1;
  uint32_t low = 0;
  const Runs runs = runs_of(g, part);
  each_run(
      x, g.cols, g.run_cols, runs.end, runs.begin + (int)threadIdx.x / kWave, kWaves,
      [&](const Pack<__bf16, 8>& p, int) {
        B::Two least = (B::Two)((short)B::kSide), most = (B::Two)((short)0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          B::Two rank;
          const B::Two b = B::of_two(p.w[j], &rank);
          least = __builtin_elementwise_min(least, rank);
          most = __builtin_elementwise_max(most, rank);
          if (b.x < kLow) atomicAdd(&h.count[b.x], 1u);
          else ++low;
          if (b.y < kLow) atomicAdd(&h.count[b.y], 1u);
          else ++low;
        }
        if (min(least.x, least.y) == 0 || max(most.x, most.y) > B::kSide)
          each_several(p, [&](float v) {
            if (fabsf(v) < 1.f && a.temp >= kTinyTemp)
              atomicAdd(&h.mass[1], __builtin_bit_cast(u64, exp2_product((double)v, a.k) + g.magic) & 0xfffffffffffffull);
            else
              atomicAdd(&h.mass[kFlag], 1ull);
          });
      },
      [](int) {});
  low = wave_total(low);
  if (threadIdx.x % kWave == 0) atomicAdd(&h.count[kLow], low);
}

// The row's maximum, sum and cut from the counts of all its columns. CHOOSES: choose_part comes after it.
template <bool CHOOSES>
__device__ __forceinline__ void cut_counted(CutShared<__bf16>& sh, CountShared& own, const SampleArgs& g, int64_t row,
                                            const Asked& a) {
  typedef Bins<__bf16> B;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const __bf16* x = static_cast<const __bf16*>(g.logits) + row * g.ld;
  __syncthreads();
  // the first bin with a count
  constexpr int kEach = B::kCount / kLanes;
  int first = B::kCount;
#pragma unroll
  for (int i = kEach - 1; i >= 0; --i)
    if (sh.hist.count[kEach * threadIdx.x + i]) first = kEach * threadIdx.x + i;
  const u64 some = __ballot(first < B::kCount);
  if (lane == 0) own.first[wave] = B::kCount;
  if (some && lane == __builtin_ctzll(some)) own.first[wave] = first;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) first = min(first, own.first[i]);
  float max = B::value(first), sum = 0.f;
  Cut cut = {-INFINITY, 0xffffffffu, 0, 0xffffffffu};
  const bool cuts = a.by_k || a.by_p, again = sh.hist.mass[kFlag] || B::several(first);
  if (again) scan_block(x, g, 0, 1, (float)a.k, nullptr, own.scan, &max, &sum);
  const Row<__bf16> r(g, row, a, max);
  const bool ok = !again || (sum > 0.f && sum < INFINITY && max < INFINITY);
  if (CHOOSES && threadIdx.x == 0) own.max = max, own.counted = !again && a.in_range;
  __syncthreads();
  if (again && ok && cuts) r.fill(sh.hist, 0, 1, a.by_p);
  if (!again && threadIdx.x == 0)  // in terms of the maximum from here on
    sh.hist.mass[1] = (u64)((double)sh.hist.mass[1] * exp2_product(-(double)max, a.k) + 0.5);
  if (ok && (cuts || !again)) {
    const Share<B::kCount> share(
        sh.hist.count, [&](int b, uint32_t c) { return r.mass_of_bin(sh.hist, b, c); }, sh);
    if (!again) sum = (float)((double)share.all_mass / (double)r.fixed(1.0));
    if (cuts) cut = r.find(sh, a, share, false);
  }
  if (threadIdx.x < g.split) {
    g.part_max[row * g.split + threadIdx.x] = threadIdx.x == 0 ? max : -INFINITY;
    g.part_sum[row * g.split + threadIdx.x] = threadIdx.x == 0 ? sum : 0.f;
  }
  if (threadIdx.x == 0) {
    g.cuts[row] = cut;
    if constexpr (CHOOSES) own.cut = cut;
  }
}

template <bool WHOLE>
__global__ __launch_bounds__(kLanes) void sample_count_kernel(SampleArgs g) {
  __shared__ __align__(16) typename std::conditional<WHOLE, CutShared<__bf16>, HistShared<__bf16>>::type sh;
  __shared__ CountShared own;
  const int64_t row = blockIdx.x / g.split;
  const int part = (int)(blockIdx.x % g.split);
  const Asked a = asked(g, row);
  const __bf16* x = static_cast<const __bf16*>(g.logits) + row * g.ld;
  count_block(sh.hist, g, x, a, part);
  if constexpr (WHOLE) {
    cut_counted<false>(sh, own, g, row, a);
  } else {
    __syncthreads();
    u32x4* to = reinterpret_cast<u32x4*>(static_cast<Hist<__bf16>*>(g.hist) + blockIdx.x);
    for (int i = threadIdx.x; i < (int)(sizeof(Hist<__bf16>) / 16); i += kLanes)
      to[i] = reinterpret_cast<const u32x4*>(&sh.hist)[i];
  }
}

// The part that the token lies in, from the parts' counts: the masses of that part's runs are all that is left to sum
// (256 rows of 151936 with top-p 0.95: two parts a row, mass 21 us, 34 for whole rows).
struct ChooseShared {
  double table[Bins<__bf16>::kUsed];
  double part[kWaves];
  uint32_t ties[kMaxSplit];
};
__device__ __forceinline__ Chosen choose_part(const SampleArgs& g, int64_t row, const Asked& a, float max, const Cut& cut,
                                              ChooseShared& sh) {
  typedef Bins<__bf16> B;
  Chosen none = {0.0, 0.0, 0, -1};
  // (a cut among |x| < 2^-16, or below -2^8 and not at -inf, splits a bin)
  const bool all = cut.x == -INFINITY;
  if (!all && B::several(B::of(cut.x))) return none;
  // the bin of |x| < 2^-16, as count_block sums it: with a maximum below it has none, and with one far above it too little
  // to say which of its logits have any mass
  const bool zero = cut.x < 0.f && max > 0.f;
  const double of_zero = zero ? exp2_product(-(double)max, a.k) : 0.0;
  if (zero && of_zero < 0x1p-1000) return none;
  const Row<__bf16> r(g, row, a, max);
  const Hist<__bf16>* from = static_cast<const Hist<__bf16>*>(g.hist) + row * g.split;
  const bool all_ties = cut.ties >= cut.equal;
  const int tie_bin = B::of(cut.x);  // (all_ties: not looked at)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const float u = g.u[row];
#pragma unroll 1
  for (int b = threadIdx.x; b < B::kUsed; b += kLanes) {
    const float v = B::value(b);
    const bool keep = !B::several(b) && v <= max && (all_ties ? v >= cut.x : v > cut.x);
    sh.table[b] = keep ? r.mass(v) : 0.0;
  }
  if (threadIdx.x < g.split && !all_ties) sh.ties[threadIdx.x] = from[threadIdx.x].count[tie_bin];
  __syncthreads();
  // several waves a part
  const int each = kWaves / g.split, part = wave / each, sub = wave % each;
  double mass = 0.0;
  if (part < g.split) {
    const int used = all ? B::kUsed : min(B::kUsed, B::of(cut.x) + 1);
#pragma unroll 4
    for (int b = (sub * kWave + lane) * 4; b < used; b += each * kWave * 4) {
      const u32x4 n = *reinterpret_cast<const u32x4*>(&from[part].count[b]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (b + i < B::kUsed) mass += (double)n[i] * sh.table[b + i];
    }
    if (sub == 0 && lane == 0 && zero) mass += (double)from[part].mass[1] / (double)r.fixed(1.0) * of_zero;
  }
  mass = wave_total(mass);
  if (lane == 0) sh.part[wave] = mass;
  __syncthreads();
  // (every wave goes through the parts by itself)
  const double sums = lane < kWaves ? sh.part[lane] : 0.0, one = all_ties ? 0.0 : r.mass(cut.x);
  const uint32_t equal = lane < g.split && !all_ties ? sh.ties[lane] : 0;
  Chosen c = none;
  const double total = wave_total(sums) + (all_ties ? 0.0 : one * (double)cut.ties);
  uint32_t ties = 0;
  double before = 0.0;
#pragma unroll 1
  for (int p = 0; p < g.split; ++p) {
    const uint32_t n = of_lane(equal, p), left = cut.ties - min(cut.ties, ties);
    double m = all_ties ? 0.0 : one * (double)min(left, n);
    for (int i = 0; i < each; ++i) m += of_lane(sums, p * each + i);
    if (m > 0.0) c = {before, total, ties, p};
    ties += n;
    before += m;
    if (m > 0.0 && before > (double)u * total) break;
  }
  return c;
}

// (split > 1)
__global__ __launch_bounds__(kLanes) void sample_count_cut_kernel(SampleArgs g) {
  typedef Bins<__bf16> B;
  __shared__ union __align__(16) All {
    CutShared<__bf16> cut;
    ChooseShared choose;
    __device__ All() {}
  } all;
  __shared__ CountShared own;
  CutShared<__bf16>& sh = all.cut;
  const int64_t row = blockIdx.x;
  const Hist<__bf16>* from = static_cast<const Hist<__bf16>*>(g.hist) + row * g.split;
  const Asked a = asked(g, row);
#pragma unroll 1
  for (int i = 4 * threadIdx.x; i < B::kCount; i += 4 * kLanes)
    *reinterpret_cast<u32x4*>(&sh.hist.count[i]) =
        sum_parts<u32x4>((const char*)&from->count[i], sizeof(Hist<__bf16>), g.split);
  if (threadIdx.x < B::kMasses) sh.hist.mass[threadIdx.x] =
      sum_parts<u64>((const char*)&from->mass[threadIdx.x], sizeof(Hist<__bf16>), g.split);
  cut_counted<true>(sh, own, g, row, a);
  __syncthreads();
  Chosen c = {0.0, 0.0, 0, -1};
  // (if fewer are kept than a wave's 512 logits hold one of, their masses cost less than the choice)
  if (g.chosen && own.counted && own.cut.count > (uint32_t)g.cols / 512) {
    Cut cut = own.cut;
    const Asked again = asked(g, row);  // (not kept in registers over all this)
    apply_min_p(cut, again, own.max);
    c = choose_part(g, row, again, own.max, cut, all.choose);
  }
  if (g.chosen && threadIdx.x == 0) g.chosen[row] = c;
}

// How a call is cut up. One block a CU, so want = CUs / rows blocks a row (two a CU have more bins to put together and a
// cut of their own to launch; us with one and two: 64 x 151936 bf16 top-p 42 and 46, min-p 22 and 26; 256 rows top-k 5000
// 55 and 63, no filter 33 and 36; fp32 61 and 65, 24 and 25, 125 and 129, 61 and 60), but two a CU for fp32 and fp16
// without top-k and top-p, whose fp64 exponentials need the waves (256 rows with min-p 0.02 87 and 72); and two blocks a
// row to choose from for bf16 rows that top-p alone cuts (256 rows with 0.95 70 and 75 us, with 0.5 60 and 52; 300 rows 102
// and 118, 88 and 88; 600 rows the same). Runs as long as they can be (each costs a sum over the wave) while there are
// eight for every wave, so that no wave has much more than another; and of the blocks that need the same number of turns,
// the fewest.
struct Shape {
  int64_t run_cols, runs, split;
};
Shape shape_of(int64_t rows, int64_t cols, int64_t cus, bool cuts, bool bf16, bool chooses) {
  Shape s;
  s.run_cols = 2048;
  while (s.run_cols > 512 && rows * cdiv(cols, s.run_cols) < 8 * cus * kWaves) s.run_cols /= 2;
  s.runs = cdiv(cols, s.run_cols);
  const int64_t blocks = cuts || bf16 ? cus : 2 * cus;
  int64_t want = std::max<int64_t>(1, std::min<int64_t>(kMaxSplit, blocks / std::max<int64_t>(rows, 1)));
  if (chooses && bf16 && want == 1 && rows <= 2 * cus && cols >= 2 * kChooseCols) want = 2;
  const int64_t turns = cdiv(s.runs, want * kWaves);
  s.split = cdiv(s.runs, turns * kWaves);
  return s;
}

struct Layout {
  size_t part_max, part_sum, quarters, run_mass, run_ties, run_max, run_ref, hist, cuts, chosen, list, listed, total;
};
Layout layout_of(int64_t rows, int64_t cols, const Shape& shape, bool cuts, bool bf16) {
  const int64_t runs = shape.runs, split = shape.split;
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
  l.run_ref = take((size_t)(rows * runs) * sizeof(float));
  l.part_max = take((size_t)(rows * split) * sizeof(float));
  l.part_sum = take((size_t)(rows * split) * sizeof(float));
  if (cuts) {
    l.cuts = take((size_t)rows * sizeof(Cut));
    if (cols >= kListCols) {
      l.quarters = take((size_t)(rows * runs) * 4 * sizeof(float));
      l.list = take((size_t)(rows * split) * kPartList * sizeof(Listed));
      l.listed = take((size_t)(rows * split) * sizeof(uint32_t));
    }
    if (split > 1 && bf16 && runs * shape.run_cols >= split * kChooseCols) l.chosen = take((size_t)rows * sizeof(Chosen));
    if (split > 1) l.hist = take((size_t)(rows * split) * (bf16 ? sizeof(Hist<__bf16>) : sizeof(Hist<float>)));
  }
  l.total = at;
  return l;
}

}  // namespace
}  // namespace hk

using namespace hk;

extern "C" {

size_t hk_sample_workspace_size(int64_t rows, int64_t cols, int cuts, int dtype, int device) {
  if (rows < 0 || rows >= (1LL << 31) || cols <= 0 || cols > (1 << 30)) return 0;
  const int cus = cu_count(device) > 0 ? cu_count(device) : 256;
  size_t most = 256;
  for (const bool chooses : {false, true})
    most = std::max(most, layout_of(rows, cols, shape_of(rows, cols, cus, cuts != 0, dtype == kBF16, chooses), cuts != 0,
                                    dtype == kBF16).total);
  return most;
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
  const bool cuts = top_k_rows || (top_k > 0 && top_k < cols) || top_p_rows || top_p < 1;
  const bool by_mass = (top_p_rows || top_p < 1) && !top_k_rows && !(top_k > 0 && top_k < cols);
  const Shape shape = shape_of(rows, cols, cus > 0 ? cus : 256, cuts, dtype == kBF16, by_mass);
  const int split = (int)shape.split;
  HK_REQUIRE(rows * split < (1LL << 32) / kLanes, "rows=%lld too many for one launch", (long long)rows);
  const bool masses = cuts || min_p_rows || min_p > 0;
  const Layout l = layout_of(rows, cols, shape, cuts, dtype == kBF16);
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
  g.run_cols = (int)shape.run_cols;
  g.runs = (int)shape.runs;
  g.split = split;
  g.open = !masses;
  g.has_cuts = cuts;
  int log2_cols = 0;
  while ((1LL << log2_cols) < cols + 2048) ++log2_cols;  // (with the last run's filling)
  g.magic = (double)(1ULL << (52 - std::min(43, 63 - log2_cols)));
  g.part_max = (float*)(ws + l.part_max);
  g.part_sum = (float*)(ws + l.part_sum);
  g.quarters = (float*)(ws + l.quarters);
  g.run_mass = (double*)(ws + l.run_mass);
  g.run_ties = (uint32_t*)(ws + l.run_ties);
  g.run_max = (float*)(ws + l.run_max);
  g.run_ref = (float*)(ws + l.run_ref);
  g.hist = ws + l.hist;
  g.cuts = (Cut*)(ws + l.cuts);
  g.list = (Listed*)(ws + l.list);
  g.listed = (uint32_t*)(ws + l.listed);
  // Lists: bf16 rows with a top-k each are counted instead, which takes one launch (and reading) fewer than the scan and
  // the counts or lists that the row's own k asks for.
  g.lists = cols >= kListCols && !(top_k_rows && dtype == kBF16);
  const bool all_listed = g.lists && !top_k_rows && top_k > 0 && top_k < cols && top_k <= list_most(g.runs);
  if (cuts && !all_listed && split > 1 && dtype == kBF16 && shape.runs * shape.run_cols >= split * kChooseCols)
    g.chosen = (Chosen*)(ws + l.chosen);
  const hipStream_t st = (hipStream_t)stream;
  const dim3 parts((unsigned)(rows * split)), each((unsigned)rows);
  const auto run = [&](void (*kernel)(SampleArgs), const dim3& grid, const char* name) {
    hipLaunchKernelGGL(kernel, grid, dim3(kLanes), 0, st, g);
    return check_launch(name);
  };
  auto launch = [&](auto tag) -> int {
    using T = decltype(tag);
    constexpr bool kCounts = Bins<T>::kExact;
    int rc = HK_OK;
    if (!masses) {
      rc = run(sample_open_kernel<T>, parts, "sample_open_kernel");
    } else if (!kCounts || !cuts || all_listed) {
      rc = run(sample_scan_kernel<T>, parts, "sample_scan_kernel");
    }
    if (rc != HK_OK) return rc;
    if (all_listed) {
      rc = run(sample_list_kernel<T>, parts, "sample_list_kernel");
      return rc != HK_OK ? rc : run(sample_draw_kernel<T>, each, "sample_draw_kernel");
    }
    if (cuts) {
      if constexpr (kCounts) {
        rc = run(split == 1 ? sample_count_kernel<true> : sample_count_kernel<false>, parts, "sample_count_kernel");
        if (rc == HK_OK && split > 1) rc = run(sample_count_cut_kernel, each, "sample_count_cut_kernel");
      } else {
        auto bins = [&](auto mixed) {
          constexpr bool kMixed = decltype(mixed)::value;
          const int bad = run(split == 1 ? sample_hist_kernel<T, true, kMixed> : sample_hist_kernel<T, false, kMixed>,
                              parts, "sample_hist_kernel");
          return bad != HK_OK || split == 1 ? bad : run(sample_cut_kernel<T, kMixed>, each, "sample_cut_kernel");
        };
        rc = top_k_rows ? bins(std::true_type{}) : bins(std::false_type{});
      }
    }
    if (rc == HK_OK && masses) rc = run(sample_mass_kernel<T>, parts, "sample_mass_kernel");
    return rc != HK_OK ? rc : run(sample_pick_kernel<T>, each, "sample_pick_kernel");
  };
  if (dtype == kF32) return launch(float{});
  if (dtype == kF16) return launch(_Float16{});
  return launch(__bf16{});
}

}  // extern "C"
