// RMSNorm and FusedAddRMSNorm with the output in 8 bits (OCP e4m3) and fp32
// scales, for gfx950: the input of an 8-bit projection in one pass.
//
//   s = round_T(x + r)                 (stored; without a residual s = x)
//   y = s * rstd * w,  rstd = 1 / sqrt(mean(s^2) + eps)
//   scale = max(max|y| / 448, 2^-100)  over the row, or a group of g columns
//   q = e4m3(y / scale)                round to nearest even
//
// rstd is one positive number a row, so max|y| = rstd * max|s w| and
// y / scale = s w * (rstd / scale): the sum of squares and the maxima come
// from the same look at the row and one exchange between its waves, and the
// row is quantised from s w once. y is never rounded to 16 bits on the way
// (the unquantised norms round s * rstd to T before the weight): the only
// roundings are s, which is an output, and q.
// The floor 2^-100 keeps an all-zero group at q = 0 with a usable scale.
// Maxima are taken over the bits of |s w| as integers, so that a NaN wins, as
// it does in a maximum over y: its group's scale and values come out NaN.
//
// HBM-bound: (1 + 2 add) es + 1 bytes an element. A row group of wpr waves
// holds its row in registers (16-byte vectors at any element alignment; a
// partial last vector is loaded by elements), as the unquantised kernels do.
// Stores are non-temporal: 45.7 us against 49.8 at 8192 x 4096 bf16 with a
// residual and groups of 128, 20.0 against 22.7 without the residual.
#include "hk_common.h"
#include "../../include/hilda_kernel_amd.h"

#include <algorithm>
#include <type_traits>

namespace hk {
namespace {

constexpr int kMaxWaves = 16;
constexpr float kE4m3Max = 448.f;
constexpr float kScaleMin = 0x1p-100f;

// 16 bytes at element alignment; past `left` elements: zeros
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_row(const T* p, int left) {
  if (left >= VEC) return load_pack_any<T, VEC>(p);
  float v[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = i < left ? to_f32<T>(p[i]) : 0.f;
  return pack<T, VEC>(v);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_row(T* p, const Pack<T, VEC>& v, int left) {
  if (left >= VEC) {
    store_pack_nt_any<T, VEC>(p, v);
    return;
  }
  float f[VEC];
  unpack(v, f);
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (i < left) p[i] = from_f32<T>(f[i]);
}
// VEC weights of W (which may be wider than the row's type) as floats
template <typename W, int VEC>
__device__ __forceinline__ void load_weight(const W* p, int left, float (&out)[VEC]) {
  if (left >= VEC) {
    if constexpr (sizeof(W) * VEC == 32) {
      float lo[VEC / 2], hi[VEC / 2];
      unpack(load_pack_any<W, VEC / 2>(p), lo);
      unpack(load_pack_any<W, VEC / 2>(p + VEC / 2), hi);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) out[i] = lo[i], out[VEC / 2 + i] = hi[i];
    } else {
      unpack(load_pack_any<W, VEC>(p), out);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) out[i] = i < left ? to_f32<W>(p[i]) : 0.f;
}

// four values to e4m3, lowest in the lowest byte
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
typedef u32x2 any_u32x2 __attribute__((aligned(1)));
typedef uint32_t any_u32 __attribute__((aligned(1)));
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&v)[VEC], int left) {
  uint32_t w[VEC / 4];
#pragma unroll
  for (int i = 0; i < VEC / 4; ++i) w[i] = e4m3x4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  if (left >= VEC) {
    if constexpr (VEC == 8) __builtin_nontemporal_store(u32x2{w[0], w[1]}, reinterpret_cast<any_u32x2*>(p));
    else __builtin_nontemporal_store(w[0], reinterpret_cast<any_u32*>(p));
    return;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (i < left) p[i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return f32_bits(v) & 0x7fffffffu; }
template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, ROW_MASK, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  v = dpp_umax<dpp::kXor1>(v);
  v = dpp_umax<dpp::kXor2>(v);
  v = dpp_umax<dpp::kHalfMirror>(v);
  v = dpp_umax<dpp::kMirror>(v);
  v = dpp_umax<dpp::kBcast15, 0xa>(v);
  v = dpp_umax<dpp::kBcast31, 0xc>(v);
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// the maximum over aligned runs of `lanes` lanes (4, 8, 16, 32 or 64), in every lane of the run
__device__ __forceinline__ uint32_t lanes_umax(uint32_t v, int lanes) {
  v = dpp_umax<dpp::kXor1>(v);
  v = dpp_umax<dpp::kXor2>(v);
  if (lanes >= 8) v = dpp_umax<dpp::kHalfMirror>(v);
  if (lanes >= 16) v = dpp_umax<dpp::kMirror>(v);
  if (lanes >= 32) v = max(v, (uint32_t)__shfl_xor((int)v, 16, kWave));
  if (lanes >= 64) v = max(v, (uint32_t)__shfl_xor((int)v, 32, kWave));
  return v;
}

// scale and the factor that turns s w into q, from rstd and max|s w|
__device__ __forceinline__ void scale_of(float rstd, uint32_t amax, float* scale, float* mult) {
  const float v = rstd * bits_f32(amax) * (1.f / kE4m3Max);
  *scale = !(v <= kScaleMin) ? v : kScaleMin;  // (a NaN stays)
  *mult = rstd * rcp_fast(*scale);
}

template <typename T, typename W, int NCH, bool ADD, bool GROUPS, int LB>
__global__ __launch_bounds__(LB) void rmsnorm_quant_kernel(uint8_t* __restrict__ q, float* __restrict__ scale_out,
                                                           T* __restrict__ s_out, float* __restrict__ rstd_out,
                                                           const T* __restrict__ x, const T* __restrict__ r,
                                                           const W* __restrict__ w, int64_t rows, int cols, int64_t ld,
                                                           int wpr, int group_lanes, float eps) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ float red_sum[kMaxWaves];
  __shared__ uint32_t red_max[kMaxWaves];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int rpb = blockDim.x / (kWave * wpr);
  const int rib = wave / wpr;
  const int lr = (wave % wpr) * kWave + lane;
  const int gl = wpr * kWave;
  const int64_t row = (int64_t)blockIdx.x * rpb + rib;
  const bool valid = row < rows;

  Pack<T, VEC> xv[NCH];
  float wf[NCH][VEC];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int col = (j * gl + lr) * VEC;
    if (valid && col < cols) {
      const int left = cols - col;
      xv[j] = load_row<T, VEC>(x + row * ld + col, left);
      if constexpr (ADD) {
        const Pack<T, VEC> rv = load_row<T, VEC>(r + row * ld + col, left);
        float a[VEC], b[VEC];
        unpack(xv[j], a);
        unpack(rv, b);
#pragma unroll
        for (int i = 0; i < VEC; ++i) a[i] += b[i];
        xv[j] = pack<T, VEC>(a);
        store_row<T, VEC>(s_out + row * cols + col, xv[j], left);
      }
      load_weight<W, VEC>(w + col, left, wf[j]);
    }
  }
  float ss = 0.f;
  uint32_t am[NCH];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int col = (j * gl + lr) * VEC;
    am[j] = 0;
    if (valid && col < cols) {
      float a[VEC];
      unpack(xv[j], a);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        ss = fmaf(a[i], a[i], ss);
        am[j] = max(am[j], abs_bits(a[i] * wf[j][i]));
      }
    }
  }
  ss = wave_sum(ss);
  uint32_t row_max = 0;
  if constexpr (!GROUPS) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) row_max = max(row_max, am[j]);
    row_max = wave_umax(row_max);
  }
  if (wpr > 1) {
    if (lane == 0) {
      red_sum[wave] = ss;
      if constexpr (!GROUPS) red_max[wave] = row_max;
    }
    __syncthreads();
    ss = 0.f;
    for (int i = 0; i < wpr; ++i) {
      ss += red_sum[rib * wpr + i];
      if constexpr (!GROUPS) row_max = max(row_max, red_max[rib * wpr + i]);
    }
  }
  const float rstd = __builtin_amdgcn_rsqf(ss / (float)cols + eps);
  if (rstd_out && valid && lr == 0) rstd_out[row] = rstd;
  float scale, mult;
  if constexpr (!GROUPS) {
    scale_of(rstd, row_max, &scale, &mult);
    if (valid && lr == 0) scale_out[row] = scale;
  }
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    const int col = (j * gl + lr) * VEC;
    if constexpr (GROUPS) scale_of(rstd, lanes_umax(am[j], group_lanes), &scale, &mult);
    if (valid && col < cols) {
      float a[VEC];
      unpack(xv[j], a);
#pragma unroll
      for (int i = 0; i < VEC; ++i) a[i] = a[i] * wf[j][i] * mult;
      store_e4m3<VEC>(q + row * cols + col, a, cols - col);
      if constexpr (GROUPS) {
        if (lane % group_lanes == 0)
          scale_out[row * (cols / (group_lanes * VEC)) + col / (group_lanes * VEC)] = scale;
      }
    }
  }
}

// Rows too long for the register form: one 1024-lane block a row, two passes
// (the sum of squares and the row's maximum while s is stored; then s is read
// back, by the lane that wrote it, and quantised).
constexpr int kStreamLanes = 1024;
template <typename T, typename W, bool ADD, bool GROUPS>
__global__ __launch_bounds__(kStreamLanes) void rmsnorm_quant_stream_kernel(
    uint8_t* __restrict__ q, float* __restrict__ scale_out, T* s_out, float* __restrict__ rstd_out,
    const T* __restrict__ x, const T* __restrict__ r, const W* __restrict__ w, int cols, int64_t ld, int group_lanes,
    float eps) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int NW = kStreamLanes / kWave;
  __shared__ float red_sum[NW];
  __shared__ uint32_t red_max[NW];
  const int64_t row = blockIdx.x;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  float ss = 0.f;
  uint32_t am = 0;
  for (int col = (int)threadIdx.x * VEC; col < cols; col += kStreamLanes * VEC) {
    const int left = cols - col;
    Pack<T, VEC> xv = load_row<T, VEC>(x + row * ld + col, left);
    float a[VEC], wf[VEC];
    unpack(xv, a);
    if constexpr (ADD) {
      float b[VEC];
      unpack(load_row<T, VEC>(r + row * ld + col, left), b);
#pragma unroll
      for (int i = 0; i < VEC; ++i) a[i] += b[i];
      xv = pack<T, VEC>(a);
      store_row<T, VEC>(s_out + row * cols + col, xv, left);
      unpack(xv, a);
    }
    if constexpr (!GROUPS) load_weight<W, VEC>(w + col, left, wf);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      ss = fmaf(a[i], a[i], ss);
      if constexpr (!GROUPS) am = max(am, abs_bits(a[i] * wf[i]));
    }
  }
  ss = wave_sum(ss);
  am = wave_umax(am);
  if (lane == 0) red_sum[wave] = ss, red_max[wave] = am;
  __syncthreads();
  ss = 0.f;
  for (int i = 0; i < NW; ++i) ss += red_sum[i], am = max(am, red_max[i]);
  const float rstd = __builtin_amdgcn_rsqf(ss / (float)cols + eps);
  float scale, mult;
  if constexpr (!GROUPS) scale_of(rstd, am, &scale, &mult);
  if (threadIdx.x == 0) {
    if (rstd_out) rstd_out[row] = rstd;
    if constexpr (!GROUPS) scale_out[row] = scale;
  }
  // every lane takes every turn: the groups' maxima move between lanes
  for (int c0 = 0; c0 < cols; c0 += kStreamLanes * VEC) {
    const int col = c0 + (int)threadIdx.x * VEC;
    const int left = cols - col;
    float a[VEC], wf[VEC];
    am = 0;
    if (left > 0) {
      unpack(load_row<T, VEC>(ADD ? s_out + row * cols + col : x + row * ld + col, left), a);
      load_weight<W, VEC>(w + col, left, wf);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        a[i] *= wf[i];
        am = max(am, abs_bits(a[i]));
      }
    }
    if constexpr (GROUPS) scale_of(rstd, lanes_umax(am, group_lanes), &scale, &mult);
    if (left > 0) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) a[i] *= mult;
      store_e4m3<VEC>(q + row * cols + col, a, left);
      if constexpr (GROUPS) {
        if (lane % group_lanes == 0)
          scale_out[row * (cols / (group_lanes * VEC)) + col / (group_lanes * VEC)] = scale;
      }
    }
  }
}

template <typename T> struct Tag { using type = T; };

// w has the dtype of x, or is fp32
template <typename F>
int dispatch_xw(int dt_x, int dt_w, F&& f) {
  if (dt_x == kF32 && dt_w == kF32) return f(Tag<float>{}, Tag<float>{});
  if (dt_x == kBF16 && dt_w == kBF16) return f(Tag<__bf16>{}, Tag<__bf16>{});
  if (dt_x == kBF16 && dt_w == kF32) return f(Tag<__bf16>{}, Tag<float>{});
  if (dt_x == kF16 && dt_w == kF16) return f(Tag<_Float16>{}, Tag<_Float16>{});
  if (dt_x == kF16 && dt_w == kF32) return f(Tag<_Float16>{}, Tag<float>{});
  set_error("unsupported dtype pair (x=%d, w=%d): w must match x or be fp32", dt_x, dt_w);
  return HK_EINVAL;
}

struct Geom {
  int nch;  // 16-byte vectors a lane: 1, 2 or 4
  int wpr;  // waves a row, 1..16
};

// 16 elements a lane and as many waves as that takes (5 for 5120 16-bit columns, not a power of two), 4 vectors a lane
// for 16-bit rows longer than 16 waves hold. With a residual 8 elements a lane while a row then has 2 to 8 waves: the
// two streams in and two out want more rows on their way (8192 x 4096 bf16, 235 MB: 43.0 us against 45.5 with 16
// elements and 50.1 with 32, a copy of the same bytes 40.7; without a residual 20.7 against 19.9).
bool choose_geom(int64_t cols, int vec, bool add, Geom* g) {
  const int64_t nv = cdiv(cols, (int64_t)vec);
  int nch = 16 / vec;
  const int64_t eights = cdiv(nv, (int64_t)kWave * nch / 2);
  if (add && eights > 2 && eights <= 8) nch /= 2;
  while (nch > 1 && nv <= kWave * nch / 2) nch /= 2;
  while (nch < 4 && cdiv(nv, (int64_t)kWave * nch) > kMaxWaves) nch *= 2;
  const int64_t wpr = cdiv(nv, (int64_t)kWave * nch);
  if (wpr > kMaxWaves) return false;
  *g = {nch, (int)wpr};
  return true;
}

}  // namespace
}  // namespace hk

using namespace hk;

extern "C" {

int hk_rms_norm_quant_fwd(void* q, float* scale, void* s, float* rstd, const void* x, const void* r, const void* w,
                          int64_t rows, int64_t cols, int64_t ld, int64_t group, int dtype_x, int dtype_w, float eps,
                          hk_stream_t stream) {
  HK_REQUIRE(dtype_x == kF32 || dtype_x == kF16 || dtype_x == kBF16, "invalid dtype code x=%d", dtype_x);
  HK_REQUIRE(rows >= 0 && cols > 0, "invalid shape rows=%lld cols=%lld", (long long)rows, (long long)cols);
  HK_REQUIRE(cols <= (1 << 30) && rows < (1LL << 31), "rows=%lld cols=%lld too large", (long long)rows,
             (long long)cols);
  HK_REQUIRE(ld >= cols, "row stride smaller than cols");
  HK_REQUIRE(group == 0 || group == 32 || group == 64 || group == 128 || group == 256,
             "group %lld: 0 (the row), 32, 64, 128 or 256 columns", (long long)group);
  HK_REQUIRE(group == 0 || cols % group == 0, "cols=%lld is not a multiple of the group %lld", (long long)cols,
             (long long)group);
  HK_REQUIRE(rows == 0 || (s == nullptr) == (r == nullptr), "s and r are given together, or neither");
  if (rows == 0) return HK_OK;
  HK_REQUIRE(q && scale && x && w, "null pointer argument");
  const hipStream_t st = (hipStream_t)stream;
  return dispatch_xw(dtype_x, dtype_w, [&](auto tx, auto tw) {
    using T = typename decltype(tx)::type;
    using W = typename decltype(tw)::type;
    constexpr int VEC = 16 / sizeof(T);
    const int group_lanes = (int)(group / VEC);
    auto with = [&](auto add_c, auto groups_c) {
      constexpr bool ADD = decltype(add_c)::value, GROUPS = decltype(groups_c)::value;
      Geom g;
      if (!choose_geom(cols, VEC, ADD, &g)) {
        HK_REQUIRE(rows < (1LL << 32) / kStreamLanes, "rows=%lld too many for one launch", (long long)rows);
        hipLaunchKernelGGL((rmsnorm_quant_stream_kernel<T, W, ADD, GROUPS>), dim3((unsigned)rows), dim3(kStreamLanes),
                           0, st, (uint8_t*)q, scale, (T*)s, rstd, (const T*)x, (const T*)r, (const W*)w, (int)cols,
                           ld, group_lanes, eps);
        return check_launch("rmsnorm_quant_stream_kernel");
      }
      const int rows_block = std::max(1, 4 / g.wpr), block = rows_block * g.wpr * kWave;
      const int64_t grid = cdiv(rows, (int64_t)rows_block);
      HK_REQUIRE(grid < (1LL << 32) / block, "rows=%lld too many for one launch", (long long)rows);
      auto launch = [&](auto nch_c, auto lb_c) {
        constexpr int NCH = decltype(nch_c)::value, LB = decltype(lb_c)::value;
        hipLaunchKernelGGL((rmsnorm_quant_kernel<T, W, NCH, ADD, GROUPS, LB>), dim3((unsigned)grid), dim3(block), 0, st,
                           (uint8_t*)q, scale, (T*)s, rstd, (const T*)x, (const T*)r, (const W*)w, rows, (int)cols, ld,
                           g.wpr, group_lanes, eps);
        return check_launch("rmsnorm_quant_kernel");
      };
      auto bound = [&](auto nch_c) {
        if (block <= 256) return launch(nch_c, std::integral_constant<int, 256>{});
        if (block <= 512) return launch(nch_c, std::integral_constant<int, 512>{});
        return launch(nch_c, std::integral_constant<int, 1024>{});
      };
      if (g.nch == 1) return bound(std::integral_constant<int, 1>{});
      if (g.nch == 2) return bound(std::integral_constant<int, 2>{});
      return bound(std::integral_constant<int, 4>{});
    };
    if (r) return group ? with(std::true_type{}, std::true_type{}) : with(std::true_type{}, std::false_type{});
    return group ? with(std::false_type{}, std::true_type{}) : with(std::false_type{}, std::false_type{});
  });
}

}  // extern "C"
