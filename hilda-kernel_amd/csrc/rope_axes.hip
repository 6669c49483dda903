// Rotary position embedding with several position axes (time, height, width
// of images and video) for gfx950.
//
// Pair i < D/2 of a head turns by the angle of ONE axis a(i):
//   P = positions[a(i), b, t],  c = cos[P, i],  s = sin[P, i]
//   y[i]       = x[i] c - x[i + D/2] s
//   y[i + D/2] = x[i + D/2] c + x[i] s
// a(i) is given by sections n_0 .. n_{A-1} (sum D/2): either runs of n_a
// pairs, or interleaved (a = i mod A while i < A n_a, else axis 0). The
// backward is the same map with -s. Arithmetic is fp32, rounded once.
//
// HBM-bound: every element of q and k is read and written once, 3 flops an
// element. A block takes a few tokens with all their heads: its threads gather
// the tokens' (cos, sin) into LDS, one pair each (position, then table entry;
// caches hold both), while the loads of their first heads are in flight; then a
// lane walks over heads with the cos/sin of its VEC pairs in registers. With
// the angles fetched by every lane for itself, 8 pairs of up to 3 axes each,
// the selects alone took as long as the copy (53 us instead of 31.4 for q and k
// of 8192 tokens x 40 heads x 128 bf16, 168 MB; a copy of them 30.2).
// Consecutive lanes cover the chunks of a head, then heads of the token
// ([B, T, H, D] storage) or tokens of the head ([B, H, T, D] storage), so that
// a wave touches one contiguous span either way. Stores are non-temporal (1 us
// of the 31.4).
//
// A position outside [0, table rows) reads nothing and gives NaN in the pairs
// of its axis.
#include "hk_common.h"
#include "../../include/hilda_kernel_amd.h"

#include <algorithm>
#include <type_traits>

namespace hk {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxAxes = 4;

struct Axes {
  int count;
  int interleaved;
  int n[kMaxAxes];  // sections; runs: n[a] = first pair past axis a
};

struct Heads {
  int count;
  int64_t is_b, is_h, is_t;  // element strides of the input
  int64_t os_b, os_h, os_t;  // and of the output
};

struct RopeAxesArgs {
  Heads q, k;
  const void* positions;
  int64_t ps_a, ps_b, ps_t;
  int64_t table_rows, table_ld;
  Axes axes;
  uint32_t T, half;
  uint32_t chunks;       // half / VEC
  uint32_t lanes;        // lanes of one head: min(chunks, 256)
  uint32_t slots;        // a lane walks heads slot, slot + slots, ...
  uint32_t tokens_block; // tokens a block covers
  int64_t tokens;        // B * T
  float sgn;
};

__device__ __forceinline__ int axis_of(const Axes& ax, int pair) {
  if (ax.interleaved) {
    int a = pair % ax.count;
    int n = ax.n[0];
#pragma unroll
    for (int j = 1; j < kMaxAxes; ++j) n = a == j ? ax.n[j] : n;
    return pair < ax.count * n ? a : 0;
  }
  int a = 0;
#pragma unroll
  for (int j = 0; j < kMaxAxes - 1; ++j) a += (j < ax.count - 1 && pair >= ax.n[j]) ? 1 : 0;
  return a;
}

// Block: g.tokens_block tokens of all heads. Its threads first fetch one
// (cos, sin) each into LDS, while their first heads' loads are in flight.
template <typename T, typename C, typename P, int VEC, bool HEAD_MAJOR, int UNROLL>
__global__ __launch_bounds__(kThreads) void rope_axes_kernel(T* __restrict__ q_out, const T* __restrict__ q_in,
                                                             T* __restrict__ k_out, const T* __restrict__ k_in,
                                                             const C* __restrict__ cosp, const C* __restrict__ sinp,
                                                             RopeAxesArgs g) {
  __shared__ __align__(16) float angle[2][kThreads * VEC];  // cos and sin of [token of the block][pair]
  const uint32_t lane = threadIdx.x % g.lanes;
  const uint32_t rest = threadIdx.x / g.lanes;
  const uint32_t local = HEAD_MAJOR ? rest % g.tokens_block : rest / g.slots;
  const uint32_t slot = HEAD_MAJOR ? rest / g.tokens_block : rest % g.slots;
  const uint32_t chunk = blockIdx.y * g.lanes + lane;
  const int64_t n = (int64_t)blockIdx.x * g.tokens_block + local;
  const bool live = local < g.tokens_block && slot < g.slots && n < g.tokens && chunk < g.chunks;
  const uint32_t b = live ? (uint32_t)n / g.T : 0, t = live ? (uint32_t)n % g.T : 0;
  const int first = (int)chunk * VEC;
  const int heads = live ? g.q.count + g.k.count : 0;

  Pack<T, VEC> p1[UNROLL], p2[UNROLL];
  T* out[UNROLL];
  const int64_t iq = b * g.q.is_b + t * g.q.is_t + first, ik = b * g.k.is_b + t * g.k.is_t + first;
  const int64_t oq = b * g.q.os_b + t * g.q.os_t + first, ok = b * g.k.os_b + t * g.k.os_t + first;
  auto load = [&](int h0) {
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int h = h0 + j * (int)g.slots;
      if (h < heads) {
        const T* in = h < g.q.count ? q_in + (iq + h * g.q.is_h) : k_in + (ik + (h - g.q.count) * g.k.is_h);
        out[j] = h < g.q.count ? q_out + (oq + h * g.q.os_h) : k_out + (ok + (h - g.q.count) * g.k.os_h);
        p1[j] = load_pack<T, VEC>(in);
        p2[j] = load_pack<T, VEC>(in + g.half);
      }
    }
  };
  load((int)slot);
  const int at = (int)(local * g.lanes + lane) * VEC;
  if (live) {
    const P* pos = static_cast<const P*>(g.positions) + b * g.ps_b + t * g.ps_t;
    for (int i = (int)slot; i < VEC; i += (int)g.slots) {
      const int64_t p = (int64_t)pos[axis_of(g.axes, first + i) * g.ps_a];
      float c = __builtin_nanf(""), s = c;
      if (p >= 0 && p < g.table_rows) {
        c = to_f32<C>(cosp[p * g.table_ld + first + i]);
        s = to_f32<C>(sinp[p * g.table_ld + first + i]) * g.sgn;
      }
      angle[0][at + i] = c;
      angle[1][at + i] = s;
    }
  }
  __syncthreads();
  if (!live) return;
  float c[VEC], s[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) c[i] = angle[0][at + i], s[i] = angle[1][at + i];

  for (int h0 = (int)slot; h0 < heads;) {
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      if (h0 + j * (int)g.slots < heads) {
        float x1[VEC], x2[VEC], y1[VEC], y2[VEC];
        unpack(p1[j], x1);
        unpack(p2[j], x2);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          y1[i] = x1[i] * c[i] - x2[i] * s[i];
          y2[i] = x2[i] * c[i] + x1[i] * s[i];
        }
        store_pack_nt<T, VEC>(out[j], pack<T, VEC>(y1));
        store_pack_nt<T, VEC>(out[j] + g.half, pack<T, VEC>(y2));
      }
    }
    h0 += (int)g.slots * UNROLL;
    load(h0);
  }
}

template <typename T> struct Tag { using type = T; };

template <typename F>
int dispatch_t(int dt, F&& f) {
  switch (dt) {
    case kF32: return f(Tag<float>{});
    case kF16: return f(Tag<_Float16>{});
    case kBF16: return f(Tag<__bf16>{});
  }
  set_error("invalid dtype code %d", dt);
  return HK_EINVAL;
}

bool heads_ok(const Heads& h, const void* in, const void* out, int vec, int es) {
  const int64_t s[6] = {h.is_b, h.is_h, h.is_t, h.os_b, h.os_h, h.os_t};
  for (const int64_t v : s)
    if (v % vec) return false;
  return h.count == 0 || (aligned_to(in, (size_t)vec * es) && aligned_to(out, (size_t)vec * es));
}

}  // namespace
}  // namespace hk

using namespace hk;

extern "C" {

int hk_rope_axes(void* q_out, const void* q_in, void* k_out, const void* k_in, const void* cos, const void* sin,
                 const void* positions, const hk_rope_axes_shape* shape, hk_stream_t stream) {
  HK_REQUIRE(shape != nullptr, "null pointer argument");
  const int64_t B = shape->B, T = shape->T, D = shape->D, Hq = shape->Hq, Hk = shape->Hk;
  const int64_t table_rows = shape->table_rows, table_ld = shape->table_ld;
  const int64_t* sections = shape->sections;
  const int axes = shape->axes, dtype_x = shape->dtype_x, dtype_cs = shape->dtype_cs, pos_type = shape->pos_type;
  HK_REQUIRE(B >= 0 && T >= 0 && Hq >= 0 && Hk >= 0 && D > 0, "invalid shape B=%lld T=%lld Hq=%lld Hk=%lld D=%lld",
             (long long)B, (long long)T, (long long)Hq, (long long)Hk, (long long)D);
  HK_REQUIRE(D % 2 == 0, "head_dim D=%lld must be even", (long long)D);
  HK_REQUIRE(dtype_cs == kF32 || dtype_cs == kF16 || dtype_cs == kBF16, "invalid cos/sin dtype %d", dtype_cs);
  HK_REQUIRE(dtype_x == kF32 || dtype_x == kF16 || dtype_x == kBF16, "invalid dtype code %d", dtype_x);
  HK_REQUIRE(pos_type == HK_I32 || pos_type == HK_I64, "positions must be int32 or int64, got code %d", pos_type);
  HK_REQUIRE(axes >= 1 && axes <= kMaxAxes, "1..%d position axes, got %d", kMaxAxes, axes);
  const int64_t half = D / 2;
  RopeAxesArgs g = {};
  int64_t sum = 0;
  for (int a = 0; a < axes; ++a) HK_REQUIRE(sections[a] >= 0, "sections must not be negative");
  for (int a = 0; a < axes; ++a) {
    HK_REQUIRE(sections[a] <= half, "section %d has %lld pairs of D/2 = %lld", a, (long long)sections[a], (long long)half);
    sum += sections[a];
    g.axes.n[a] = (int)(shape->interleaved ? sections[a] : sum);
  }
  HK_REQUIRE(sum == half, "sections sum to %lld, need D/2 = %lld", (long long)sum, (long long)half);
  if (shape->interleaved) {
    // axis a > 0 owns pairs a, a + A, ..., a + A (n_a - 1); all of them must exist
    for (int a = 1; a < axes; ++a)
      HK_REQUIRE(sections[a] == 0 || a + axes * (sections[a] - 1) < half,
                 "interleaved section %d of %lld pairs does not fit D/2 = %lld", a, (long long)sections[a],
                 (long long)half);
  }
  g.axes.count = axes;
  g.axes.interleaved = shape->interleaved ? 1 : 0;
  const int64_t* const strides[] = {shape->q_in, shape->q_out, shape->k_in, shape->k_out, shape->pos};
  for (const int64_t* v : strides)
    HK_REQUIRE(v[0] >= 0 && v[1] >= 0 && v[2] >= 0, "negative strides are not supported");
  HK_REQUIRE(table_rows >= 0 && table_ld >= half, "cos/sin row stride %lld smaller than D/2 = %lld",
             (long long)table_ld, (long long)half);
  HK_REQUIRE(B == 0 || T <= ((1LL << 31) - 1) / B, "B * T = %lld * %lld too large", (long long)B, (long long)T);
  HK_REQUIRE(Hq + Hk < (1 << 20) && D <= (1 << 20), "too many heads or too long a head");
  if (B == 0 || T == 0 || Hq + Hk == 0) return HK_OK;
  HK_REQUIRE((Hq == 0 || (q_out && q_in)) && (Hk == 0 || (k_out && k_in)) && cos && sin && positions,
             "null pointer argument");
  auto heads = [](int64_t n, const int64_t* in, const int64_t* out) {
    return Heads{(int)n, in[0], in[1], in[2], out[0], out[1], out[2]};
  };
  g.q = heads(Hq, shape->q_in, shape->q_out);
  g.k = heads(Hk, shape->k_in, shape->k_out);
  g.positions = positions;
  g.ps_a = shape->pos[0];
  g.ps_b = shape->pos[1];
  g.ps_t = shape->pos[2];
  g.table_rows = table_rows;
  g.table_ld = table_ld;
  g.T = (uint32_t)T;
  g.half = (uint32_t)half;
  g.tokens = B * T;
  g.sgn = shape->inverse ? -1.f : 1.f;
  // the storage order of the larger tensor decides how lanes walk memory
  const Heads& lead = Hq >= Hk ? g.q : g.k;
  const bool head_major = T > 1 && lead.is_t < lead.is_h;
  const hipStream_t st = (hipStream_t)stream;

  return dispatch_t(dtype_x, [&](auto tx) {
    using TX = typename decltype(tx)::type;
    return dispatch_t(dtype_cs, [&](auto tc) {
      using TC = typename decltype(tc)::type;
      auto launch = [&](auto vec_c) {
        constexpr int VEC = decltype(vec_c)::value;
        g.chunks = (uint32_t)(half / VEC);
        g.lanes = std::min<uint32_t>(g.chunks, kThreads);
        const uint32_t per_block = kThreads / g.lanes;
        const int64_t heads = Hq + Hk;
        // Tokens a block. Eight slots (a lane walks heads / 8 heads with one set of angles) once that leaves about
        // four blocks a CU; fewer tokens and more slots before that, so that a few tokens still spread over the GPU
        // (64 tokens x 40 heads: one block a token). 8 slots of 8 lanes: 31.4 us for q and k of 8192 tokens x 40
        // heads x 128 bf16 (4 slots 34, 20 slots 33 and more; a copy of the same bytes 30.2).
        uint32_t tb = (uint32_t)std::max<int64_t>(1, per_block / heads);
        while (tb * 16 <= per_block && g.tokens >= (int64_t)tb * 2048) tb *= 2;
        g.tokens_block = tb;
        g.slots = (uint32_t)std::min<int64_t>(heads, per_block / tb);
        const int64_t blocks = cdiv(g.tokens, (int64_t)tb);
        HK_REQUIRE(blocks < (1LL << 32) / kThreads, "B * T = %lld too many for one launch", (long long)g.tokens);
        const dim3 grid((unsigned)blocks, (unsigned)cdiv((int64_t)g.chunks, (int64_t)g.lanes));
        auto go = [&](auto tp, auto order) {
          using TP = typename decltype(tp)::type;
          constexpr bool HM = decltype(order)::value;
          hipLaunchKernelGGL((rope_axes_kernel<TX, TC, TP, VEC, HM, 2>), grid, dim3(kThreads), 0, st, (TX*)q_out,
                             (const TX*)q_in, (TX*)k_out, (const TX*)k_in, (const TC*)cos, (const TC*)sin, g);
          return check_launch("rope_axes_kernel");
        };
        if (pos_type == HK_I64)
          return head_major ? go(Tag<int64_t>{}, std::true_type{}) : go(Tag<int64_t>{}, std::false_type{});
        return head_major ? go(Tag<int32_t>{}, std::true_type{}) : go(Tag<int32_t>{}, std::false_type{});
      };
      constexpr int V = 16 / sizeof(TX);
      const bool whole = half % V == 0 && heads_ok(g.q, q_in, q_out, V, sizeof(TX)) &&
                         heads_ok(g.k, k_in, k_out, V, sizeof(TX));
      if (whole) return launch(std::integral_constant<int, V>{});
      const bool halves = half % (V / 2) == 0 && heads_ok(g.q, q_in, q_out, V / 2, sizeof(TX)) &&
                          heads_ok(g.k, k_in, k_out, V / 2, sizeof(TX));
      if (halves) return launch(std::integral_constant<int, V / 2>{});  // (D = 72 in 16 bits)
      return launch(std::integral_constant<int, 1>{});
    });
  });
}

}  // extern "C"
