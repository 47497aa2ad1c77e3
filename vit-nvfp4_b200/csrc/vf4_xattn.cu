// Cross attention: queries of one length over keys and values of another (an encoder's states), with
// shared key / value heads, a key count per image and a mask of keys.
//
//   out[b, h, i] = sum_j p_j v[b, h / G, j] / sum_j p_j,   p_j = exp(scale q[b, h, i] . k[b, h / G, j])
//
// over the keys j that image b keeps (j < kv_lens[b] and key_mask[b, j]); a row that keeps none is 0.
// Masked keys and values are never used, whatever they hold (NaN and infinities included).  No
// counterpart in the reference, whose attention is self attention of a ViT (nvfp4/attention.py:53-86).
//
// The G query heads that share a key / value head and their Sq queries are the rows of one problem:
// R = G * Sq rows against the same keys, so a decoder's single token still reads each key once.
//
//   xattn_tc_kernel    tcgen05: 128-row tiles, 128 keys at a time, online softmax
//   xattn_rows_kernel  up to 4 rows over short keys (plain_rows), plain FMAs: the keys stream through registers
//
// With fewer tiles than SMs the keys are cut into chunks: each CTA leaves its rows' maxima, sums and
// unnormalised outputs in the workspace and xattn_join_kernel adds them up in order.
#include <string.h>

#include "vf4_common.cuh"
#include "vf4_host.h"

namespace vf4 {

static __device__ int g_xattn_err;

int xattn_device_error(int clear) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_xattn_err, sizeof(int));
  if (clear) {
    int z = 0;
    cudaMemcpyToSymbol(g_xattn_err, &z, sizeof(int));
  }
  return v;
}

struct XParams {
  const __nv_bfloat16 *q, *k, *v;
  int64_t qb, qh, qs, kb, kh, ks, vb, vh, vs;   // element strides
  __nv_bfloat16* out;
  int64_t ob, oh, os;
  const int32_t* lens;     // (B,) or NULL
  const uint8_t* mask;     // (B, Skv) bytes, non-zero = keep, or NULL; rows mask_b apart
  int64_t mask_b;
  int B, Hkv, G, Sq, Skv, D;
  int R;                   // G * Sq
  int negate;              // scale < 0: the queries are negated and c is its magnitude
  float c;                 // |scale| * log2(e)
  int chunk, chunks;       // keys per CTA and CTAs per row tile; chunks > 1: partial results to the workspace
  float* part_o;           // [B * Hkv][chunks][R][D]
  float2* part_ml;         // [B * Hkv][chunks][R]: {maximum of the scores, sum of the weights}; {-inf, 0}: no key kept,
                           // {-inf, 1}: keys kept, every score -inf
  int tiles;               // 128-row tiles (tcgen05 kernel)
};

VF4_DEV int keys_of(const XParams& p, int b) {
  return p.lens ? max(0, min(p.lens[b], p.Skv)) : p.Skv;
}

// Row r of head group hk: query element pointer offsets.
VF4_DEV int64_t q_offset(const XParams& p, int b, int hk, int r) {
  const int g = r / p.Sq, i = r - g * p.Sq;
  return b * p.qb + (int64_t)(hk * p.G + g) * p.qh + i * p.qs;
}
VF4_DEV int64_t o_offset(const XParams& p, int b, int hk, int r) {
  const int g = r / p.Sq, i = r - g * p.Sq;
  return b * p.ob + (int64_t)(hk * p.G + g) * p.oh + i * p.os;
}

// ---------------------------------------------------------------------------------------
// Up to 4 rows.  LPK lanes hold one key's D <= 8 LPK elements (16 bytes each), so a warp reads 32 / LPK keys
// per load; every group of lanes keeps its own maximum, sum and output for the keys it sees, kU of them at a
// time (all their loads in flight together), and the groups are joined at the end: lanes by shuffles, warps
// through shared memory.  Bound by memory latency first, which the SM's other CTAs hide (1024 problems of 257
// keys: 4.2 TB/s); a few problems get eight warps each, which take an image's 257 tokens of 64 elements in one
// batch (kU = 9: 36 keys per warp).
// ---------------------------------------------------------------------------------------
constexpr int kRowWarps = 8;   // at most

template <int LPK, int R>
__global__ void __launch_bounds__(kRowWarps * 32) xattn_rows_kernel(const XParams p) {
  constexpr int KPW = 32 / LPK, kU = R <= 2 ? 9 : 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = lane / LPK, el = (lane % LPK) * 8;     // key group and first element of this lane
  const int chunk = blockIdx.x % p.chunks, item = blockIdx.x / p.chunks;
  const int b = item / p.Hkv, hk = item - b * p.Hkv;
  const bool on = el < p.D;
  const int k0 = chunk * p.chunk, k1 = min(keys_of(p, b), k0 + p.chunk);
  // this warp's share of the keys
  const int warps = blockDim.x >> 5, share = ((k1 - k0 + warps - 1) / warps + KPW - 1) / KPW * KPW;
  const int w0 = k0 + warp * share, w1 = min(k1, w0 + share);

  float q[R][8], acc[R][8], m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (on && r < p.R) w = __ldg(reinterpret_cast<const uint4*>(p.q + q_offset(p, b, hk, r) + el));
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    const float f = p.negate ? -p.c : p.c;   // scores come out in units of log2
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      q[r][i] = __uint_as_float((i & 1) ? (u[i / 2] & 0xFFFF0000u) : (u[i / 2] << 16)) * f;
      acc[r][i] = 0.f;
    }
  }
  const __nv_bfloat16* kp = p.k + b * p.kb + hk * p.kh + el;
  const __nv_bfloat16* vp = p.v + b * p.vb + hk * p.vh + el;
  const uint8_t* mp = p.mask ? p.mask + b * p.mask_b : nullptr;
  bool some = false;   // any key kept
  for (int base = w0; base < w1; base += KPW * kU) {
    uint4 kc[kU], vc[kU];
    bool kept[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int j = base + u * KPW + grp;
      kept[u] = j < w1 && (!mp || mp[j] != 0);
      some = some || kept[u];
      kc[u] = vc[u] = make_uint4(0, 0, 0, 0);
      if (kept[u] && on) {
        kc[u] = __ldg(reinterpret_cast<const uint4*>(kp + (int64_t)j * p.ks));
        vc[u] = __ldg(reinterpret_cast<const uint4*>(vp + (int64_t)j * p.vs));
      }
    }
    float s[kU][R];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const uint32_t w[4] = {kc[u].x, kc[u].y, kc[u].z, kc[u].w};
#pragma unroll
      for (int r = 0; r < R; ++r) s[u][r] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = __uint_as_float((i & 1) ? (w[i / 2] & 0xFFFF0000u) : (w[i / 2] << 16));
#pragma unroll
        for (int r = 0; r < R; ++r) s[u][r] = fmaf(q[r][i], x, s[u][r]);
      }
    }
#pragma unroll
    for (int o = 1; o < LPK; o <<= 1)
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) s[u][r] += __shfl_xor_sync(0xFFFFFFFFu, s[u][r], o);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float mx = m[r];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (!kept[u]) s[u][r] = -INFINITY;
        mx = fmaxf(mx, s[u][r]);
      }
      const float ms = mx == -INFINITY ? 0.f : mx;   // nothing kept so far: weights 2^-inf = 0
      const float f = ex2_approx(m[r] - ms);
      m[r] = mx;
      l[r] *= f;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[r][i] *= f;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        s[u][r] = ex2_approx(s[u][r] - ms);
        l[r] += s[u][r];
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const uint32_t w[4] = {vc[u].x, vc[u].y, vc[u].z, vc[u].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = __uint_as_float((i & 1) ? (w[i / 2] & 0xFFFF0000u) : (w[i / 2] << 16));
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][i] = fmaf(s[u][r], x, acc[r][i]);
      }
    }
  }
  // join the key groups of the warp, then the warps
  __shared__ float red_o[kRowWarps][R][LPK * 8];
  __shared__ float2 red_ml[kRowWarps][R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int o = LPK; o < 32; o <<= 1) {
      const float m2 = __shfl_xor_sync(0xFFFFFFFFu, m[r], o), l2 = __shfl_xor_sync(0xFFFFFFFFu, l[r], o);
      const float mx = fmaxf(m[r], m2), ms = mx == -INFINITY ? 0.f : mx;
      const float f1 = ex2_approx(m[r] - ms), f2 = ex2_approx(m2 - ms);
      // the same order of the two summands in both lanes, so that they agree to the last bit
      l[r] = (lane & o) ? fmaf(l2, f2, l[r] * f1) : fmaf(l[r], f1, l2 * f2);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a2 = __shfl_xor_sync(0xFFFFFFFFu, acc[r][i], o);
        acc[r][i] = (lane & o) ? fmaf(a2, f2, acc[r][i] * f1) : fmaf(acc[r][i], f1, a2 * f2);
      }
      m[r] = mx;
    }
    if (grp == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) red_o[warp][r][el + i] = acc[r][i];
      if (lane == 0) red_ml[warp][r] = make_float2(m[r], l[r]);
    }
  }
  const bool seen = __syncthreads_or(some);
  for (int t = threadIdx.x; t < R * LPK; t += blockDim.x) {
    const int r = t / LPK, e = (t - r * LPK) * 8;
    if (r >= p.R || e >= p.D) continue;
    float mx = -INFINITY, ls = 0.f, o[8];
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w)
      if (w < warps) mx = fmaxf(mx, red_ml[w][r].x);
    const float ms = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      if (w >= warps) break;
      const float f = ex2_approx(red_ml[w][r].x - ms);
      ls = fmaf(red_ml[w][r].y, f, ls);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = fmaf(red_o[w][r][e + i], f, o[i]);
    }
    if (seen && ls == 0.f) ls = p.chunks > 1 ? 1.f : __uint_as_float(0x7FFFFFFFu);   // every kept score is -inf
    if (p.chunks > 1) {
      const int64_t row = ((int64_t)item * p.chunks + chunk) * p.R + r;
      float4* dst = reinterpret_cast<float4*>(p.part_o + row * p.D + e);
      dst[0] = make_float4(o[0], o[1], o[2], o[3]);
      dst[1] = make_float4(o[4], o[5], o[6], o[7]);
      if (e == 0) p.part_ml[row] = make_float2(mx, ls);
    } else {
      const float f = ls > 0.f ? __fdividef(1.f, ls) : (ls == 0.f ? 0.f : ls);   // nothing kept: 0; NaN stays
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = bf16x2_round(f32x2_pack(o[2 * i] * f, o[2 * i + 1] * f));
      *reinterpret_cast<uint4*>(p.out + o_offset(p, b, hk, r) + e) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// per_row warps per row (1, 2, 4 or 8 of the CTA's 8; by the number of chunks): warp w of them joins chunks w,
// w + per_row, .., then the warps are joined, all in a fixed order.  Maxima are in units of log2.  Started while the
// chunks' kernel ends.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(kJoinWarps * 32) xattn_join_kernel(const XParams p, const int per_row) {
  __shared__ float4 red_o[kJoinWarps][32];
  __shared__ float red_l[kJoinWarps];
  griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp & (per_row - 1);
  const int64_t rows = (int64_t)p.B * p.Hkv * p.R, own = blockIdx.x * (int64_t)(kJoinWarps / per_row) + warp / per_row;
  const int64_t row = own < rows ? own : rows - 1;   // past the last row: the last one, without storing it
  const int item = (int)(row / p.R), r = (int)(row - (int64_t)item * p.R);
  const int b = item / p.Hkv, hk = item - b * p.Hkv;
  const int n = min(p.chunks, (keys_of(p, b) + p.chunk - 1) / p.chunk);   // chunks that hold keys
  const int64_t at = (int64_t)item * p.chunks * p.R + r;
  float mx = -INFINITY;
  bool some = false;
  for (int c = lane; c < n; c += 32) {
    const float2 ml = p.part_ml[at + (int64_t)c * p.R];
    mx = fmaxf(mx, ml.x);
    some = some || ml.y != 0.f;
  }
  some = __any_sync(0xFFFFFFFFu, some);
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
  const float ms = mx == -INFINITY ? 0.f : mx;
  const int e = lane * 4;
  float ls = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kU = 4;   // chunks whose loads are in flight together
  for (int c0 = sub; c0 < n; c0 += per_row * kU) {
    float2 ml[kU];
    float4 o[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int c = c0 + u * per_row;
      ml[u] = make_float2(-INFINITY, 0.f);
      o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c < n) {
        ml[u] = p.part_ml[at + (int64_t)c * p.R];
        if (e < p.D) o[u] = *reinterpret_cast<const float4*>(p.part_o + (at + (int64_t)c * p.R) * p.D + e);
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (ml[u].x == -INFINITY && ml[u].y == 0.f) continue;   // a chunk without kept keys
      const float f = ex2_approx(ml[u].x - ms);
      ls = fmaf(ml[u].y, f, ls);
      acc.x = fmaf(o[u].x, f, acc.x);
      acc.y = fmaf(o[u].y, f, acc.y);
      acc.z = fmaf(o[u].z, f, acc.z);
      acc.w = fmaf(o[u].w, f, acc.w);
    }
  }
  red_o[warp][lane] = acc;
  if (lane == 0) red_l[warp] = ls;
  __syncthreads();
  if (sub == 0 && own < rows && e < p.D) {
    for (int w = warp + 1; w < warp + per_row; ++w) {
      const float4 o = red_o[w][lane];
      acc.x += o.x;
      acc.y += o.y;
      acc.z += o.z;
      acc.w += o.w;
      ls += red_l[w];
    }
    if (some && mx == -INFINITY) ls = __uint_as_float(0x7FFFFFFFu);   // keys kept, every score -inf
    const float f = ls > 0.f ? __fdividef(1.f, ls) : (ls == 0.f ? 0.f : ls);
    *reinterpret_cast<uint2*>(p.out + o_offset(p, b, hk, r) + e) =
        make_uint2(bf16x2_round(f32x2_pack(acc.x * f, acc.y * f)), bf16x2_round(f32x2_pack(acc.z * f, acc.w * f)));
  }
}

// ---------------------------------------------------------------------------------------
// Many rows or many keys: tcgen05.  A CTA takes 128 rows and runs over its keys in tiles of 128:
//   S = Q K^T (128 x 128, fp32, tensor memory) -> softmax warps: maximum, P = 2^(c s - c m) in bf16, back to
//   tensor memory -> O += P V (accumulated in tensor memory)
// Two CTAs share an SM (half of its shared and tensor memory each), so that one's softmax runs while the
// tensor core works for the other, and one's first and last steps hide behind the other's middle ones.
// Up to 64 elements per head P has columns of its own, and the next tile's S is computed while this one's P
// is; beyond, P takes S's place and the next S follows O += P V.
//
// The running maximum m is only moved (and O and the sums rescaled) when it grows by more than 2^8: P stays
// below 256, which bf16 and the fp32 sums hold as well as P <= 1.  P is rounded to bf16 (half a step, 2^-9 to
// 2^-8 of each weight): the second product's operands are of one type, and in 32 bits V would have to be
// converted and the product run at half the rate.  The sums take P unrounded.  The relative error against 64 bits
// is 0.0023, with the fp32 weights of the kernel above 0.0017, which the output's own rounding makes.
//
//   warp 0      TMA of K and V tiles (128-byte swizzle, panels of 64 elements)
//   warp 1      TMEM allocation, MMAs
//   warps 2, 3  masks (with a mask or key counts): clear the dropped rows of each K and V tile in shared memory, so
//               that none of their NaNs reaches a score or meets a weight of 0, and set the tile's extra column:
//               S gets one more step of its product, with 1 in every query's column and 0 or -inf in each
//               key's, so a dropped key's score is -inf without a thread of the softmax looking at the mask
//               (which took it as long as its maximum).  Whether any key at all is kept they tell the softmax warps
//               after the last tile: a NaN in the query makes dropped scores NaN, and without a kept key that row is 0
//   warps 4-7   softmax, a thread per row, which holds the row's 128 scores in registers
//
// Bound by the exponentials: 16 per clock and SM on the special-function unit is 1024 clocks per 128 x 128
// scores (the products take 512 at 64 elements per head), so one in kPolyEvery pairs is computed by a polynomial
// on the FMA pipes instead.
// ---------------------------------------------------------------------------------------
template <int DP>
struct XCfg {
  static constexpr int PANELS = DP / 64, PANEL = 128 * 128;    // bytes of 128 rows x 64 elements
  static constexpr int TILE = PANELS * PANEL;
  static constexpr int NK = DP == 64 ? 2 : 1, NV = NK;         // tiles in flight of K and of V
  static constexpr bool kOwnP = DP == 64;
  static constexpr uint32_t P_COL = kOwnP ? 128 : 0, O_COL = kOwnP ? 192 : 128;
  static constexpr int EXT = 128 * 32;                         // the extra step: 128 rows x 16 elements, not swizzled
  static constexpr int V_OFF = 0, K_OFF = NV * TILE, Q_OFF = (NV + NK) * TILE;
  static constexpr int QX_OFF = Q_OFF + TILE, KX_OFF = QX_OFF + EXT;
  static constexpr int BAR_OFF = KX_OFF + NK * EXT;
  static constexpr int NBAR = 3 * (NK + NV) + 8;
  static constexpr int SMEM = 1024 + BAR_OFF + 8 * NBAR + 16;   // behind the barriers: tensor memory address, `seen`
  // 4 x 16 heads of 1024 x 4096 x 128: 146 us with 3, 152 with 4, 157 with 2; 32 x 16 of 64 x 1025 x 80: 36.4, 38.2 and
  // 36.9; 8 x 16 of 1024 x 4096 x 64: 197 with 4, 200 with 3, 205 without the polynomial
  static constexpr int kPolyEvery = DP == 64 ? 4 : 3;
  static constexpr int THREADS = 256;
  static constexpr int kLaunchRegs = 128, kControlRegs = 40, kSoftRegs = 216;
  static_assert(128 * kControlRegs + 128 * kSoftRegs <= THREADS * kLaunchRegs, "register split");
  static_assert(SMEM <= 113 * 1024, "two CTAs share an SM");
};

VF4_DEV void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// max(a, b, c), NaN if any is: a NaN score has to reach its row's maximum, whose whole row it makes NaN
VF4_DEV float max3nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x of a pair on the FMA pipes: x = j + f with j the nearest integer (by adding 1.5 * 2^23) and |f| <= 1/2,
// 2^f by the degree-4 polynomial of least relative error (2.6e-6, fitted on that interval), j added to the
// exponent.  x below -126 counts as -126; a NaN's row is NaN already through its maximum.
VF4_DEV unsigned long long ex2_poly_x2(unsigned long long x) {
  float x0, x1;
  f32x2_unpack(x, &x0, &x1);
  const unsigned long long v = f32x2_pack(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
  const unsigned long long big = f32x2_pack(12582912.f, 12582912.f), nbig = f32x2_pack(-12582912.f, -12582912.f);
  const unsigned long long t = add_f32x2(v, big), j = add_f32x2(t, nbig);
  const unsigned long long f = fma_f32x2(j, f32x2_pack(-1.f, -1.f), v);
  unsigned long long y = fma_f32x2(f, f32x2_pack(0.0095701f, 0.0095701f), f32x2_pack(0.05591786f, 0.05591786f));
  y = fma_f32x2(y, f, f32x2_pack(0.24024745f, 0.24024745f));
  y = fma_f32x2(y, f, f32x2_pack(0.69312181f, 0.69312181f));
  y = fma_f32x2(y, f, f32x2_pack(0.99999926f, 0.99999926f));
  float y0, y1, t0, t1;
  f32x2_unpack(y, &y0, &y1);
  f32x2_unpack(t, &t0, &t1);
  return f32x2_pack(__uint_as_float(__float_as_uint(y0) + (__float_as_uint(t0) << 23)),
                    __uint_as_float(__float_as_uint(y1) + (__float_as_uint(t1) << 23)));
}


template <int DP>
__global__ void __launch_bounds__(XCfg<DP>::THREADS, 2)
    xattn_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const int k_bm,
                    const int k_hm, const int v_bm, const int v_hm, const XParams p) {
  using C = XCfg<DP>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw0 = smem_u32(smem_raw);
  const uint32_t base = (raw0 + 1023u) & ~1023u;
  uint8_t* gb = smem_raw + (base - raw0);
  const uint32_t bar = base + C::BAR_OFF;
  auto k_full = [&](int i) { return bar + 8u * i; };
  auto k_free = [&](int i) { return bar + 8u * (C::NK + i); };
  auto k_clean = [&](int i) { return bar + 8u * (2 * C::NK + i); };   // dropped rows cleared, extra column set
  auto v_full = [&](int i) { return bar + 8u * (3 * C::NK + i); };
  auto v_free = [&](int i) { return bar + 8u * (3 * C::NK + C::NV + i); };
  auto v_clean = [&](int i) { return bar + 8u * (3 * C::NK + 2 * C::NV + i); };
  const uint32_t q_full = bar + 8u * (3 * (C::NK + C::NV)), s_full = q_full + 8, s_free = q_full + 16, p_full = q_full + 24,
                 o_full = q_full + 32, p_half = q_full + 40, seen_set = q_full + 48,
                 drain = q_full + 56;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gb + C::BAR_OFF + 8 * C::NBAR);
  volatile uint32_t* seen = tmem_slot + 1;   // masked: whether any of this CTA's keys is kept; valid after seen_set
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* err = &g_xattn_err;

  // this CTA's rows and keys
  const int chunk = blockIdx.x % p.chunks, tile = blockIdx.x / p.chunks % p.tiles, item = blockIdx.x / p.chunks / p.tiles;
  const int b = item / p.Hkv, hk = item - b * p.Hkv;
  const int row0 = tile * 128, rows = min(128, p.R - row0);
  const int k0 = chunk * p.chunk, k1 = min(keys_of(p, b), k0 + p.chunk);
  const int n = k1 > k0 ? (k1 - k0 + 127) / 128 : 0;   // key tiles
  const bool masked = p.mask != nullptr || (k1 - k0) % 128 != 0;

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < C::NK; ++i) {
      mbar_init(k_full(i), 1);
      mbar_init(k_free(i), 1);
      mbar_init(k_clean(i), 1);
    }
    for (int i = 0; i < C::NV; ++i) {
      mbar_init(v_full(i), 1);
      mbar_init(v_free(i), 1);
      mbar_init(v_clean(i), 1);
    }
    mbar_init(q_full, 128);
    mbar_init(s_full, 1);
    mbar_init(s_free, 4);
    mbar_init(p_full, 4);
    mbar_init(p_half, 4);
    mbar_init(o_full, 1);
    mbar_init(seen_set, 1);
    mbar_init(drain, 1);
    fence_mbar_init();
    tma_prefetch(&tmK);
    tma_prefetch(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 256);
    tmem_relinquish();
  }
  fence_async_shared();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kControlRegs));
    const bool elected = elect_one();
    if (warp == 0) {
      // in the order of use: K0 (K1, K2), V0, K next, V1, ...; with one place for K its next tile follows V
      auto load = [&](const CUtensorMap* m, uint32_t dst, uint32_t full, uint32_t free_, int use, int t, int hm, int bm) {
        if (!__all_sync(0xFFFFFFFFu, use == 0 || mbar_wait(free_, (uint32_t)(use - 1) & 1u, err, kDevErrTimeoutEmpty)))
          return false;
        if (elected) {
          mbar_arrive_expect_tx(full, C::TILE);
#pragma unroll
          for (int c = 0; c < C::PANELS; ++c)
            tma_load_4d(dst + c * C::PANEL, m, c * 64, k0 + t * 128, hk * hm, b * bm, full);
        }
        __syncwarp();
        return true;
      };
      auto load_k = [&](int t) {
        const int i = t % C::NK;
        return load(&tmK, base + C::K_OFF + i * C::TILE, k_full(i), k_free(i), t / C::NK, t, k_hm, k_bm);
      };
      auto load_v = [&](int t) {
        const int i = t % C::NV;
        return load(&tmV, base + C::V_OFF + i * C::TILE, v_full(i), v_free(i), t / C::NV, t, v_hm, v_bm);
      };
      bool ok = true;
      int kt = 0, vt = 0;   // tiles whose copies have been issued
      while (kt < n && kt < C::NK && (ok = load_k(kt))) ++kt;
      while (vt < n && ok) {
        ok = load_v(vt);
        if (!ok) break;
        ++vt;
        if (kt < n && (ok = load_k(kt))) ++kt;   // K of tile vt - 1 + NK, free once the scores of tile vt - 1 are there
      }
      // no copy may still be writing shared memory when the CTA exits, also after a wait that gave up
      for (int t = max(0, kt - C::NK); t < kt; ++t)
        mbar_wait(k_full(t % C::NK), (uint32_t)(t / C::NK) & 1u, err, kDevErrTimeoutFull);
      for (int t = max(0, vt - C::NV); t < vt; ++t)
        mbar_wait(v_full(t % C::NV), (uint32_t)(t / C::NV) & 1u, err, kDevErrTimeoutFull);
    } else if (warp == 1) {
      const int kd = (p.D + 15) / 16;
      const uint32_t id_s = idesc_bf16(128, false), id_o = idesc_bf16((uint32_t)kd * 16u, true);
      const uint64_t qd = smem_desc(base + C::Q_OFF, 16, 1024, 2), kd0 = smem_desc(base + C::K_OFF, 16, 1024, 2);
      const uint64_t vd0 = smem_desc(base + C::V_OFF, C::PANEL, 1024, 2);
      // not swizzled: 8 rows x 16 bytes per core matrix, the step's two of them 128 bytes apart, 8-row groups 256
      const uint64_t qx = smem_desc(base + C::QX_OFF, 128, 256, 0), kx0 = smem_desc(base + C::KX_OFF, 128, 256, 0);
      bool ok = n == 0 || __all_sync(0xFFFFFFFFu, mbar_wait(q_full, 0, err, kDevErrTimeoutFull));
      auto score = [&](int t) {   // S of tile t
        const int st = t % C::NK;
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(masked ? k_clean(st) : k_full(st), (uint32_t)(t / C::NK) & 1u, err, kDevErrTimeoutFull));
        if (!ok) return;
        tc_fence_after();
        if (elected) {
          const uint64_t kk0 = kd0 + (uint32_t)(st * (C::TILE >> 4));
          for (int kk = 0; kk < kd; ++kk) {
            const uint32_t off = (uint32_t)((kk >> 2) * (C::PANEL >> 4) + (kk & 3) * 2);
            mma_f16(tmem, qd + off, kk0 + off, id_s, kk > 0 ? 1u : 0u);
          }
          if (masked) mma_f16(tmem, qx, kx0 + (uint32_t)(st * (C::EXT >> 4)), id_s, 1u);
          tc_commit(s_full);
          tc_commit(k_free(st));
        }
        __syncwarp();
      };
      if (ok && n > 0) score(0);
      for (int t = 0; t < n && ok; ++t) {
        const int st = t % C::NV;
        if (C::kOwnP && t + 1 < n) {   // S may be overwritten once the softmax warps hold it
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(s_free, (uint32_t)t & 1u, err, kDevErrTimeoutTmem));
          if (ok) score(t + 1);
          if (!ok) break;
        }
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(masked ? v_clean(st) : v_full(st), (uint32_t)(t / C::NV) & 1u, err, kDevErrTimeoutFull) &&
                                         mbar_wait(p_half, (uint32_t)t & 1u, err, kDevErrTimeoutTmem));
        if (!ok) break;
        tc_fence_after();
        const uint64_t vd = vd0 + (uint32_t)(st * (C::TILE >> 4));
        if (elected) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f16_tmem_a(tmem + C::O_COL, tmem + C::P_COL + 8u * kk, vd + (uint32_t)(kk * (2048 >> 4)), id_o,
                           (t > 0 || kk > 0) ? 1u : 0u);
        }
        __syncwarp();
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(p_full, (uint32_t)t & 1u, err, kDevErrTimeoutTmem));
        if (!ok) break;
        tc_fence_after();
        if (elected) {
#pragma unroll
          for (int kk = 4; kk < 8; ++kk)
            mma_f16_tmem_a(tmem + C::O_COL, tmem + C::P_COL + 8u * kk, vd + (uint32_t)(kk * (2048 >> 4)), id_o, 1u);
          tc_commit(o_full);
          tc_commit(v_free(st));
        }
        __syncwarp();
        if (!C::kOwnP && t + 1 < n) score(t + 1);
      }
      // the tensor core must be done with shared and tensor memory before the CTA exits, also after a wait that gave up
      if (elected) tc_commit(drain);
      __syncwarp();
      mbar_wait(drain, 0, err, kDevErrTimeoutDrain);
    } else if (masked) {
      const bool is_k = warp == 2;   // warp 2: K and its extra column, warp 3: V
      const uint8_t* mp = p.mask ? p.mask + b * p.mask_b : nullptr;
      bool next[4];
      auto kept = [&](int t) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int j = k0 + t * 128 + 32 * w + lane;
          next[w] = j < k1 && (!mp || mp[j] != 0);
        }
      };
      if (is_k)   // the extra step's other columns are 0: the second core matrix of every 8-row group
        for (int i = lane; i < C::NK * 128; i += 32)
          *reinterpret_cast<uint4*>(gb + C::KX_OFF + (i >> 3) * 256 + 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
      kept(0);
      bool some = false;
      for (int t = 0; t < n; ++t) {
        const int use = is_k ? t / C::NK : t / C::NV, st = is_k ? t % C::NK : t % C::NV;
        bool keep[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          keep[w] = next[w];
          some = some || keep[w];
        }
        if (t + 1 < n) kept(t + 1);
        // a tile's arrival also says that the one before it in this place is done with
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(is_k ? k_full(st) : v_full(st), (uint32_t)use & 1u, err, kDevErrTimeoutFull))) break;
        uint8_t* at = gb + (is_k ? C::K_OFF : C::V_OFF) + st * C::TILE;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int j = 32 * w + lane;
          if (is_k)   // 0xFF80: -inf in bf16
            *reinterpret_cast<uint4*>(gb + C::KX_OFF + st * C::EXT + (j >> 3) * 256 + (j & 7) * 16) =
                make_uint4(keep[w] ? 0u : 0xFF80u, 0, 0, 0);
          if (!keep[w]) {   // the lane clears its own row, starting at a piece of its own: no bank conflicts
#pragma unroll
            for (int c = 0; c < C::PANELS; ++c)
#pragma unroll
              for (int x = 0; x < 8; ++x)
                *reinterpret_cast<uint4*>(at + c * C::PANEL + j * 128 + ((x + lane) & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(is_k ? k_clean(st) : v_clean(st));
      }
      some = __any_sync(0xFFFFFFFFu, some);
      if (is_k && lane == 0) {
        *seen = some;
        mbar_arrive(seen_set);
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftRegs));
    const int r = (warp & 3) * 32 + lane;    // row of the tile
    const uint32_t t_s = tmem + ((uint32_t)((warp & 3) * 32) << 16), t_p = t_s + C::P_COL, t_o = t_s + C::O_COL;
    const int row = row0 + r;
    const bool valid = r < rows, act = (warp & 3) * 32 < rows;   // this row; any row of this warp
    {  // Q: each thread copies its own row (rows past the last, and elements up to a multiple of 16, as zeros)
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (valid ? q_offset(p, b, hk, row) : 0));
      uint8_t* dst = gb + C::Q_OFF + r * 128;
      const uint32_t sign = p.negate ? 0x80008000u : 0u;
      uint4 w[8 * C::PANELS];
#pragma unroll
      for (int j = 0; j < 8 * C::PANELS; ++j) w[j] = valid && j * 8 < p.D ? __ldg(src + j) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 8 * C::PANELS; ++j)
        *reinterpret_cast<uint4*>(dst + (j >> 3) * C::PANEL + (((j & 7) ^ (r & 7)) << 4)) =
            make_uint4(w[j].x ^ sign, w[j].y ^ sign, w[j].z ^ sign, w[j].w ^ sign);
      if (masked) {   // the extra step: 1 in the first column
        uint8_t* x = gb + C::QX_OFF + (r >> 3) * 256 + (r & 7) * 16;
        *reinterpret_cast<uint4*>(x) = make_uint4(0x3F80u, 0, 0, 0);
        *reinterpret_cast<uint4*>(x + 128) = make_uint4(0, 0, 0, 0);
      }
      fence_async_shared();
      mbar_arrive(q_full);
    }
    float m = -INFINITY, l = 0.f;
    const float grow = fminf(8.f / p.c, 3.4e38f);   // finite: -inf + grow stays -inf
    const unsigned long long c2 = f32x2_pack(p.c, p.c);
    bool ok = true;
    for (int t = 0; t < n && ok; ++t) {
      ok = __all_sync(0xFFFFFFFFu, mbar_wait(s_full, (uint32_t)t & 1u, err, kDevErrTimeoutTmem));
      if (!ok) break;
      tc_fence_after();
      if (act) {
        uint32_t v[128];
#pragma unroll
        for (int w = 0; w < 4; ++w) tmem_ld_32x32b_x32(t_s + 32 * w, v + 32 * w);
        tmem_wait_ld();
#pragma unroll
        for (int w = 0; w < 8; ++w) reg_fence16(v + 16 * w);
        if (C::kOwnP) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_free);
        }
        float mx[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          mx[w] = max3nan(__uint_as_float(v[32 * w]), __uint_as_float(v[32 * w + 1]), __uint_as_float(v[32 * w + 31]));
#pragma unroll
          for (int e = 2; e < 30; e += 2) mx[w] = max3nan(mx[w], __uint_as_float(v[32 * w + e]), __uint_as_float(v[32 * w + e + 1]));
          mx[w] = max3nan(mx[w], mx[w], __uint_as_float(v[32 * w + 30]));
        }
        const float top = max3nan(max3nan(mx[0], mx[1], mx[2]), mx[3], mx[3]);   // -inf: no key kept so far
        bool ready = t == 0;                 // the product of the tile before is done: O and P's columns are free
        auto finish_previous = [&]() {
          if (ready) return true;
          ready = true;
          const bool done = __all_sync(0xFFFFFFFFu, mbar_wait(o_full, (uint32_t)(t - 1) & 1u, err, kDevErrTimeoutTmem));
          tc_fence_after();
          return done;
        };
        if (t == 0) {
          m = top;
        } else {
          const bool up = !(top <= m + grow);   // also for a NaN, and from -inf
          if (__any_sync(0xFFFFFFFFu, up)) {
            ok = finish_previous();
            if (!ok) break;
            const float f = !up ? 1.f : ex2_approx((m - top) * p.c);   // m = -inf: 0 (nothing was added yet)
            if (up) m = top;
            l *= f;
            for (int c0 = 0; c0 < p.D; c0 += 16) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(t_o + c0, o);
              tmem_wait_ld();
              reg_fence16(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st_32x32b_x16(t_o + c0, o);
            }
          }
        }
        // c s - c m as one FMA is off by the rounding of c m, the same factor for all of the row's weights and its sum:
        // harmless up to 2^24, where it is 2^0.5, but beyond 2^31 it leaves the range of the weights.  There m is
        // taken off first
        float nm = m == -INFINITY ? 0.f : -m * p.c;
        const bool far = fabsf(nm) > 0x1p24f;
        if (__builtin_expect(__any_sync(0xFFFFFFFFu, far), 0)) {
          const float off = far ? m : 0.f;
#pragma unroll
          for (int e = 0; e < 128; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) - off);
          nm = far ? 0.f : nm;
        }
        const unsigned long long nm2 = f32x2_pack(nm, nm);
        unsigned long long l2[2] = {0ull, 0ull};
        // P in place of the scores: pair i of the registers becomes word i
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int e = 32 * h; e < 32 * h + 32; ++e) {
            const unsigned long long x = fma_f32x2(f32x2_pack(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), c2, nm2);
            unsigned long long pr;
            if (e % C::kPolyEvery == C::kPolyEvery - 1) {
              pr = ex2_poly_x2(x);
            } else {
              float x0, x1;
              f32x2_unpack(x, &x0, &x1);
              pr = f32x2_pack(ex2_approx(x0), ex2_approx(x1));
            }
            l2[e & 1] = add_f32x2(l2[e & 1], pr);
            v[e] = bf16x2_round(pr);
          }
          if (h == 0) {
            if (C::kOwnP) ok = finish_previous();
            if (!ok) break;
          }
          tmem_st_32x32b_x16(t_p + 32 * h, v + 32 * h);
          tmem_st_32x32b_x16(t_p + 32 * h + 16, v + 32 * h + 16);
          if (h == 0) {   // the first half of the product starts while the second half of P is computed
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_half);
          }
        }
        if (!ok) break;
        float a0, a1, a2, a3;
        f32x2_unpack(l2[0], &a0, &a1);
        f32x2_unpack(l2[1], &a2, &a3);
        l += (a0 + a1) + (a2 + a3);
        tmem_wait_st();
      } else if (C::kOwnP) {
        if (lane == 0) mbar_arrive(s_free);
        // not ahead of the warps with rows: their P of tile t - 1 must not be counted from this warp's tile t
        ok = t == 0 || __all_sync(0xFFFFFFFFu, mbar_wait(o_full, (uint32_t)(t - 1) & 1u, err, kDevErrTimeoutTmem));
        if (!ok) break;
        if (lane == 0) mbar_arrive(p_half);
      } else {
        if (lane == 0) mbar_arrive(p_half);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    // O is complete when its last product is
    if (n > 0 && ok) ok = __all_sync(0xFFFFFFFFu, mbar_wait(o_full, (uint32_t)(n - 1) & 1u, err, kDevErrTimeoutTmem));
    tc_fence_after();
    if (masked && ok) ok = __all_sync(0xFFFFFFFFu, mbar_wait(seen_set, 0, err, kDevErrTimeoutOther));
    if (n == 0 || (masked && *seen == 0)) {   // no key kept: 0, also where the query's NaNs have reached m, l and O
      m = -INFINITY;
      l = 0.f;
    } else if (l < 0x1p-64f) {   // keys kept, but no score above -inf (the polynomial's weights of 2^-126 are all there is)
      l = p.chunks > 1 && m == -INFINITY ? 1.f : __uint_as_float(0x7FFFFFFFu);
    }
    if (act && ok) {
      const int64_t part_row = ((int64_t)item * p.chunks + chunk) * p.R + row;
      const bool parts = p.chunks > 1;
      const float f = l > 0.f ? __fdividef(1.f, l) : (l == 0.f ? 0.f : l);   // nothing kept: 0; NaN stays
      __nv_bfloat16* dst = p.out + (valid ? o_offset(p, b, hk, row) : 0);
#pragma unroll
      for (int c0 = 0; c0 < DP; c0 += 32) {
        if (c0 >= p.D) break;
        uint32_t o[32];   // columns past D hold products with the tile's zero padding, or nothing
        tmem_ld_32x32b_x32(t_o + c0, o);
        tmem_wait_ld();
        reg_fence16(o);
        reg_fence16(o + 16);
        if (!valid || (parts && n == 0)) continue;   // the join does not read a chunk without keys
#pragma unroll
        for (int c = 0; c < 32; c += 8) {
          if (c0 + c >= p.D) break;
          if (parts) {
            uint4* d = reinterpret_cast<uint4*>(p.part_o + part_row * p.D + c0 + c);
            d[0] = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
            d[1] = make_uint4(o[c + 4], o[c + 5], o[c + 6], o[c + 7]);
          } else {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = l == 0.f ? 0u : bf16x2_round(f32x2_pack(__uint_as_float(o[c + 2 * e]) * f, __uint_as_float(o[c + 2 * e + 1]) * f));
            *reinterpret_cast<uint4*>(dst + c0 + c) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (valid && parts) p.part_ml[part_row] = make_float2(m == -INFINITY ? m : m * p.c, l);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 256);
}

// K or V as (elements, keys, heads, images); a dimension of stride 0 (or of one entry) is given extent 1 and its
// coordinate multiplied by 0.
static int make_kv_map(CUtensorMap* m, const void* ptr, const XParams& p, int64_t sb, int64_t sh, int64_t ss, int* bm, int* hm) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return fail(VF4_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  *bm = p.B > 1 && sb != 0;
  *hm = p.Hkv > 1 && sh != 0;
  const bool one_key = p.Skv == 1;
  cuuint64_t dims[4] = {(cuuint64_t)p.D, (cuuint64_t)p.Skv, (cuuint64_t)(*hm ? p.Hkv : 1), (cuuint64_t)(*bm ? p.B : 1)};
  cuuint64_t strides[3] = {(cuuint64_t)(one_key ? 16 : ss * 2), (cuuint64_t)(*hm ? sh * 2 : 16), (cuuint64_t)(*bm ? sb * 2 : 16)};
  cuuint32_t box[4] = {64u, 128u, 1u, 1u};
  cuuint32_t es[4] = {1u, 1u, 1u, 1u};
  CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims, strides, box, es,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(VF4_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return VF4_OK;
}

// The plain kernel takes up to 4 rows over short keys, where a CTA of the tensor-core kernel would spend most of
// its time starting and ending; its FMAs and shuffles grow with the rows, so the border falls.  Measured (64 x 16
// problems of 64 elements; plain and tcgen05): 1 row over 257 keys 16.6 and 33.8 us, over 4097 163 and 192 (16391
// keys of 128 elements, 32 problems: 80 and 51); 2 rows over 257 24.9 and 33.8, over 577 46.9 and 43.7; 4 rows
// over 65 13.6 and 20.8, over 257 42.8 and 33.8.
static bool plain_rows(int64_t R, int64_t Skv) {
  return R == 1 ? Skv <= 4096 : R == 2 ? Skv <= 512 : R <= 4 && Skv <= 128;
}

// How many keys a CTA takes, and how many CTAs share a row tile (1: no workspace).
static void plan_chunks(int64_t B, int64_t Hkv, int64_t R, int64_t Skv, int sms, int* chunk, int* chunks) {
  const bool plain = plain_rows(R, Skv);
  const int64_t items = B * Hkv * (plain ? 1 : (R + 127) / 128);
  // plain kernel: 4 CTAs per SM, at least 1024 keys each (16 problems of one row over 4000 keys of 64 elements 12.4 us;
  // with 512 9.8, with 2048 18.8; 128 problems 30.2 with each); tcgen05: as many CTAs as are resident at
  // once, at least 512 keys each (16 problems of 64 rows over 1025 keys 11.1 us; with 256 10.3, with 1024 13.2; 32 over
  // 4100 keys of 80 elements 21.0, 21.0 and 22.7).  With key counts that differ, shorter chunks would even the CTAs
  // out, but measured slower: 4 images of up to 16391 keys, 32 heads over 8 of 128 elements: 45 us, 53 with twice as many
  const int64_t want = plain ? (int64_t)sms * 4 : (int64_t)sms * 2, least = plain ? 1024 : 512;
  int64_t n = want / items;
  if (n > (Skv + least - 1) / least) n = (Skv + least - 1) / least;
  if (n < 1) n = 1;
  int64_t c = ((Skv + n - 1) / n + 127) / 128 * 128;
  if (c < 128) c = 128;
  *chunk = (int)c;
  *chunks = (int)((Skv + c - 1) / c);
  if (*chunks < 1) *chunks = 1;
}

template <int DP>
static int launch_tc(const XParams& p, cudaStream_t s) {
  using C = XCfg<DP>;
  CUtensorMap tk, tv;
  int kbm, khm, vbm, vhm;
  if (int st = make_kv_map(&tk, p.k, p, p.kb, p.kh, p.ks, &kbm, &khm)) return st;
  if (int st = make_kv_map(&tv, p.v, p, p.vb, p.vh, p.vs, &vbm, &vhm)) return st;
  auto kern = xattn_tc_kernel<DP>;
  if (int st = smem_optin(kern, C::SMEM)) return st;
  static const int regs = [] {   // the register split of the kernel relies on what its launch allocates
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, xattn_tc_kernel<DP>) == cudaSuccess ? a.numRegs : 0;
  }();
  if (regs != C::kLaunchRegs) return fail(VF4_ERR_UNSUPPORTED, "vf4_cross_attn: built with %d registers", regs);
  const int64_t grid = (int64_t)p.B * p.Hkv * p.tiles * p.chunks;
  if (grid > INT32_MAX) return fail(VF4_ERR_UNSUPPORTED, "vf4_cross_attn: sizes too large");
  kern<<<(unsigned)grid, C::THREADS, C::SMEM, s>>>(tk, tv, kbm, khm, vbm, vhm, p);
  return launch_status("vf4_cross_attn");
}

template <int LPK>
static int launch_rows(const XParams& p, cudaStream_t s) {
  const int64_t grid = (int64_t)p.B * p.Hkv * p.chunks;
  if (grid > INT32_MAX) return fail(VF4_ERR_UNSUPPORTED, "vf4_cross_attn: sizes too large");
  // as many warps per problem as keep 16 on every SM
  int warps = kRowWarps;
  while (warps > 1 && grid * warps > (int64_t)num_sms() * 24) warps /= 2;
  const unsigned threads = 32u * (unsigned)warps;
  if (p.R == 1) xattn_rows_kernel<LPK, 1><<<(unsigned)grid, threads, 0, s>>>(p);
  else if (p.R == 2) xattn_rows_kernel<LPK, 2><<<(unsigned)grid, threads, 0, s>>>(p);
  else xattn_rows_kernel<LPK, 4><<<(unsigned)grid, threads, 0, s>>>(p);
  return launch_status("vf4_cross_attn");
}

static bool sizes_ok(int64_t B, int64_t H, int64_t Hkv, int64_t Sq, int64_t Skv, int64_t D) {
  return B >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && Sq >= 0 && Skv >= 0 && D > 0;
}

}  // namespace vf4

using namespace vf4;

extern "C" {

int64_t vf4_cross_attn_workspace_size(int64_t B, int64_t H, int64_t Hkv, int64_t Sq, int64_t Skv, int64_t D) {
  if (!sizes_ok(B, H, Hkv, Sq, Skv, D) || B == 0 || Sq == 0 || Skv == 0) return 0;
  if (B > (1 << 24) || H > (1 << 16) || Sq > (1 << 24) || Skv > (1 << 30) || D > 128) return 0;   // refused by the call
  int chunk, chunks;
  plan_chunks(B, Hkv, H / Hkv * Sq, Skv, num_sms(), &chunk, &chunks);
  return chunks == 1 ? 0 : B * H * Sq * (int64_t)chunks * (D * 4 + 8);
}

int vf4_cross_attn(const void* q, int64_t q_b, int64_t q_h, int64_t q_s, const void* k, int64_t k_b, int64_t k_h,
                   int64_t k_s, const void* v, int64_t v_b, int64_t v_h, int64_t v_s, int64_t B, int64_t H, int64_t Hkv,
                   int64_t Sq, int64_t Skv, int64_t D, float scale, const int32_t* kv_lens, const uint8_t* key_mask,
                   int64_t mask_b, void* out, int64_t o_b, int64_t o_h, int64_t o_s, void* workspace,
                   int64_t workspace_bytes, vf4_stream_t stream) {
  if (int st = check_device()) return st;
  if (!sizes_ok(B, H, Hkv, Sq, Skv, D))
    return fail(VF4_ERR_ARG, "vf4_cross_attn: bad sizes (B=%lld H=%lld Hkv=%lld Sq=%lld Skv=%lld D=%lld)", (long long)B,
                (long long)H, (long long)Hkv, (long long)Sq, (long long)Skv, (long long)D);
  if (D % 8 || D > 128) return fail(VF4_ERR_UNSUPPORTED, "vf4_cross_attn: head dims that are multiples of 8 up to 128 (D=%lld)", (long long)D);
  if (B > (1 << 24) || H > (1 << 16) || Sq > (1 << 24) || Skv > (1 << 30) || H / Hkv * Sq > (1 << 28))
    return fail(VF4_ERR_UNSUPPORTED, "vf4_cross_attn: sizes too large");
  if (B == 0 || Sq == 0) return VF4_OK;
  if (B * H * Sq > INT32_MAX) return fail(VF4_ERR_UNSUPPORTED, "vf4_cross_attn: sizes too large");
  if (!q || !out || (Skv > 0 && (!k || !v))) return fail(VF4_ERR_ARG, "vf4_cross_attn: null operand");
  const int64_t strides[] = {q_b, q_h, q_s, k_b, k_h, k_s, v_b, v_h, v_s, o_b, o_h, o_s};
  for (int64_t x : strides)
    if (x % 8 || x < 0) return fail(VF4_ERR_ALIGN, "vf4_cross_attn: strides must be non-negative multiples of 8 elements");
  if (Skv > 1 && (k_s < D || v_s < D)) return fail(VF4_ERR_ARG, "vf4_cross_attn: keys or values overlap");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(workspace) ||
      reinterpret_cast<uintptr_t>(kv_lens) % 4)
    return fail(VF4_ERR_ALIGN, "vf4_cross_attn: operands must be 16-byte aligned");
  if (!(scale > -INFINITY && scale < INFINITY)) return fail(VF4_ERR_ARG, "vf4_cross_attn: scale is not finite");
  XParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.qb = q_b; p.qh = q_h; p.qs = q_s;
  p.kb = k_b; p.kh = k_h; p.ks = k_s;
  p.vb = v_b; p.vh = v_h; p.vs = v_s;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ob = o_b; p.oh = o_h; p.os = o_s;
  p.lens = kv_lens;
  p.mask = key_mask;
  p.mask_b = mask_b;
  p.B = (int)B; p.Hkv = (int)Hkv; p.G = (int)(H / Hkv); p.Sq = (int)Sq; p.Skv = (int)Skv; p.D = (int)D;
  p.R = p.G * p.Sq;
  p.negate = scale < 0.f;
  p.c = (scale < 0.f ? -scale : scale) * 1.4426950408889634f;
  if (p.c < 1.17549435e-38f) p.c = 1.17549435e-38f;   // a scale of 0: the least normal number, so that c * -inf stays -inf
  p.tiles = (p.R + 127) / 128;
  plan_chunks(B, Hkv, p.R, Skv, num_sms(), &p.chunk, &p.chunks);
  if (p.chunks > 1) {
    const int64_t rows = B * H * Sq * (int64_t)p.chunks;
    if (!workspace || workspace_bytes < rows * (D * 4 + 8))
      return fail(VF4_ERR_ARG, "vf4_cross_attn: workspace of %lld bytes needed, got %lld", (long long)(rows * (D * 4 + 8)),
                  (long long)workspace_bytes);
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + rows * D);
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int st = VF4_OK;
  if (Skv == 0) p.chunks = 0;   // without keys the rows are 0, which joining no chunks writes
  else if (plain_rows(p.R, Skv))
    st = D <= 32 ? launch_rows<4>(p, s) : D <= 64 ? launch_rows<8>(p, s) : launch_rows<16>(p, s);
  else
    st = D <= 64 ? launch_tc<64>(p, s) : launch_tc<128>(p, s);
  if (st || p.chunks == 1) return st;
  const int64_t rows = B * H * Sq;
  cudaLaunchAttribute at[1] = {early_launch()};
  cudaLaunchConfig_t cfg = {};
  // four chunks per warp have their loads in flight together: 4848 rows of 7 chunks take 31 us in all with two warps
  // per row and 43 with eight, one row of 64 chunks 13 us with eight and 31 with one
  int per_row = 1;
  while (per_row < kJoinWarps && per_row * 4 < p.chunks) per_row *= 2;
  cfg.gridDim = dim3((unsigned)((rows * per_row + kJoinWarps - 1) / kJoinWarps));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, xattn_join_kernel, p, per_row) != cudaSuccess) return launch_status("vf4_cross_attn (join)");
  return launch_status("vf4_cross_attn (join)");
}

}  // extern "C"
