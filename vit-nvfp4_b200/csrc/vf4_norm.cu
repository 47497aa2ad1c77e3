// Norms before and after a block, fused with the block's gate and residual scale:
//
//   x' = x + rs * gate (.) N_post(y)        h = N_pre(x')
//
// y is the block's output, x the residual stream; N is LayerNorm or RMSNorm with an optional weight and
// bias; the gate is one vector or one per group of rows (an image's).  h goes out in x's type or straight
// in the FP8 block format that the next layer's product reads.  The unfused chain reads and writes the
// rows up to nine times; here x and y are read once, x' and h written once.  Beside vf4_ln_cast_nvfp4,
// whose norm comes after the residual only and whose output is NVFP4.  No counterpart in the reference.
//
// A row lives in the registers of its threads (8 consecutive columns per thread and step, so that 16 lanes
// hold a block of 128).  Each thread takes the mean and the squared deviations of its own values, one pass
// over the threads joins them, all in fp32; x' enters the second norm before it is rounded for storage.
// Bound by memory for fp32 rows (32896 x 1024: 105 us, 5.1 TB/s); bf16 rows by their instructions as much (65792 x 1024,
// both norms: 100 us, 5.4 TB/s; without the post-norm 97, without the pre-norm 74, the pre-norm alone 50; to FP8 123, as the
// codes are the cast's own, whose correctly rounded quotient takes four instructions where a product takes one).
// Rows that are no multiple of 8 columns or not 16-byte aligned are read and written element by element: 30000 x 1171
// takes 200 us, 30000 x 1168 73.
#include "vf4_fp8_block.cuh"
#include "vf4_host.h"

namespace vf4 {

enum NormKind : int { kNormNone = 0, kNormLayer = 1, kNormRms = 2 };

struct NormParams {
  const void *x, *y, *gate, *w2, *b2, *w1, *b1;   // w2 / b2: post-norm, w1 / b1: pre-norm; NULL: 1 / 0
  int64_t M, ldx, ldy;
  uint32_t rows_per_gate;
  int K, post, pre;
  float rs, eps;
  void *x_out, *h;
  int64_t ldc;                 // FP8 output: bytes per code row
  float* scale;
  int64_t s_m, s_k;
};

// Eight consecutive values as four pairs: the arithmetic below runs on pairs (one issue slot for two
// elements; in scalars the bf16 rows were bound by instruction issue, not by memory).
using Pair = unsigned long long;
VF4_DEV Pair both(float a) { return f32x2_pack(a, a); }

template <typename T, bool kVec>
VF4_DEV void pairs8(const Raw8<T, kVec>& r, Pair* v) {
  if constexpr (kVec && sizeof(T) == 2) {
    v[0] = bf16x2_to_f32x2(r.w.x);
    v[1] = bf16x2_to_f32x2(r.w.y);
    v[2] = bf16x2_to_f32x2(r.w.z);
    v[3] = bf16x2_to_f32x2(r.w.w);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f32x2_pack(r.v[2 * i], r.v[2 * i + 1]);
  }
}

// Eight parameter values from element `at` on (nv valid).
template <typename P, bool kVec>
VF4_DEV void param8(const void* base, int64_t at, int nv, Pair* v) {
  Raw8<P, kVec> r;
  r.load(static_cast<const P*>(base) + at, nv);
  pairs8(r, v);
}

template <typename T, bool kVec>
VF4_DEV void store_row8(T* p, int nv, const Pair* v) {
  if (kVec && nv == 8) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(p) = make_uint4(bf16x2_round(v[0]), bf16x2_round(v[1]), bf16x2_round(v[2]), bf16x2_round(v[3]));
    } else {
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) f32x2_unpack(v[i], &f[2 * i], &f[2 * i + 1]);
      reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
  } else {
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) f32x2_unpack(v[i], &f[2 * i], &f[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < nv) p[i] = (T)f[i];
  }
}

// Sum over a row's threads: a warp, or a CTA (area: a float per warp).  One barrier per call: a call's area may be
// written again by the second call after it, whose writers have passed the barrier of the call between, which every
// reader reaches only after its reads.  So neighbouring calls take different areas, also from one row to the next.
template <int kThreads>
VF4_DEV float row_sum(float v, float* area) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if constexpr (kThreads > 32) {
    if ((threadIdx.x & 31) == 0) area[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) v += area[i];
  }
  return v;
}

// Mean and sum of squared deviations of a row whose threads hold n values each, from each thread's own: by pairs,
// as Chan, Golub and LeVeque update them ("Updating formulae and a pairwise algorithm for computing sample
// variances", 1979), so one pass over the threads gives both without the cancellation of E[v^2] - E[v]^2.
template <int kThreads>
VF4_DEV float2 row_moments(float n, float mean, float m2, float* area) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float b = __shfl_xor_sync(0xFFFFFFFFu, mean, o), d = b - mean;
    m2 += __shfl_xor_sync(0xFFFFFFFFu, m2, o);
    mean = 0.5f * (mean + b);
    m2 = fmaf(d * d, 0.5f * n, m2);
    n *= 2.f;
  }
  if constexpr (kThreads > 32) {
    constexpr int W = kThreads / 32;
    if ((threadIdx.x & 31) == 0) {
      area[threadIdx.x >> 5] = mean;
      area[W + (threadIdx.x >> 5)] = m2;
    }
    __syncthreads();
    mean = m2 = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) mean += area[i];
    mean *= 1.f / W;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float d = area[i] - mean;
      m2 += fmaf(d * d, n, area[W + i]);
    }
  }
  return make_float2(mean, m2);
}

VF4_DEV float pair_sum(Pair a) {
  float x, y;
  f32x2_unpack(a, &x, &y);
  return x + y;
}

// Pair i of a step without its elements past nv (non-vector rows; a vector row's steps are whole or empty).
VF4_DEV Pair clip(Pair v, int i, int nv) {
  float x, y;
  f32x2_unpack(v, &x, &y);
  return f32x2_pack(2 * i < nv ? x : 0.f, 2 * i + 1 < nv ? y : 0.f);
}

// Centres v (LayerNorm) over the NV * 8 values of this thread's part of the row and returns 1 / sqrt(var + eps).
// Columns past K hold 0 before and after.  area: 3 * warps floats.
template <int kThreads, int NV, bool kVec>
VF4_DEV float centre(Pair (*v)[4], const int* nv, int kind, int K, float eps, float* area) {
  constexpr int W = kThreads / 32;
  auto squares = [&](Pair neg) {   // of v + neg, over this thread's columns
    Pair q = 0ull;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        Pair d = add_f32x2(v[j][i], neg);
        if (!kVec) d = clip(d, i, nv[j]);
        if (!kVec || nv[j] > 0) q = fma_f32x2(d, d, q);
      }
    return pair_sum(q);
  };
  auto shift = [&](Pair neg) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (kVec && nv[j] <= 0) continue;
        v[j][i] = add_f32x2(v[j][i], neg);
        if (!kVec) v[j][i] = clip(v[j][i], i, nv[j]);
      }
  };
  float m2;
  if (kind == kNormLayer) {
    Pair s = 0ull;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) s = add_f32x2(s, v[j][i]);
    const float sum = pair_sum(s);
    if (K % (8 * kThreads) == 0) {   // every thread holds as many columns
      const float n = (float)(K / kThreads), mean = __fdividef(sum, n);
      const float2 mm = row_moments<kThreads>(n, mean, squares(both(-mean)), area);
      m2 = mm.y;
      shift(both(-mm.x));
    } else {                         // in two passes over the threads
      const Pair neg = both(-__fdividef(row_sum<kThreads>(sum, area), (float)K));
      shift(neg);
      m2 = row_sum<kThreads>(squares(0ull), area + 2 * W);
    }
  } else {
    m2 = row_sum<kThreads>(squares(0ull), area);
  }
  return rsqrtf(__fdividef(m2, (float)K) + eps);
}

// z = v * r * w + b for eight columns.
template <typename P, bool kVec>
VF4_DEV void affine8(Pair* v, float r, const void* w, const void* b, int col, int nv) {
  Pair p[4];
  if (w) {
    param8<P, kVec>(w, col, nv, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = mul_f32x2(p[i], both(r));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = both(r);
  }
  if (b) {
    Pair q[4];
    param8<P, kVec>(b, col, nv, q);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fma_f32x2(v[i], p[i], q[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mul_f32x2(v[i], p[i]);
  }
}

// kThreads = 32: a warp per row, 8 rows per CTA in turn; else a CTA per row.  P: the parameters' type.  kOut: 0 no
// h, 1 h in T, 2 FP8.
template <typename T, typename P, int kThreads, int NV, bool kVec, int kOut>
__global__ void __launch_bounds__(kThreads == 32 ? 256 : kThreads, kThreads == 32 ? (NV > 4 ? 2 : 3) : 1) gated_norm_kernel(const NormParams p) {
  // one of the two per norm, in turn: with one norm per row, too, no warp writes the area that another may still be
  // reading for the row before
  __shared__ float red[2][3 * (kThreads / 32)];
  int side = 0;
  constexpr int kRows = kThreads == 32 ? 8 : 1;
  const int t = kThreads == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const T *X = static_cast<const T*>(p.x), *Y = static_cast<const T*>(p.y);
  T *XO = static_cast<T*>(p.x_out), *H = static_cast<T*>(p.h);
  int nv[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) nv[j] = max(0, min(8, p.K - (j * kThreads + t) * 8));
  // with several gates, a run of neighbouring rows per warp (CTA), which share a gate that then comes from L1
  // (65792 x 1024 with 256 gates: 119 -> 102 us; without gates the runs cost 2%)
  const int64_t runs = gridDim.x * (int64_t)kRows, run = blockIdx.x * (int64_t)kRows + (kThreads == 32 ? threadIdx.x >> 5 : 0);
  const bool grouped = p.gate && p.rows_per_gate < p.M;
  const int64_t end = grouped ? p.M * (run + 1) / runs : p.M, step = grouped ? 1 : runs;
  for (int64_t row = grouped ? p.M * run / runs : run; row < end; row += step) {
    Raw8<T, kVec> xr[NV];
    Pair v[NV][4];
#pragma unroll
    for (int j = 0; j < NV; ++j) xr[j].load(X + row * p.ldx + (j * kThreads + t) * 8, nv[j]);
    if (p.y) {
      Raw8<T, kVec> yr[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) yr[j].load(Y + row * p.ldy + (j * kThreads + t) * 8, nv[j]);
#pragma unroll
      for (int j = 0; j < NV; ++j) pairs8(yr[j], v[j]);
      float r2 = 1.f;
      if (p.post != kNormNone) {
        r2 = centre<kThreads, NV, kVec>(v, nv, p.post, p.K, p.eps, red[side]);
        side ^= 1;
      }
      const int64_t gate_row = p.gate ? (int64_t)((uint32_t)row / p.rows_per_gate) * p.K : 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (nv[j] <= 0) continue;
        const int col = (j * kThreads + t) * 8;
        Pair x[4], g[4];
        if (p.post != kNormNone) affine8<P, kVec>(v[j], r2, p.w2, p.b2, col, nv[j]);
        if (p.gate) {
          param8<P, kVec>(p.gate, gate_row + col, nv[j], g);
#pragma unroll
          for (int i = 0; i < 4; ++i) g[i] = mul_f32x2(g[i], both(p.rs));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) g[i] = both(p.rs);
        }
        pairs8(xr[j], x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[j][i] = fma_f32x2(v[j][i], g[i], x[i]);
          if (!kVec) v[j][i] = clip(v[j][i], i, nv[j]);
        }
        store_row8<T, kVec>(XO + row * p.K + col, nv[j], v[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) pairs8(xr[j], v[j]);
    }
    if constexpr (kOut != 0) {
      const float r1 = centre<kThreads, NV, kVec>(v, nv, p.pre, p.K, p.eps, red[side]);
      side ^= 1;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int col = (j * kThreads + t) * 8;
        if (nv[j] > 0) affine8<P, kVec>(v[j], r1, p.w1, p.b1, col, nv[j]);
        if constexpr (kOut == 1) {
          if (nv[j] > 0) store_row8<T, kVec>(H + row * p.K + col, nv[j], v[j]);
        } else {
          float f[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) f32x2_unpack(v[j][i], &f[2 * i], &f[2 * i + 1]);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (kVec ? nv[j] <= 0 : i >= nv[j]) f[i] = 0.f;
          uint32_t m = amax8_bits(f);
#pragma unroll
          for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
          if (nv[j] > 0) {
            const Fp8Block q = fp8_block(m);   // the cast's codes and scale, bit for bit
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.h) + row * p.ldc + col) = fp8_encode8(f, q);
            if ((t & 15) == 0) p.scale[row * p.s_m + (col >> 7) * p.s_k] = q.scale;
          }
        }
      }
    }
  }
}

template <typename T, typename P, int kThreads, int NV, bool kVec>
static void launch_norm(const NormParams& p, int out, cudaStream_t s) {
  const int64_t rows = kThreads == 32 ? 8 : 1;
  const int64_t want = (p.M + rows - 1) / rows;
  const int64_t most = (int64_t)num_sms() * (kThreads == 32 ? (NV > 4 ? 2 : 3) : 16);
  const unsigned grid = (unsigned)(want < most ? want : most);
  constexpr int block = kThreads == 32 ? 256 : kThreads;
  if (out == 0) gated_norm_kernel<T, P, kThreads, NV, kVec, 0><<<grid, block, 0, s>>>(p);
  else if (out == 1) gated_norm_kernel<T, P, kThreads, NV, kVec, 1><<<grid, block, 0, s>>>(p);
  else gated_norm_kernel<T, P, kThreads, NV, kVec, 2><<<grid, block, 0, s>>>(p);
}

// Threads per row and steps of 8 columns per thread by the rows' number and length.  Up to 1280 columns a warp
// takes a row, unless there are so few rows that most SMs would get none or one (257 rows of 1024: 8.6 us with a
// warp per row, 3.9 with a CTA); then, as for longer rows, a CTA takes a row.  Threads x steps of longer rows, both norms,
// bf16: up to 2048 columns 256 x 1 (257 rows of 2048: 3.5 us, 3.9 with 128 x 2; but 32896 rows 161 us, 120 with 128 x 2),
// up to 4096 256 x 2 (16400 rows 127, with 512 x 1 205), up to 5120 320 x 2 (13000 rows 141, with 640 x 1 287), up to 8192
// 256 x 4 (8200 rows 133, with 512 x 2 220), beyond 512 x 4 (4100 rows of 16384: 155, with 1024 x 2 209): the more threads
// share a row, the longer its two reductions take beside its loads.
template <typename T, typename P, bool kVec>
static void dispatch_norm(const NormParams& p, int out, cudaStream_t s) {
  const bool few = p.M <= 8 * (int64_t)num_sms();
  if (p.K <= 256) launch_norm<T, P, 32, 1, kVec>(p, out, s);
  else if (p.K <= 512 && !few) launch_norm<T, P, 32, 2, kVec>(p, out, s);
  else if (p.K <= 1024 && !few) launch_norm<T, P, 32, 4, kVec>(p, out, s);
  else if (p.K <= 1024) launch_norm<T, P, 128, 1, kVec>(p, out, s);
  else if (p.K <= 1280 && !few) launch_norm<T, P, 32, 5, kVec>(p, out, s);
  else if (p.K <= 1280) launch_norm<T, P, 160, 1, kVec>(p, out, s);
  else if (p.K <= 2048) launch_norm<T, P, 256, 1, kVec>(p, out, s);
  else if (p.K <= 4096) launch_norm<T, P, 256, 2, kVec>(p, out, s);
  else if (p.K <= 5120) launch_norm<T, P, 320, 2, kVec>(p, out, s);
  else if (p.K <= 8192) launch_norm<T, P, 256, 4, kVec>(p, out, s);
  else launch_norm<T, P, 512, 4, kVec>(p, out, s);
}

}  // namespace vf4

using namespace vf4;

extern "C" int vf4_gated_residual_norm(const void* x, int64_t ldx, const void* y, int64_t ldy, int dtype, int64_t M,
                                       int64_t K, const void* gate, int64_t gate_groups, float residual_scale,
                                       int post, const void* post_w, const void* post_b, int pre, const void* pre_w,
                                       const void* pre_b, int param_dtype, float eps, void* x_out, void* h,
                                       int h_fp8, int64_t ldc, float* scale, int64_t stride_m, int64_t stride_k,
                                       vf4_stream_t stream) {
  const char* me = "vf4_gated_residual_norm";
  if (int st = check_device()) return st;
  if (M < 0 || K <= 0 || ldx < K || (y && ldy < K)) return fail(VF4_ERR_ARG, "%s: bad sizes (M=%lld K=%lld)", me, (long long)M, (long long)K);
  if (M > INT32_MAX) return fail(VF4_ERR_UNSUPPORTED, "%s: too many rows (%lld)", me, (long long)M);
  if (K > 16384) return fail(VF4_ERR_UNSUPPORTED, "%s: rows of at most 16384 columns (K=%lld)", me, (long long)K);
  if ((dtype != VF4_BF16 && dtype != VF4_F32) || (param_dtype != VF4_BF16 && param_dtype != VF4_F32))
    return fail(VF4_ERR_ARG, "%s: bad dtype", me);
  if (dtype == VF4_F32 && param_dtype != VF4_F32 && (gate || post_w || post_b || pre_w || pre_b))
    return fail(VF4_ERR_UNSUPPORTED, "%s: fp32 rows take fp32 parameters", me);
  if (post < kNormNone || post > kNormRms || pre < kNormNone || pre > kNormRms) return fail(VF4_ERR_ARG, "%s: bad norm", me);
  if ((!y && (post != kNormNone || gate || pre == kNormNone)) || (post == kNormNone && (post_w || post_b)) ||
      (pre == kNormNone && (pre_w || pre_b)))
    return fail(VF4_ERR_ARG, "%s: a norm, its parameters or the gate without what it applies to", me);
  if (gate && (gate_groups < 1 || M % gate_groups)) return fail(VF4_ERR_ARG, "%s: %lld rows do not divide into %lld gates", me, (long long)M, (long long)gate_groups);
  if (M == 0) return VF4_OK;
  if (!x || (y && !x_out) || (pre != kNormNone && !h) || (h_fp8 && pre != kNormNone && !scale))
    return fail(VF4_ERR_ARG, "%s: missing pointer", me);
  if (h_fp8 && pre != kNormNone && (!aligned16(h) || ldc % 16 || ldc < K))
    return fail(VF4_ERR_ALIGN, "%s: code rows need 16-byte aligned starts of at least K bytes (ldc=%lld)", me, (long long)ldc);
  const int esz = dtype == VF4_BF16 ? 2 : 4, psz = param_dtype == VF4_BF16 ? 2 : 4;
  const void* rows[] = {x, y, x_out, h_fp8 ? nullptr : h};
  const void* params[] = {gate, post_w, post_b, pre_w, pre_b};
  bool vec = K % 8 == 0 && ldx * esz % 16 == 0 && (!y || ldy * esz % 16 == 0);
  for (const void* q : rows) {
    if (reinterpret_cast<uintptr_t>(q) % esz) return fail(VF4_ERR_ALIGN, "%s: a pointer is misaligned for its type", me);
    vec = vec && aligned16(q);
  }
  for (const void* q : params) {
    if (reinterpret_cast<uintptr_t>(q) % psz) return fail(VF4_ERR_ALIGN, "%s: a pointer is misaligned for its type", me);
    vec = vec && aligned16(q);
  }
  NormParams p{};
  p.x = x; p.y = y; p.gate = gate; p.w2 = post_w; p.b2 = post_b; p.w1 = pre_w; p.b1 = pre_b;
  p.M = M; p.ldx = ldx; p.ldy = ldy;
  p.rows_per_gate = gate ? (uint32_t)(M / gate_groups) : 1u;
  p.K = (int)K; p.post = post; p.pre = pre;
  p.rs = residual_scale; p.eps = eps;
  p.x_out = x_out; p.h = h;
  p.ldc = ldc; p.scale = scale; p.s_m = stride_m; p.s_k = stride_k;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int out = pre == kNormNone ? 0 : h_fp8 ? 2 : 1;
  if (dtype == VF4_F32) {
    if (vec) dispatch_norm<float, float, true>(p, out, s);
    else dispatch_norm<float, float, false>(p, out, s);
  } else if (param_dtype == VF4_F32) {
    if (vec) dispatch_norm<__nv_bfloat16, float, true>(p, out, s);
    else dispatch_norm<__nv_bfloat16, float, false>(p, out, s);
  } else {
    if (vec) dispatch_norm<__nv_bfloat16, __nv_bfloat16, true>(p, out, s);
    else dispatch_norm<__nv_bfloat16, __nv_bfloat16, false>(p, out, s);
  }
  return launch_status(me);
}
