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
#include "vf4_fp8_block.cuh"
#include "vf4_host.h"

namespace vf4 {

enum NormKind : int { kNormNone = 0, kNormLayer = 1, kNormRms = 2 };

struct NormParams {
  const void *x, *y, *gate, *w2, *b2, *w1, *b1;   // w2 / b2: post-norm, w1 / b1: pre-norm; NULL: 1 / 0
  int64_t M, ldx, ldy;
  uint32_t rows_per_gate;
  int K, post, pre, p_f32;     // p_f32: the parameters' type (gate, weights, biases)
  float rs, eps;
  void *x_out, *h;
  int64_t ldc;                 // FP8 output: bytes per code row
  float* scale;
  int64_t s_m, s_k;
};

// Eight parameter values from column col (nv valid), of either type.
template <bool kVec>
VF4_DEV void param8(const void* base, int64_t at, int f32, int nv, float* v) {
  if (f32) load8<float, kVec>(static_cast<const float*>(base) + at, nv, v);
  else load8<__nv_bfloat16, kVec>(static_cast<const __nv_bfloat16*>(base) + at, nv, v);
}

template <typename T, bool kVec>
VF4_DEV void store_row8(T* p, int nv, const float* v) {
  if (kVec && nv == 8) {
    if constexpr (sizeof(T) == 2) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = bf16x2_round(f32x2_pack(v[2 * i], v[2 * i + 1]));
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < nv) p[i] = (T)v[i];
  }
}

// (count, mean, sum of squared deviations) of two disjoint parts, by the update of Chan, Golub and LeVeque
// ("Updating formulae and a pairwise algorithm for computing sample variances", 1979): one pass over the
// threads gives mean and variance without the cancellation of E[v^2] - E[v]^2.
struct Moments {
  float n, mean, m2;
};
VF4_DEV Moments join(const Moments& a, const Moments& b) {
  const float n = a.n + b.n, f = n > 0.f ? __fdividef(b.n, n) : 0.f, d = b.mean - a.mean;
  return {n, fmaf(d, f, a.mean), a.m2 + b.m2 + d * d * a.n * f};
}

// The row's moments, joined over its threads: a warp, or a CTA (red: its warps' moments; the caller
// alternates between two such areas, so one barrier per call is enough).  kind RMS: mean 0, m2 the sum of
// squares.  even: every thread holds as many columns, and the joins need no weights.
template <int kThreads>
VF4_DEV Moments row_moments(Moments v, int kind, bool even, Moments* red) {
  if (kind == kNormRms) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v.m2 += __shfl_xor_sync(0xFFFFFFFFu, v.m2, o);
  } else if (even) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float mean = __shfl_xor_sync(0xFFFFFFFFu, v.mean, o), m2 = __shfl_xor_sync(0xFFFFFFFFu, v.m2, o);
      const float d = mean - v.mean;
      v.mean = 0.5f * (v.mean + mean);
      v.m2 = fmaf(d * d, 0.5f * v.n, v.m2 + m2);
      v.n *= 2.f;
    }
  } else {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      Moments q{__shfl_xor_sync(0xFFFFFFFFu, v.n, o), __shfl_xor_sync(0xFFFFFFFFu, v.mean, o),
                __shfl_xor_sync(0xFFFFFFFFu, v.m2, o)};
      // both lanes of a pair join in the same order, so that all lanes end with the same values
      v = (threadIdx.x & o) ? join(q, v) : join(v, q);
    }
  }
  if constexpr (kThreads > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < kThreads / 32; ++i) {
      if (kind == kNormRms) v.m2 += red[i].m2;
      else v = join(v, red[i]);
    }
  }
  return v;
}

// Centres v (LayerNorm) over the NV * 8 values of this thread's part of the row and returns 1 / sqrt(var + eps).
template <int kThreads, int NV, bool kVec>
VF4_DEV float centre(float (*v)[8], const int* nv, int kind, int K, float eps, Moments* red) {
  Moments m{0.f, 0.f, 0.f};
  if (kind == kNormLayer) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      m.n += (float)nv[j];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[j][i];   // columns past K hold 0
    }
    m.mean = m.n > 0.f ? __fdividef(s, m.n) : 0.f;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (kVec ? nv[j] > 0 : i < nv[j]) {
        const float d = v[j][i] - m.mean;
        m.m2 = fmaf(d, d, m.m2);
      }
  m = row_moments<kThreads>(m, kind, K % (8 * kThreads) == 0, red);
  if (kind == kNormLayer) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (kVec ? nv[j] > 0 : i < nv[j]) v[j][i] -= m.mean;   // columns past K stay 0
  }
  return rsqrtf(__fdividef(m.m2, (float)K) + eps);
}

// z = v * r * w + b for eight columns.
template <bool kVec>
VF4_DEV void affine8(float* v, float r, const void* w, const void* b, int col, int f32, int nv) {
  float p[8];
  if (w) {
    param8<kVec>(w, col, f32, nv, p);
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] *= r;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = r;
  }
  if (b) {
    float q[8];
    param8<kVec>(b, col, f32, nv, q);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(v[i], p[i], q[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= p[i];
  }
}

// kThreads = 32: a warp per row, 8 rows per CTA in turn; else a CTA per row.  kOut: 0 no h, 1 h in T, 2 FP8.
template <typename T, int kThreads, int NV, bool kVec, int kOut>
__global__ void __launch_bounds__(kThreads == 32 ? 256 : kThreads, kThreads == 32 ? 2 : 1) gated_norm_kernel(const NormParams p) {
  __shared__ Moments red[2][kThreads > 32 ? kThreads / 32 : 1];
  constexpr int kRows = kThreads == 32 ? 8 : 1;
  const int t = kThreads == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const T *X = static_cast<const T*>(p.x), *Y = static_cast<const T*>(p.y);
  T *XO = static_cast<T*>(p.x_out), *H = static_cast<T*>(p.h);
  int nv[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) nv[j] = max(0, min(8, p.K - (j * kThreads + t) * 8));
  // kAhead: the next row's x and y are loaded while this one is worked on (one warp per row leaves too few
  // warps per SM to keep the memory busy otherwise)
  constexpr bool kAhead = kThreads == 32 && sizeof(T) == 2 && kVec;
  const int64_t row0 = blockIdx.x * (int64_t)kRows + (kThreads == 32 ? threadIdx.x >> 5 : 0), step = gridDim.x * (int64_t)kRows;
  Raw8<T, kVec> xr[NV], yr[NV], xn[kAhead ? NV : 1], yn[kAhead ? NV : 1];
  auto fetch = [&](int64_t row, Raw8<T, kVec>* a, Raw8<T, kVec>* b) {
#pragma unroll
    for (int j = 0; j < NV; ++j) a[j].load(X + row * p.ldx + (j * kThreads + t) * 8, row < p.M ? nv[j] : 0);
    if (p.y) {
#pragma unroll
      for (int j = 0; j < NV; ++j) b[j].load(Y + row * p.ldy + (j * kThreads + t) * 8, row < p.M ? nv[j] : 0);
    }
  };
  if (kAhead) fetch(row0, xn, yn);
  for (int64_t row = row0; row < p.M; row += step) {
    if constexpr (kAhead) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        xr[j] = xn[j];
        yr[j] = yn[j];
      }
      fetch(row + step, xn, yn);
    } else {
      fetch(row, xr, yr);
    }
    float v[NV][8];
    if (p.y) {
#pragma unroll
      for (int j = 0; j < NV; ++j) yr[j].get(v[j]);
      float r2 = 1.f;
      if (p.post != kNormNone) r2 = centre<kThreads, NV, kVec>(v, nv, p.post, p.K, p.eps, red[0]);
      const int64_t gate_row = p.gate ? (int64_t)((uint32_t)row / p.rows_per_gate) * p.K : 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (nv[j] <= 0) continue;
        const int col = (j * kThreads + t) * 8;
        float x[8], g[8];
        if (p.post != kNormNone) affine8<kVec>(v[j], r2, p.w2, p.b2, col, p.p_f32, nv[j]);
        if (p.gate) {
          param8<kVec>(p.gate, gate_row + col, p.p_f32, nv[j], g);
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] *= p.rs;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] = p.rs;
        }
        xr[j].get(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = fmaf(v[j][i], g[i], x[i]);
        store_row8<T, kVec>(XO + row * p.K + col, nv[j], v[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) xr[j].get(v[j]);
    }
    if constexpr (kOut != 0) {
      const float r1 = centre<kThreads, NV, kVec>(v, nv, p.pre, p.K, p.eps, red[1]);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int col = (j * kThreads + t) * 8;
        if (nv[j] > 0) affine8<kVec>(v[j], r1, p.w1, p.b1, col, p.p_f32, nv[j]);
        if constexpr (kOut == 1) {
          if (nv[j] > 0) store_row8<T, kVec>(H + row * p.K + col, nv[j], v[j]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i >= nv[j]) v[j][i] = 0.f;
          uint32_t m = amax8_bits(v[j]);
#pragma unroll
          for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
          if (nv[j] > 0) {
            // the quotient as one product: h is itself an fp32 result, off by more than the product's two
            // roundings (the cast's correctly rounded quotient costs four times as much here)
            float a = __uint_as_float(m);
            a = a < 1e-12f ? 1e-12f : a;
            const float q = __fdividef(448.f, a);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = e4m3x2(v[j][2 * i] * q, v[j][2 * i + 1] * q);
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.h) + row * p.ldc + col) =
                make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
            if ((t & 15) == 0) p.scale[row * p.s_m + (col >> 7) * p.s_k] = __fdiv_rn(a, 448.f);
          }
        }
      }
    }
  }
}

template <typename T, int kThreads, int NV, bool kVec>
static void launch_norm(const NormParams& p, int out, cudaStream_t s) {
  const int64_t rows = kThreads == 32 ? 8 : 1;
  const int64_t want = (p.M + rows - 1) / rows;
  const int64_t most = (int64_t)num_sms() * (kThreads == 32 ? 4 : 16);
  const unsigned grid = (unsigned)(want < most ? want : most);
  constexpr int block = kThreads == 32 ? 256 : kThreads;
  if (out == 0) gated_norm_kernel<T, kThreads, NV, kVec, 0><<<grid, block, 0, s>>>(p);
  else if (out == 1) gated_norm_kernel<T, kThreads, NV, kVec, 1><<<grid, block, 0, s>>>(p);
  else gated_norm_kernel<T, kThreads, NV, kVec, 2><<<grid, block, 0, s>>>(p);
}

// Threads per row and steps of 8 columns per thread by the rows' number and length.  Up to 1024 columns a warp
// takes a row, unless there are so few rows that most SMs would get none or one: then, as for longer rows, a
// CTA takes a row, of the threads that the row fills in one step where that is at most 256.
template <typename T, bool kVec>
static void dispatch_norm(const NormParams& p, int out, cudaStream_t s) {
  const bool few = p.M <= 8 * (int64_t)num_sms();
  if (p.K <= 256) launch_norm<T, 32, 1, kVec>(p, out, s);
  else if (p.K <= 512 && !few) launch_norm<T, 32, 2, kVec>(p, out, s);
  else if (p.K <= 1024 && !few) launch_norm<T, 32, 4, kVec>(p, out, s);
  else if (p.K <= 1024) launch_norm<T, 128, 1, kVec>(p, out, s);
  else if (p.K <= 1280) launch_norm<T, 160, 1, kVec>(p, out, s);
  else if (p.K <= 2048) launch_norm<T, 256, 1, kVec>(p, out, s);
  else if (p.K <= 4096) launch_norm<T, 256, 2, kVec>(p, out, s);
  else if (p.K <= 8192) launch_norm<T, 256, 4, kVec>(p, out, s);
  else launch_norm<T, 512, 4, kVec>(p, out, s);
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
  p.p_f32 = param_dtype == VF4_F32;
  p.rs = residual_scale; p.eps = eps;
  p.x_out = x_out; p.h = h;
  p.ldc = ldc; p.scale = scale; p.s_m = stride_m; p.s_k = stride_k;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int out = pre == kNormNone ? 0 : h_fp8 ? 2 : 1;
  if (dtype == VF4_BF16) {
    if (vec) dispatch_norm<__nv_bfloat16, true>(p, out, s);
    else dispatch_norm<__nv_bfloat16, false>(p, out, s);
  } else {
    if (vec) dispatch_norm<float, true>(p, out, s);
    else dispatch_norm<float, false>(p, out, s);
  }
  return launch_status(me);
}
