// FP8 block format (E4M3 codes, one fp32 scale per 128 columns or per 128 x 128 block): the cast and
// the product
//
//   y[m, n] = sum_g sa[m, g] sb[n / 128, g] sum_{k in block g} a[m, k] b[n, k]  (+ bias[n])
//
// No counterpart in the reference, whose formats are bf16 and NVFP4; the framework's layers that stay
// out of NVFP4 (heads, first and last blocks, projections of a cross attention) take this one.
#include <cuda_fp16.h>
#include <string.h>

#include "vf4_fp8_block.cuh"
#include "vf4_host.h"

namespace vf4 {

static __device__ int g_fp8_err;

int fp8_device_error(int clear) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_fp8_err, sizeof(int));
  if (clear) {
    int z = 0;
    cudaMemcpyToSymbol(g_fp8_err, &z, sizeof(int));
  }
  return v;
}

// ---------------------------------------------------------------------------------------
// Cast of activations: 16 lanes hold the 128 columns of one block, 8 each (one 16-byte load of bf16).
// The blocks of all rows are numbered in one sequence, row by row, and dealt to the half-warps, so
// short and long rows fill the machine alike.  Bound by memory: 1 byte out per 2 (bf16) or 4 (fp32)
// bytes in; kU blocks per half-warp are loaded before the first is reduced, to keep enough bytes in
// flight, as few as leave registers for five CTAs per SM (16400 x 1280 and 16400 x 5120 bf16: 16.6 and 58.2 us with two
// blocks; 17.4 and 58.9 with four and four CTAs, 17.5 and 61.3 with three, 20.6 and 72.5 with one).  fp32 rows go at
// the memory's rate (16400 x 5120: 66 us, 64 for its bytes).  Rows that are no multiple of 8 columns or not 16-byte
// aligned are read element by element: 8000 x 1171 takes 11.9 us, 8000 x 1168 9.8.
// ---------------------------------------------------------------------------------------
template <typename T, bool kVec, int kU>
__global__ void __launch_bounds__(256, 5) fp8_cast_rows_kernel(const T* __restrict__ x, int64_t M, int K, int64_t ld,
                                                               uint8_t* __restrict__ codes, int64_t ldc,
                                                               float* __restrict__ scale, int64_t s_m, int64_t s_k) {
  const int kb = (K + 127) >> 7;
  const int l = threadIdx.x & 15;
  const int hw = (blockIdx.x * blockDim.x + threadIdx.x) >> 4, n_hw = (gridDim.x * blockDim.x) >> 4;
  // (row, column block) of this half-warp's next block; a step of n_hw blocks is (d_row, d_g) with a carry,
  // so no division runs per block.  Both halves of a warp take as many steps (the shuffles name all lanes).
  const int d_row = n_hw / kb, d_g = n_hw - d_row * kb;
  int row = hw / kb, g = hw - row * kb;
  const int64_t steps = (M * kb - (hw & ~1) + n_hw - 1) / n_hw;
  griddep_launch();   // the product may set itself up meanwhile
  for (int64_t i = 0; i < steps; i += kU) {
    Raw8<T, kVec> v[kU];
    int at_row[kU], at_g[kU], nv[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      at_row[u] = row;
      at_g[u] = g;
      const int col = g * 128 + l * 8;
      nv[u] = row < M ? min(8, K - col) : 0;
      v[u].load(x + row * ld + col, nv[u]);
      row += d_row;
      g += d_g;
      if (g >= kb) {
        g -= kb;
        ++row;
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      uint32_t m = v[u].amax_bits();
#pragma unroll
      for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
      const Fp8Block q = fp8_block(m);
      if (nv[u] > 0) {   // columns of the row's padding (ldc >= K rounded up to 16) are written as 0
        float f[8];
        v[u].get(f);
        *reinterpret_cast<uint2*>(codes + at_row[u] * ldc + at_g[u] * 128 + l * 8) = fp8_encode8(f, q);
        if (l == 0) scale[at_row[u] * s_m + at_g[u] * s_k] = q.scale;
      }
    }
  }
}

// Cast of weights: one CTA per 128 x 128 block, every thread 8 columns of 8 rows.  Runs once per weight (5120 x 1280: 7.4 us
// from bf16, 8.4 from fp32, whose bytes take 3.0 and 5.0).
template <typename T, bool kVec>
__global__ void __launch_bounds__(256) fp8_cast_tile_kernel(const T* __restrict__ x, int64_t M, int K, int64_t ld,
                                                            uint8_t* __restrict__ codes, int64_t ldc,
                                                            float* __restrict__ scale, int64_t s_m, int64_t s_k) {
  __shared__ uint32_t red[8];
  const int kb = (K + 127) >> 7;
  const int64_t mb = blockIdx.x / kb;
  const int g = (int)(blockIdx.x - mb * kb);
  const int l = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int col = g * 128 + l * 8;
  const int nc = min(8, K - col);
  float v[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = mb * 128 + r0 + 16 * i;
    load8<T, kVec>(x + row * ld + col, row < M ? nc : 0, v[i]);
    m = max(m, amax8_bits(v[i]));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, red[i]);
  const Fp8Block q = fp8_block(m);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = mb * 128 + r0 + 16 * i;
    if (row < M && nc > 0) *reinterpret_cast<uint2*>(codes + row * ldc + col) = fp8_encode8(v[i], q);
  }
  if (threadIdx.x == 0) scale[mb * s_m + g * s_k] = q.scale;
}

// ---------------------------------------------------------------------------------------
// The product.  One K block of 128 columns is four tcgen05 MMAs (kind::f8f6f4, K = 32) into an
// accumulator of its own in tensor memory; the epilogue warps read it, multiply it by the block's
// scales and add it to the running fp32 sums in their registers, while the tensor cores fill the next
// accumulator.  The scales are arbitrary fp32 numbers, so they cannot go through the MMA (its
// hardware scales are powers of two or E4M3).
//
//   warp 0      TMA: 128 rows of A and BN rows of B, 128 bytes of K each, 128-byte swizzle
//   warp 1      TMEM allocation, MMAs
//   warps 2..   epilogue (4.. with the 256-column tile): each TMEM lane quadrant's rows, NC of the BN
//               columns per warp
//
// Two roles of the operands:
//   kSwap = false  A = activations, B = weight.  A row's scale is per thread, the weight's per 128
//                  columns: one multiplication per thread and block.
//   kSwap = true   A = weight, B = activations, for up to 64 rows of activations: BN is 16, 32 or 64
//                  instead of padding the activations to 128 rows; y^T comes out, a lane per n.
//
// Few tiles: a cluster of `split` CTAs shares one tile, each taking a run of K blocks, and adds its
// sums up through distributed shared memory, in the order of the ranks (no atomics, no workspace: the
// result does not depend on timing).
// ---------------------------------------------------------------------------------------
template <int BN, bool kSwap>
struct F8Cfg {
  // 256 columns: a pair of CTAs (one cluster) shares a 256 x 256 tile, each holding 128 rows of A and 128
  // of B's 256 rows in its own shared memory
  static constexpr bool kPair = BN == 256;
  static constexpr int A_BYTES = 128 * 128, B_BYTES = (kPair ? 128 : BN) * 128, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int ROWS = kPair ? 256 : 128;         // rows of a tile
  // 16 and 32 columns: two CTAs on an SM, one's epilogue beside the other's loads (32 x 5120 x 5120: 10.3 us, 13.0 with
  // one CTA of 8 stages).  64 columns: one (64 x 5120 x 1280: 7.1 us, 8.6 with two of 4 stages)
  static constexpr int PER_SM = kSwap && BN < 64 ? 2 : 1;
  static constexpr int STAGES = kPair ? 4 : kSwap && BN == 64 ? 8 : 5;
  static constexpr int ACCS = BN == 256 ? 2 : 4;
  static constexpr int TMEM_COLS = ACCS * BN;            // 64 .. 512, a power of two
  static constexpr int EW = kPair ? 4 : BN >= 64 ? 2 : 1;   // epilogue warps per lane quadrant
  static constexpr int NC = BN / EW;                     // columns per epilogue warp
  static constexpr int EPI_WARPS = 4 * EW;
  // columns per TMEM load, and loads whose registers a thread holds: with two, the next load is in flight while one
  // is multiplied in.  The 256-column tile has sixteen warps of 64 columns with one load each: eight warps of 128
  // columns and two loads are as fast over long K (8192 x 5120 x 5120: 229 us) but 3 to 7% slower over K of 1280 to
  // 4096, where their two staged halves of the output wait for each other
  static constexpr int CH = NC >= 64 ? 32 : 16, BUF = kPair ? 1 : 2;
  // those take registers over from the four warps of the control group (two of them idle)
  static constexpr bool kRegs = kPair;
  static constexpr int EPI0 = kRegs ? 4 : 2;             // first epilogue warp
  static constexpr int THREADS = 32 * (EPI0 + EPI_WARPS);
  static constexpr int kLaunchRegs = 96, kControlRegs = 32, kEpiRegs = 112;   // 640 threads: 96 at launch
  static_assert(!kRegs || 128 * kControlRegs + 512 * kEpiRegs <= THREADS * kLaunchRegs, "register split");
  static constexpr int STG_OFF = STAGES * STAGE_BYTES;   // bf16 output staging, 32 rows x 64 columns per warp
  static constexpr int STG_BYTES = kSwap ? 0 : EPI_WARPS * 4096;
  // scales on their way to the epilogue threads: kRing K blocks ahead, across tiles, {own row's, weight block's}
  // per thread.  kSwap loads them into registers instead and hands each block's to the warp's other lanes through
  // SW_OFF: two blocks of NC values per warp (read as broadcasts; a shuffle per column held the block up)
  static constexpr int kRing = kSwap ? 0 : 6;
  static constexpr int RING_OFF = STG_OFF + STG_BYTES, RING_SLOT = 32 * EPI_WARPS * 8;
  static constexpr int BIAS_OFF = RING_OFF + kRing * RING_SLOT;   // each epilogue warp's bias values
  static constexpr int SW_OFF = BIAS_OFF;
  static constexpr int BAR_OFF = BIAS_OFF + (kSwap ? 2 : 1) * EPI_WARPS * NC * 4;
  static constexpr int NBAR = 2 * STAGES + 2 * ACCS;
  static constexpr int SMEM = 1024 + BAR_OFF + 8 * NBAR + 16;
  static_assert(PER_SM * (SMEM + 1024) <= 228 * 1024 && PER_SM * TMEM_COLS <= 512, "shared and tensor memory of an SM");
  static_assert(kPair || BN * 128 * 4 <= STAGES * STAGE_BYTES, "the split sums reuse the stages");
};

struct F8Params {
  const float* sa;     // activation scales: element (m, g) at m * sa_m + g * sa_k
  const float* sb;     // weight scales: element (n / 128, g) at (n / 128) * sb_n + g * sb_k
  int64_t sa_m, sa_k, sb_n, sb_k;
  int M, N, kb;
  int tiles_r, tiles_c, split;   // tiles of ROWS (A rows) and of BN (B rows); CTAs that share a tile's K blocks
  const void* bias;
  int bias_f32, bias_vec;   // its type; whether 8 values may be loaded at once
  void* out;
  int64_t ldo;
  int out_vec;         // rows of out may be written 16 bytes at a time
  int out_tma;         // bf16 rows are staged in shared memory and written by TMA (tmO)
};

VF4_DEV float bias_at(const F8Params& p, int n) {
  if (!p.bias || n >= p.N) return 0.f;
  return p.bias_f32 ? __ldg(static_cast<const float*>(p.bias) + n)
                    : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]);
}

// The bias of columns n0 .. n0 + 7 (0 past N).
VF4_DEV void bias8(const F8Params& p, int n0, float* y) {
  if (p.bias_vec && n0 + 8 <= p.N) {
    if (p.bias_f32) load8<float, true>(static_cast<const float*>(p.bias) + n0, 8, y);
    else load8<__nv_bfloat16, true>(static_cast<const __nv_bfloat16*>(p.bias) + n0, 8, y);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = bias_at(p, n0 + i);
  }
}

// Eight sums of one row of y, columns n0 .. n0 + 7, with one rounding to the output type.  A lane per row: without
// 16-byte rows every store of a warp writes a few bytes in each of 32 rows, which outlasts the products (4096 x 1001 x
// 1280, bf16: 49 us, with 1008 columns, which go out by TMA, 13; 512 x 21841 x 1024: 147 and 24).  fp32 rows always go
// out here (16400 x 5120 x 1280: 294 us, bf16 133).
template <bool kF32>
VF4_DEV void store8(const F8Params& p, int64_t m, int n0, const float* z) {
  if (m >= p.M || n0 >= p.N) return;
  if constexpr (kF32) {
    float* o = static_cast<float*>(p.out) + m * p.ldo + n0;
    if (p.out_vec && n0 + 8 <= p.N) {
      reinterpret_cast<float4*>(o)[0] = make_float4(z[0], z[1], z[2], z[3]);
      reinterpret_cast<float4*>(o)[1] = make_float4(z[4], z[5], z[6], z[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n0 + i < p.N) o[i] = z[i];
    }
  } else {
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + m * p.ldo + n0;
    if (p.out_vec && n0 + 8 <= p.N) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = bf16x2_round(f32x2_pack(z[2 * i], z[2 * i + 1]));
      *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n0 + i < p.N) o[i] = __float2bfloat16_rn(z[i]);
    }
  }
}

template <bool kF32>
VF4_DEV void store1(const F8Params& p, int m, int n, float y) {
  if (m >= p.M || n >= p.N) return;
  if constexpr (kF32) static_cast<float*>(p.out)[(int64_t)m * p.ldo + n] = y;
  else static_cast<__nv_bfloat16*>(p.out)[(int64_t)m * p.ldo + n] = __float2bfloat16_rn(y);
}

// 4 bytes global -> shared, or zeros; tracked by this thread's groups.
VF4_DEV void cp_async4(uint32_t dst, const float* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
VF4_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
VF4_DEV void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
VF4_DEV float2 ld_shared_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

VF4_DEV float ld_shared_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int BN, bool kSwap, bool kF32>
__global__ void __launch_bounds__(F8Cfg<BN, kSwap>::THREADS, F8Cfg<BN, kSwap>::PER_SM)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmO, const F8Params p) {
  using C = F8Cfg<BN, kSwap>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw0 = smem_u32(smem_raw);
  const uint32_t base = (raw0 + 1023u) & ~1023u;
  uint8_t* gb = smem_raw + (base - raw0);
  const uint32_t bar = base + C::BAR_OFF;
  auto full = [&](int i) { return bar + 8u * i; };
  auto empty = [&](int i) { return bar + 8u * (C::STAGES + i); };
  auto tfull = [&](int i) { return bar + 8u * (2 * C::STAGES + i); };
  auto tempty = [&](int i) { return bar + 8u * (2 * C::STAGES + C::ACCS + i); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gb + C::BAR_OFF + 8 * C::NBAR);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* err = &g_fp8_err;
  // kPair: rank in the pair; otherwise the rank among the CTAs that share a tile's K blocks
  const int rank = C::kPair || p.split > 1 ? (int)cluster_ctarank() : 0;

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(full(i), 1);
      mbar_init(empty(i), 1);
    }
    for (int i = 0; i < C::ACCS; ++i) {
      mbar_init(tfull(i), 1);
      mbar_init(tempty(i), C::EPI_WARPS * (C::kPair ? 2 : 1));
    }
    fence_mbar_init();
    tma_prefetch(&tmA);
    tma_prefetch(&tmB);
    if (p.out_tma) tma_prefetch(&tmO);
  }
  if (warp == 1) {
    if constexpr (C::kPair) {
      tmem_alloc_pair(smem_u32(tmem_slot), C::TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
      tmem_relinquish();
    }
  }
  fence_async_shared();
  tc_fence_before();
  if constexpr (C::kPair) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  // this CTA's run of K blocks, and its tiles (split > 1: one per cluster)
  const int k0 = C::kPair ? 0 : (int)((int64_t)p.kb * rank / p.split);
  const int k1 = C::kPair ? p.kb : (int)((int64_t)p.kb * (rank + 1) / p.split);
  const int tiles = p.tiles_r * p.tiles_c;
  const int share = C::kPair ? 2 : p.split;   // CTAs per tile
  const int first = blockIdx.x / share, step = gridDim.x / share;

  if (warp < C::EPI0) {
    if constexpr (C::kRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kControlRegs));
    // Both loops run as whole warps with one elected lane issuing: their addresses and descriptors then stay
    // warp-uniform.  Inside a one-lane branch each MMA's operands were moved into uniform registers one at a
    // time, and a block of four MMAs took 600 clocks to issue whatever its size (513 of 512 now).
    const bool elected = elect_one();
    if (warp == 0) {
      griddep_wait();
      int s = 0, it = 0;
      uint32_t ph = 1;   // an unused stage counts as released
      bool ok = true;
      for (int tile = first; tile < tiles && ok; tile += step) {
        const int tr = tile / p.tiles_c, tc = tile - tr * p.tiles_c;
        const int ya = tr * C::ROWS + (C::kPair ? rank * 128 : 0), yb = tc * BN + (C::kPair ? rank * 128 : 0);
        for (int kb = k0; kb < k1; ++kb, ++it) {
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(empty(s), ph, err, kDevErrTimeoutEmpty));
          if (!ok) break;
          const uint32_t st = base + s * C::STAGE_BYTES;
          if (elected) {
            if constexpr (C::kPair) {   // both CTAs' copies complete on the leader's barrier
              if (rank == 0) mbar_arrive_expect_tx(full(s), 2 * C::STAGE_BYTES);
              const uint32_t fb = mapa_shared(full(s), 0);
              tma_load_2d_pair(st, &tmA, kb * 128, ya, fb);
              tma_load_2d_pair(st + C::A_BYTES, &tmB, kb * 128, yb, fb);
            } else {
              mbar_arrive_expect_tx(full(s), C::STAGE_BYTES);
              tma_load_2d(st, &tmA, kb * 128, ya, full(s));
              tma_load_2d(st + C::A_BYTES, &tmB, kb * 128, yb, full(s));
            }
          }
          __syncwarp();
          if (++s == C::STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // no copy may still be writing shared memory when the CTA exits (a pair leaves together)
      if (!C::kPair || rank == 0)
        for (int i = it > C::STAGES ? it - C::STAGES : 0; i < it; ++i)
          mbar_wait(full(i % C::STAGES), (uint32_t)(i / C::STAGES) & 1u, err, kDevErrTimeoutFull);
      __syncwarp();
    } else if (warp == 1) {
      if (!C::kPair || rank == 0) {   // one CTA issues for the pair
        int s = 0, a = 0, it = 0;
        uint32_t ph = 0, pa = 1;
        bool ok = true;
        constexpr uint32_t idesc = idesc_f8_e4m3(BN, C::ROWS);
        const uint64_t ad0 = smem_desc(base, 16, 1024, 2), bd0 = smem_desc(base + C::A_BYTES, 16, 1024, 2);
        auto both = [&](uint32_t b_full, uint32_t b_free) {
          if constexpr (C::kPair)
            return mbar_wait_cluster(b_full, ph, err, kDevErrTimeoutFull) &&
                   mbar_wait_cluster(b_free, pa, err, kDevErrTimeoutTmem);
          else
            return mbar_wait(b_full, ph, err, kDevErrTimeoutFull) && mbar_wait(b_free, pa, err, kDevErrTimeoutTmem);
        };
        for (int tile = first; tile < tiles && ok; tile += step) {
          for (int kb = k0; kb < k1; ++kb, ++it) {
            ok = __all_sync(0xFFFFFFFFu, both(full(s), tempty(a)));
            if (!ok) break;
            tc_fence_after();
            if (elected) {
              const uint64_t ad = ad0 + (uint32_t)(s * (C::STAGE_BYTES >> 4)), bd = bd0 + (uint32_t)(s * (C::STAGE_BYTES >> 4));
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) {   // 32 bytes of K further: the descriptors' addresses count 16 bytes
                if constexpr (C::kPair) mma_f8f6f4_pair(tmem + a * BN, ad + 2 * kk, bd + 2 * kk, idesc, kk > 0 ? 1u : 0u);
                else mma_f8f6f4(tmem + a * BN, ad + 2 * kk, bd + 2 * kk, idesc, kk > 0 ? 1u : 0u);
              }
              if constexpr (C::kPair) {
                tc_commit_pair(empty(s), 3);
                tc_commit_pair(tfull(a), 3);
              } else {
                tc_commit(empty(s));
                tc_commit(tfull(a));
              }
            }
            __syncwarp();
            if (++s == C::STAGES) {
              s = 0;
              ph ^= 1u;
            }
            if (++a == C::ACCS) {
              a = 0;
              pa ^= 1u;
            }
          }
        }
        // the tensor core must be done with shared and tensor memory before the CTA leaves
        if (it > 0) mbar_wait(tfull((it - 1) % C::ACCS), (uint32_t)((it - 1) / C::ACCS) & 1u, err, kDevErrTimeoutDrain);
      }
      __syncwarp();
    }
  } else {
    if constexpr (C::kRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kEpiRegs));
    griddep_wait();   // the launch may have come before the operands' cast had ended (the barriers above did not need it)
    const int quad = warp & 3, half = (warp - C::EPI0) >> 2;
    const int r = quad * 32 + lane;                       // row of the tile, lane of tensor memory
    const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(half * C::NC);
    bool ok = true;
    // !kSwap: the scales of the K blocks ahead, copied by each thread for itself through shared memory.  They
    // have to be asked for that early: read two blocks ahead into registers they still cost the 16400 x 5120 x
    // 5120 product a third of its time (each block's column of scales is a line that L1 has not seen).
    uint32_t ring = 0;
    int f_tile = first, f_kb = k1;
    uint32_t f_dst = 0;
    const float *f_a = p.sa, *f_b = p.sb;
    bool f_row = false;
    auto fetch_ring = [&]() {
      if (f_kb == k1 && f_tile < tiles) {   // the first block of the next tile
        const int tr = f_tile / p.tiles_c, tc = f_tile - tr * p.tiles_c;
        const int row = tr * C::ROWS + (C::kPair ? rank * 128 : 0) + r;
        f_row = row < p.M;
        f_a = p.sa + (int64_t)(f_row ? row : 0) * p.sa_m + k0 * p.sa_k;
        f_b = p.sb + (int64_t)(min(tc * BN + half * C::NC, p.N - 1) >> 7) * p.sb_n + k0 * p.sb_k;
        f_kb = k0;
        f_tile += step;
      }
      if (f_kb < k1) {
        cp_async4(ring + f_dst, f_a, f_row);
        cp_async4(ring + f_dst + 4, f_b, true);
        f_a += p.sa_k;
        f_b += p.sb_k;
        ++f_kb;
      }
      cp_async_commit();   // also without a copy: the waits below count groups
      f_dst = f_dst == (uint32_t)((C::kRing - 1) * C::RING_SLOT) ? 0u : f_dst + C::RING_SLOT;
    };
    if constexpr (!kSwap) {
      ring = base + C::RING_OFF + (uint32_t)(threadIdx.x - 32 * C::EPI0) * 8u;
      for (int i = 0; i + 1 < C::kRing; ++i) fetch_ring();
    }
    uint32_t use = 0;
    int a = 0;
    uint32_t pa = 0;
    for (int tile = first; tile < tiles; tile += step) {
      const int tr = tile / p.tiles_c, tc = tile - tr * p.tiles_c;
      const int row0 = tr * C::ROWS + (C::kPair ? rank * 128 : 0) + quad * 32;   // first row of this warp
      const int row = row0 + lane, col0 = tc * BN + half * C::NC;
      // kSwap: one activation row's scale per lane, the weight's alike for all.  The values of the next kAhead - 1
      // blocks are on their way while kb is worked on, multiplied only when used.
      constexpr int kAhead = kSwap ? 6 : 3;
      [[maybe_unused]] float sw[kAhead], sx[kAhead];
      const bool have = kSwap && lane < C::NC && col0 + lane < p.M;
      const float* s_own = p.sa + (int64_t)(have ? col0 + lane : 0) * p.sa_m;
      const float* s_blk = p.sb + (int64_t)tr * p.sb_n;
      auto fetch = [&](int kb, int slot) {
        if (kb >= k1) return;
        sw[slot] = __ldg(s_blk + kb * p.sb_k);
        sx[slot] = have ? __ldg(s_own + kb * p.sa_k) : 0.f;
      };
      if constexpr (kSwap) __syncwarp();   // the last tile's scales have been read
      unsigned long long acc[C::NC / 2];
#pragma unroll
      for (int i = 0; i < C::NC / 2; ++i) acc[i] = 0ull;
      // this warp's NC bias values, NC / 32 per lane, asked for here and needed after the last block
      constexpr int BPL = C::NC >= 32 ? C::NC / 32 : 1;
      [[maybe_unused]] float bias[BPL];
      if (!kSwap && p.bias && p.split == 1) {
#pragma unroll
        for (int i = 0; i < BPL; ++i) bias[i] = bias_at(p, col0 + BPL * lane + i);
      }
      if constexpr (kSwap) {
#pragma unroll
        for (int u = 0; u + 1 < kAhead; ++u) fetch(k0 + u, u);
      }
      auto block = [&](int kb, int slot) {
        [[maybe_unused]] float s0 = 0.f;
        // kAhead is even, so neighbouring blocks use different halves; a half is written again after two __syncwarp
        [[maybe_unused]] float* sc = reinterpret_cast<float*>(gb + C::SW_OFF) + ((warp - C::EPI0) * 2 + (slot & 1)) * C::NC;
        if constexpr (kSwap) {
          fetch(kb + kAhead - 1, (slot + kAhead - 1) % kAhead);
          if (lane < C::NC) sc[lane] = sx[slot] * sw[slot];
          __syncwarp();
        } else {
          cp_async_wait<C::kRing - 2>();   // this block's pair, the oldest of the groups in flight
          const float2 q = ld_shared_f2(ring + use);
          use = use == (uint32_t)((C::kRing - 1) * C::RING_SLOT) ? 0u : use + C::RING_SLOT;
          s0 = q.x * q.y;
          fetch_ring();                    // into the slot read one block ago
        }
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(tfull(a), pa, err, kDevErrTimeoutTmem)))
          ok = false;   // the whole warp gives up together: the loads below are warp-wide
        if (!ok) return;
        tc_fence_after();
        constexpr int CH = C::CH;
        constexpr int BUF = C::BUF;
        uint32_t v[BUF][CH];
        auto load = [&](int c) {
          if constexpr (CH == 32) tmem_ld_32x32b_x32(lane_base + a * BN + CH * c, v[c % BUF]);
          else tmem_ld_32x32b_x16(lane_base + a * BN + CH * c, v[c % BUF]);
        };
        load(0);
#pragma unroll
        for (int c = 0; c < C::NC / CH; ++c) {
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < CH; i += 16) reg_fence16(&v[c % BUF][i]);
          if (c + 1 < C::NC / CH) {
            if (BUF > 1) load(c + 1);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (C::kPair) mbar_arrive_peer(mapa_shared(tempty(a), 0));
              else mbar_arrive(tempty(a));
            }
          }
#pragma unroll
          for (int i = 0; i < CH / 2; i += 2) {
            unsigned long long s2[2];
            if constexpr (!kSwap) {
              s2[0] = s2[1] = f32x2_pack(s0, s0);
            } else {
              const float4 q = *reinterpret_cast<const float4*>(sc + CH * c + 2 * i);
              s2[0] = f32x2_pack(q.x, q.y);
              s2[1] = f32x2_pack(q.z, q.w);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              unsigned long long& d = acc[CH / 2 * c + i + e];
              d = fma_f32x2(f32x2_pack(__uint_as_float(v[c % BUF][2 * (i + e)]), __uint_as_float(v[c % BUF][2 * (i + e) + 1])),
                            s2[e], d);
            }
          }
          if (BUF == 1 && c + 1 < C::NC / CH) load(c + 1);
        }
        if (++a == C::ACCS) {
          a = 0;
          pa ^= 1u;
        }
      };
      for (int kb = k0; kb < k1 && ok; kb += kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (kb + u < k1 && ok) block(kb + u, u);
      }
      if (!kSwap && p.bias && p.split == 1) {   // sums += bias, through shared memory (every lane needs all)
        float* bs = reinterpret_cast<float*>(gb + C::BIAS_OFF) + (warp - C::EPI0) * C::NC;
#pragma unroll
        for (int i = 0; i < BPL; ++i) bs[BPL * lane + i] = bias[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < C::NC / 4; ++i) {
          const float4 q = reinterpret_cast<const float4*>(bs)[i];
          acc[2 * i] = add_f32x2(acc[2 * i], f32x2_pack(q.x, q.y));
          acc[2 * i + 1] = add_f32x2(acc[2 * i + 1], f32x2_pack(q.z, q.w));
        }
      }
      if (!kSwap && !kF32 && p.out_tma) {
        // bf16: 64 columns of the warp's 32 rows at a time through shared memory (128-byte swizzle), one TMA
        // store each, so the warp is free for the next tile as soon as the sums are in shared memory
        uint8_t* stg = gb + C::STG_OFF + (warp - C::EPI0) * 4096;
#pragma unroll
        for (int c = 0; c < C::NC / 64; ++c) {
          if (lane == 0) bulk_wait_read();
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = bf16x2_round(acc[32 * c + 4 * j + i]);
            *reinterpret_cast<uint4*>(stg + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          fence_async_shared();
          __syncwarp();
          if (lane == 0 && col0 + 64 * c < p.N && row0 < p.M) {   // rows past M and columns past N are clipped
            tma_store_2d(&tmO, smem_u32(stg), col0 + 64 * c, row0);
            bulk_commit();
          }
        }
      } else if (p.split == 1) {
        float y[8];
        const float own = kSwap ? bias_at(p, row) : 0.f;
#pragma unroll
        for (int c = 0; c < C::NC / 8; ++c) {
#pragma unroll
          for (int i = 0; i < 4; ++i) f32x2_unpack(acc[4 * c + i], &y[2 * i], &y[2 * i + 1]);
          if constexpr (!kSwap) {
            store8<kF32>(p, row, col0 + 8 * c, y);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) store1<kF32>(p, col0 + 8 * c + i, row, y[i] + own);
          }
        }
      } else {
        // this CTA's sums, column by column, into the stages (every MMA that read them is done)
        float* red = reinterpret_cast<float*>(gb) + (half * C::NC) * 128 + r;
#pragma unroll
        for (int i = 0; i < C::NC / 2; ++i) {
          float y0, y1;
          f32x2_unpack(acc[i], &y0, &y1);
          red[(2 * i) * 128] = y0;
          red[(2 * i + 1) * 128] = y1;
        }
      }
    }
    if constexpr (!kSwap) cp_async_wait<0>();
    if (!kSwap && !kF32 && p.out_tma) {
      if (lane == 0) bulk_wait_all();
      __syncwarp();
    }
  }

  if (!C::kPair && p.split > 1) {
    __syncwarp();
    cluster_sync_all();
    // rank's share of the columns, summed over the ranks in their order.  The loads of two ranks (split is even)
    // are in flight together: one at a time, each waited for by its addition, they took longer than the MMAs
    auto add2 = [&](auto& y, int q, int c, int r) {
      constexpr int U = sizeof(y) / sizeof(float);
      const uint32_t at = (uint32_t)(c * 128 + r) * 4u;
      const uint32_t s0 = mapa_shared(base, (uint32_t)q) + at, s1 = mapa_shared(base, (uint32_t)q + 1) + at;
      float v0[U], v1[U];
#pragma unroll
      for (int i = 0; i < U; ++i) v0[i] = ld_shared_cluster(s0 + (uint32_t)i * 512u);
#pragma unroll
      for (int i = 0; i < U; ++i) v1[i] = ld_shared_cluster(s1 + (uint32_t)i * 512u);
#pragma unroll
      for (int i = 0; i < U; ++i) y[i] = (y[i] + v0[i]) + v1[i];
    };
    if (warp >= C::EPI0 && first < tiles) {
      const int tr = first / p.tiles_c, tc = first - tr * p.tiles_c;
      const int quad = warp & 3, half = (warp - C::EPI0) >> 2, r = quad * 32 + lane;
      const int per = BN / 8 / p.split;   // runs of 8 columns
      if constexpr (!kSwap) {
        for (int c = rank * per + half; c < (rank + 1) * per; c += C::EW) {
          float y[8];
          bias8(p, tc * BN + 8 * c, y);
          for (int q = 0; q < p.split; q += 2) add2(y, q, 8 * c, r);
          store8<kF32>(p, tr * 128 + r, tc * BN + 8 * c, y);
        }
      } else {
        constexpr int U = BN / 8;   // columns at a time: the share of one of 8 ranks
        const int cols = BN / p.split;
        const float bias = bias_at(p, tr * 128 + r);
        for (int c = rank * cols + half * U; c < (rank + 1) * cols; c += C::EW * U) {
          float y[U];
#pragma unroll
          for (int i = 0; i < U; ++i) y[i] = 0.f;
          for (int q = 0; q < p.split; q += 2) add2(y, q, c, r);
#pragma unroll
          for (int i = 0; i < U; ++i) store1<kF32>(p, tc * BN + c + i, tr * 128 + r, y[i] + bias);
        }
      }
    }
    __syncwarp();
    cluster_sync_all();   // no CTA leaves while another reads its shared memory
  }
  tc_fence_before();
  if constexpr (C::kPair) {
    __syncwarp();
    cluster_sync_all();   // the pair's MMAs read both CTAs' shared memory, and barriers are arrived on remotely
  } else {
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 1) {
    if constexpr (C::kPair) tmem_dealloc_pair(tmem, C::TMEM_COLS);
    else tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------------------
// Linear layer of one or two rows (a decoder's token, a class token): cast and product in one launch.  Bound by
// reading the weight once.  Every CTA casts the rows for itself into shared memory (decoded: code * scale, in
// the order in which the lanes read them), while its warps' first weights are on their way; then a warp takes
// two weight rows at a time, 512 columns (16 per lane) by 512.  The tensor core would pad the rows to 16 and
// needs a cast kernel before it and a reduction after it.
// ---------------------------------------------------------------------------------------
constexpr int kVecRows = 2, kVecChunks = 4, kVecWarps = 8;

struct F8Vec {
  const void* x;
  int64_t ldx;
  const uint8_t* b;
  int64_t ldb;
  int K, chunks;       // chunks of 512 columns
  int x_vec;           // x rows may be read 4 elements at a time
};

// Codes k .. k + 15 of a row (0 past K, whatever the row's padding holds).
VF4_DEV uint4 load_codes(const uint8_t* row, int k, int K) {
  if (k + 16 <= K) return __ldg(reinterpret_cast<const uint4*>(row + k));
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  for (int i = 0; k + i < K && i < 16; ++i) w[i >> 2] |= (uint32_t)__ldg(row + k + i) << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

VF4_DEV float2 e4m3x2_to_f32x2(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(two & 0xFFFFu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

template <typename T, int R>
__global__ void __launch_bounds__(kVecWarps * 32, 2) fp8_linear_rows_kernel(const F8Vec a, const F8Params p) {
  extern __shared__ __align__(16) float xs[];   // [R][chunk][4][32 lanes][4]: lane's columns 16 lane + 4 j ..
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wid = blockIdx.x * kVecWarps + warp, total = gridDim.x * kVecWarps;
  const int row_floats = a.chunks * 512;
  // two weight rows n and n + total, chunk by chunk, kDeep chunks on their way
  constexpr int kDeep = 2;
  uint4 w[kDeep][2];
  int fn = wid, fc = 0;
  auto fetch = [&](uint4* d) {
    if (fn >= p.N) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = fn + i * total;
      d[i] = r < p.N ? load_codes(a.b + (int64_t)r * a.ldb, fc * 512 + lane * 16, a.K) : make_uint4(0, 0, 0, 0);
    }
    if (++fc == a.chunks) {
      fc = 0;
      fn += 2 * total;
    }
  };
#pragma unroll
  for (int u = 0; u < kDeep; ++u) fetch(w[u]);
  // the cast: a warp per block of 128 columns, 4 per lane
  for (int i = warp; i < R * a.chunks * 4; i += kVecWarps) {
    const int m = i / (a.chunks * 4), g = i - m * (a.chunks * 4), k = g * 128 + lane * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (m < p.M && k < a.K) {
      const T* src = static_cast<const T*>(a.x) + m * a.ldx + k;
      if (a.x_vec && k + 4 <= a.K) {
        if constexpr (sizeof(T) == 2) {
          const uint2 u = __ldg(reinterpret_cast<const uint2*>(src));
          v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xFFFF0000u);
          v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xFFFF0000u);
        } else {
          const float4 u = __ldg(reinterpret_cast<const float4*>(src));
          v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < a.K) v[e] = (float)src[e];
      }
    }
    uint32_t top = max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3])));
#pragma unroll
    for (int o = 16; o; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    const Fp8Block q = fp8_block(top);
    const float2 lo = e4m3x2_to_f32x2(e4m3x2(fp8_quotient(v[0], q), fp8_quotient(v[1], q)));
    const float2 hi = e4m3x2_to_f32x2(e4m3x2(fp8_quotient(v[2], q), fp8_quotient(v[3], q)));
    const int in = (k & 511) >> 4, j = (k & 15) >> 2;   // the lane that will read these 4, and its piece
    *reinterpret_cast<float4*>(xs + m * row_floats + ((((k >> 9) * 4 + j) * 32 + in) << 2)) =
        make_float4(lo.x * q.scale, lo.y * q.scale, hi.x * q.scale, hi.y * q.scale);
  }
  __syncthreads();
  float acc[2][R];
  int n = wid, c = 0;
  while (n < p.N) {
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      if (n >= p.N) break;
      if (c == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int m = 0; m < R; ++m) acc[i][m] = 0.f;
      }
      const int g = min(c * 4 + (lane >> 3), p.kb - 1);   // this lane's block (past K its codes are 0)
      float4 x[R][4];
#pragma unroll
      for (int m = 0; m < R; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[m][j] = *reinterpret_cast<const float4*>(xs + m * row_floats + (((c * 4 + j) * 32 + lane) << 2));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float s = __ldg(p.sb + (int64_t)(min(n + i * total, p.N - 1) >> 7) * p.sb_n + g * p.sb_k);
        const uint32_t v[4] = {w[u][i].x, w[u][i].y, w[u][i].z, w[u][i].w};
        float d[R];
#pragma unroll
        for (int m = 0; m < R; ++m) d[m] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 lo = e4m3x2_to_f32x2(v[j]), hi = e4m3x2_to_f32x2(v[j] >> 16);
#pragma unroll
          for (int m = 0; m < R; ++m) {
            d[m] = fmaf(lo.x, x[m][j].x, d[m]);
            d[m] = fmaf(lo.y, x[m][j].y, d[m]);
            d[m] = fmaf(hi.x, x[m][j].z, d[m]);
            d[m] = fmaf(hi.y, x[m][j].w, d[m]);
          }
        }
#pragma unroll
        for (int m = 0; m < R; ++m) acc[i][m] = fmaf(d[m], s, acc[i][m]);
      }
      fetch(w[u]);
      if (++c == a.chunks) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int m = 0; m < R; ++m) {
#pragma unroll
            for (int o = 16; o; o >>= 1) acc[i][m] += __shfl_xor_sync(0xFFFFFFFFu, acc[i][m], o);
            if (lane == 0) store1<sizeof(T) == 4>(p, m, n + i * total, acc[i][m] + bias_at(p, n + i * total));
          }
        c = 0;
        n += 2 * total;
      }
    }
  }
}

// What the kernel above takes.  Measured, whole layer (cast and tensor-core product in brackets): 1 x 4096 x 1024
// 3.7 us (6.7), 1 x 5120 x 1280 5.9 (6.5), 1 x 4096 x 2048 5.4 (6.7), 2 x 4096 x 1024 4.9 (6.7); beyond that its decoding of
// the codes costs more than two launches: 1 x 16384 x 1024 7.6 (6.8), 1 x 1280 x 5120 9.7 (6.5), 2 x 16384 x 512 7.4 (5.8),
// 2 x 1280 x 2560 8.4 (6.1), and with four rows 4 x 4096 x 1024 7.3 (6.7).
static bool few_rows(int64_t M, int64_t N, int64_t K) {
  const int64_t chunks = M * ((K + 511) / 512);
  return M <= kVecRows && chunks <= kVecChunks && chunks * N <= 16384;
}

template <typename T>
static int launch_rows(const F8Vec& a, const F8Params& p, cudaStream_t s) {
  const size_t smem = (size_t)p.M * a.chunks * 2048;
  const int sms = num_sms();
  int64_t grid = ((int64_t)p.N + 2 * kVecWarps - 1) / (2 * kVecWarps);   // two rows per warp, if that fills the machine
  if (grid < sms) grid = ((int64_t)p.N + kVecWarps - 1) / kVecWarps;
  if (grid > 2 * sms) grid = 2 * sms;
  if (p.M == 1) fp8_linear_rows_kernel<T, 1><<<(unsigned)grid, kVecWarps * 32, smem, s>>>(a, p);
  else fp8_linear_rows_kernel<T, 2><<<(unsigned)grid, kVecWarps * 32, smem, s>>>(a, p);
  return launch_status("vf4_linear_fp8_block");
}

static int make_code_map(CUtensorMap* m, const void* ptr, int64_t rows, int64_t K, int64_t ld, int box_rows) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return fail(VF4_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {128u, (cuuint32_t)box_rows};
  cuuint32_t es[2] = {1u, 1u};
  CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, es,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(VF4_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return VF4_OK;
}

// Output map of the TMA-store epilogue: bf16 (M, N), boxes of 32 rows x 64 columns, 128-byte swizzle.
static int make_bf16_out_map(CUtensorMap* m, void* ptr, int64_t rows, int64_t cols, int64_t ld) {
  EncodeTiledFn enc = encode_tiled();
  if (!enc) return fail(VF4_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {64u, 32u};
  cuuint32_t es[2] = {1u, 1u};
  CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ptr, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(VF4_ERR_CUDA, "cuTensorMapEncodeTiled (output) failed (%d)", (int)r);
  return VF4_OK;
}

struct F8Operand {
  const uint8_t* ptr;
  int64_t rows, ld;
};

template <int BN, bool kSwap, bool kF32>
static int launch_fp8_gemm(F8Operand a, F8Operand b, int64_t K, F8Params p, cudaStream_t s) {
  using C = F8Cfg<BN, kSwap>;
  CUtensorMap ta, tb, to;
  memset(&to, 0, sizeof(to));
  if (int st = make_code_map(&ta, a.ptr, a.rows, K, a.ld, 128)) return st;
  if (int st = make_code_map(&tb, b.ptr, b.rows, K, b.ld, C::kPair ? 128 : BN)) return st;
  auto kern = fp8_gemm_kernel<BN, kSwap, kF32>;
  if (int st = smem_optin(kern, C::SMEM)) return st;
  if (C::kRegs) {   // the register split of the kernel relies on what its launch allocates
    static const int regs = [] {
      cudaFuncAttributes a;
      return cudaFuncGetAttributes(&a, fp8_gemm_kernel<BN, kSwap, kF32>) == cudaSuccess ? a.numRegs : 0;
    }();
    if (regs != C::kLaunchRegs) return fail(VF4_ERR_UNSUPPORTED, "vf4_gemm_fp8_block: built with %d registers", regs);
  }
  p.tiles_r = (int)((a.rows + C::ROWS - 1) / C::ROWS);
  p.tiles_c = (int)((b.rows + BN - 1) / BN);
  const int tiles = p.tiles_r * p.tiles_c, sms = num_sms();
  // Share a tile among up to 8 CTAs (the portable cluster size) while all are resident at once, if that takes enough
  // K blocks off each: joining the sums costs 1 us and more, a block 0.2 to 0.4.  16 x 1280 x 5120 takes 5.6 us shared
  // by 8 and 13.4 alone, 257 x 1280 x 5120 11.8 (4) and 19.4, 257 x 1280 x 2560 9.7 (4) and 11.5; but 257 x 1280 x
  // 1280 8.8 (4) and 7.8, 16 x 5120 x 1280 6.3 (2) and 5.9.  16 columns with two CTAs on most SMs already read
  // the weight at the memory's rate: 16 x 16384 x 4096 takes 15.1 us alone, 16.5 shared by 2.
  const int most = BN == 16 ? sms + sms / 4 : sms * C::PER_SM;
  p.split = 1;
  while (!C::kPair && p.split < 8 && tiles * p.split * 2 <= most && p.split * 2 <= p.kb) p.split *= 2;
  if (p.kb - p.kb / p.split < (kSwap ? 8 : 10)) p.split = 1;
  p.out_tma = !kSwap && !kF32 && p.split == 1 && p.out_vec;
  if (p.out_tma) {
    if (int st = make_bf16_out_map(&to, p.out, p.M, p.N, p.ldo)) return st;
  }
  cudaLaunchConfig_t cfg = {};
  const int pairs = sms / 2;
  cfg.gridDim = dim3((unsigned)(C::kPair ? 2 * (tiles < pairs ? tiles : pairs)
                                         : p.split > 1 ? tiles * p.split : (tiles < sms * C::PER_SM ? tiles : sms * C::PER_SM)));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute at[2] = {{}, early_launch()};
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)(C::kPair ? 2 : p.split);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  const bool cluster = C::kPair || p.split > 1;
  cfg.attrs = cluster ? at : at + 1;
  cfg.numAttrs = cluster ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, ta, tb, to, p) != cudaSuccess) return launch_status("vf4_gemm_fp8_block");
  return launch_status("vf4_gemm_fp8_block");
}

template <bool kF32>
static int dispatch_fp8_gemm(F8Operand x, F8Operand w, int64_t K, const F8Params& p, cudaStream_t s) {
  // Up to 64 rows: operands swapped, in the narrowest tile that holds them.  16 x 5120 x 1280 takes 6.0 us with 16
  // columns, 6.5 with 32, 9.8 unswapped; 32 x 5120 x 5120 10.3 with 32, 12.8 with 64, 15.5 unswapped; 64 x 5120 x 1280 7.1 with
  // 64 and 9.9 unswapped; 65 x 5120 x 5120 15.7 unswapped and 18.4 in two tiles of 64.
  if (x.rows <= 16) return launch_fp8_gemm<16, true, kF32>(w, x, K, p, s);
  if (x.rows <= 32) return launch_fp8_gemm<32, true, kF32>(w, x, K, p, s);
  if (x.rows <= 64) return launch_fp8_gemm<64, true, kF32>(w, x, K, p, s);
  // A round of 256 x 256 tiles (a pair of SMs each) takes 1.5 times a round of 128 x 128 tiles (one SM each): 2056 x
  // 1280 x 5120 is one round in 29 us against two in 37, 4112 x 5120 x 1280 five in 41 against nine in 48; but 1024 x 2048 x 2048
  // one in 15.8 against one in 10.8.
  const int64_t sms = num_sms(), pairs = sms / 2;
  const int64_t big = ((x.rows + 255) / 256 * ((w.rows + 255) / 256) + pairs - 1) / pairs;
  const int64_t small = ((x.rows + 127) / 128 * ((w.rows + 127) / 128) + sms - 1) / sms;
  if (3 * big <= 2 * small) return launch_fp8_gemm<256, false, kF32>(x, w, K, p, s);
  return launch_fp8_gemm<128, false, kF32>(x, w, K, p, s);
}

}  // namespace vf4

using namespace vf4;

extern "C" {

int vf4_cast_fp8_block(const void* x, int dtype, int64_t M, int64_t K, int64_t ld, int block_rows, uint8_t* codes,
                       int64_t ldc, float* scale, int64_t stride_m, int64_t stride_k, vf4_stream_t stream) {
  if (int st = check_device()) return st;
  if (M < 0 || K <= 0 || ld < K || (block_rows != 1 && block_rows != 128))
    return fail(VF4_ERR_ARG, "vf4_cast_fp8_block: bad sizes (M=%lld K=%lld ld=%lld block_rows=%d)", (long long)M,
                (long long)K, (long long)ld, block_rows);
  if (dtype != VF4_BF16 && dtype != VF4_F32) return fail(VF4_ERR_ARG, "vf4_cast_fp8_block: bad dtype %d", dtype);
  if (K > (1 << 20) || M > (1 << 30)) return fail(VF4_ERR_UNSUPPORTED, "vf4_cast_fp8_block: sizes too large");
  if (M == 0) return VF4_OK;
  if (!x || !codes || !scale) return fail(VF4_ERR_ARG, "vf4_cast_fp8_block: null pointer");
  if (!aligned16(codes) || ldc % 16 || ldc < K)
    return fail(VF4_ERR_ALIGN, "vf4_cast_fp8_block: code rows need 16-byte aligned starts of at least K bytes (ldc=%lld)",
                (long long)ldc);
  const int esz = dtype == VF4_BF16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(x) % esz) return fail(VF4_ERR_ALIGN, "vf4_cast_fp8_block: x is misaligned for its type");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool vec = aligned16(x) && K % 8 == 0 && ld * esz % 16 == 0;
  const int64_t kb = (K + 127) / 128;
  const auto* xb = static_cast<const __nv_bfloat16*>(x);
  const auto* xf = static_cast<const float*>(x);
  if (block_rows == 1) {
    const int64_t want = (M * kb + 15) / 16;   // 16 blocks per CTA and step
    const int64_t most = (int64_t)num_sms() * 5;   // the CTAs that are resident at once
    const unsigned grid = (unsigned)(want < most ? want : most);
    const int K32 = (int)K;
#define VF4_CAST_ROWS(T, X, V) \
  fp8_cast_rows_kernel<T, V, 2><<<grid, 256, 0, s>>>(X, M, K32, ld, codes, ldc, scale, stride_m, stride_k)
    if (dtype == VF4_BF16) {
      if (vec) VF4_CAST_ROWS(__nv_bfloat16, xb, true);
      else VF4_CAST_ROWS(__nv_bfloat16, xb, false);
    } else {
      if (vec) VF4_CAST_ROWS(float, xf, true);
      else VF4_CAST_ROWS(float, xf, false);
    }
#undef VF4_CAST_ROWS
  } else {
    const int64_t tiles = (M + 127) / 128 * kb;
    if (tiles > INT32_MAX) return fail(VF4_ERR_UNSUPPORTED, "vf4_cast_fp8_block: sizes too large");
    const unsigned grid = (unsigned)tiles;
    const int K32 = (int)K;
#define VF4_CAST_TILE(T, X, V) \
  fp8_cast_tile_kernel<T, V><<<grid, 256, 0, s>>>(X, M, K32, ld, codes, ldc, scale, stride_m, stride_k)
    if (dtype == VF4_BF16) {
      if (vec) VF4_CAST_TILE(__nv_bfloat16, xb, true);
      else VF4_CAST_TILE(__nv_bfloat16, xb, false);
    } else {
      if (vec) VF4_CAST_TILE(float, xf, true);
      else VF4_CAST_TILE(float, xf, false);
    }
#undef VF4_CAST_TILE
  }
  return launch_status("vf4_cast_fp8_block");
}

int vf4_gemm_fp8_block(const uint8_t* a, int64_t lda, const float* a_scale, int64_t as_m, int64_t as_k,
                       const uint8_t* b, int64_t ldb, const float* b_scale, int64_t bs_n, int64_t bs_k, int64_t M,
                       int64_t N, int64_t K, const void* bias, int bias_dtype, void* out, int64_t ldo, int out_dtype,
                       vf4_stream_t stream) {
  if (int st = check_device()) return st;
  if (M < 0 || N <= 0 || K <= 0 || ldo < N)
    return fail(VF4_ERR_ARG, "vf4_gemm_fp8_block: bad sizes M=%lld N=%lld K=%lld ldo=%lld", (long long)M, (long long)N,
                (long long)K, (long long)ldo);
  if (M > (1 << 30) || N > (1 << 24) || K > (1 << 20) || (M + 127) / 128 * ((N + 127) / 128) > INT32_MAX)
    return fail(VF4_ERR_UNSUPPORTED, "vf4_gemm_fp8_block: sizes too large");
  if ((out_dtype != VF4_BF16 && out_dtype != VF4_F32) || (bias && bias_dtype != VF4_BF16 && bias_dtype != VF4_F32))
    return fail(VF4_ERR_ARG, "vf4_gemm_fp8_block: bad dtype");
  if (M == 0) return VF4_OK;
  if (!a || !b || !a_scale || !b_scale || !out) return fail(VF4_ERR_ARG, "vf4_gemm_fp8_block: null operand");
  if (!aligned16(a) || !aligned16(b) || lda % 16 || ldb % 16 || lda < K || ldb < K)
    return fail(VF4_ERR_ALIGN, "vf4_gemm_fp8_block: code rows need 16-byte aligned starts of at least K bytes "
                "(lda=%lld ldb=%lld)", (long long)lda, (long long)ldb);
  const int esz = out_dtype == VF4_BF16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(out) % esz || reinterpret_cast<uintptr_t>(a_scale) % 4 ||
      reinterpret_cast<uintptr_t>(b_scale) % 4 || (bias && reinterpret_cast<uintptr_t>(bias) % (bias_dtype == VF4_BF16 ? 2 : 4)))
    return fail(VF4_ERR_ALIGN, "vf4_gemm_fp8_block: out, scales or bias misaligned for their types");
  F8Params p{};
  p.sa = a_scale;
  p.sb = b_scale;
  p.sa_m = as_m;
  p.sa_k = as_k;
  p.sb_n = bs_n;
  p.sb_k = bs_k;
  p.M = (int)M;
  p.N = (int)N;
  p.kb = (int)((K + 127) / 128);
  p.bias = bias;
  p.bias_f32 = bias_dtype == VF4_F32;
  p.bias_vec = bias && aligned16(bias);   // (no bias: bias_at gives zeros)
  p.out = out;
  p.ldo = ldo;
  p.out_vec = aligned16(out) && ldo * esz % 16 == 0;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const F8Operand x{a, M, lda}, w{b, N, ldb};
  return out_dtype == VF4_F32 ? dispatch_fp8_gemm<true>(x, w, K, p, s) : dispatch_fp8_gemm<false>(x, w, K, p, s);
}

// workspace of vf4_linear_fp8_block: the rows' codes, then their scales, column block by column block
int64_t vf4_linear_fp8_block_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > (1 << 30) || N > (1 << 24) || K > (1 << 20) || few_rows(M, N, K)) return 0;
  return M * ((K + 15) / 16 * 16) + M * ((K + 127) / 128) * 4;
}

int vf4_linear_fp8_block(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const uint8_t* w, int64_t ldw,
                         const float* w_scale, int64_t ws_n, int64_t ws_k, int64_t N, const void* bias, int bias_dtype,
                         void* out, int64_t ldo, void* workspace, int64_t workspace_bytes, vf4_stream_t stream) {
  if (int st = check_device()) return st;
  const int64_t need = vf4_linear_fp8_block_workspace_size(M, N, K);
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return fail(VF4_ERR_ARG, "vf4_linear_fp8_block: %lld bytes of 16-byte aligned workspace needed, got %lld", (long long)need,
                (long long)workspace_bytes);
  if (M > 0 && N > 0 && K > 0 && few_rows(M, N, K)) {
    if (ldx < K || ldo < N)
      return fail(VF4_ERR_ARG, "vf4_linear_fp8_block: bad sizes M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
    if ((dtype != VF4_BF16 && dtype != VF4_F32) || (bias && bias_dtype != VF4_BF16 && bias_dtype != VF4_F32))
      return fail(VF4_ERR_ARG, "vf4_linear_fp8_block: bad dtype");
    if (!x || !w || !w_scale || !out) return fail(VF4_ERR_ARG, "vf4_linear_fp8_block: null operand");
    const int esz = dtype == VF4_BF16 ? 2 : 4;
    if (!aligned16(w) || ldw % 16 || ldw < K)
      return fail(VF4_ERR_ALIGN, "vf4_linear_fp8_block: code rows need 16-byte aligned starts of at least K bytes (ldw=%lld)", (long long)ldw);
    if (reinterpret_cast<uintptr_t>(x) % esz || reinterpret_cast<uintptr_t>(out) % esz || reinterpret_cast<uintptr_t>(w_scale) % 4 ||
        (bias && reinterpret_cast<uintptr_t>(bias) % (bias_dtype == VF4_BF16 ? 2 : 4)))
      return fail(VF4_ERR_ALIGN, "vf4_linear_fp8_block: a pointer is misaligned for its type");
    F8Vec a{x, ldx, w, ldw, (int)K, (int)((K + 511) / 512), reinterpret_cast<uintptr_t>(x) % (4 * esz) == 0 && (M == 1 || ldx % 4 == 0)};
    F8Params p{};
    p.sb = w_scale;
    p.sb_n = ws_n;
    p.sb_k = ws_k;
    p.M = (int)M;
    p.N = (int)N;
    p.kb = (int)((K + 127) / 128);
    p.bias = bias;
    p.bias_f32 = bias_dtype == VF4_F32;
    p.out = out;
    p.ldo = ldo;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return dtype == VF4_BF16 ? launch_rows<__nv_bfloat16>(a, p, s) : launch_rows<float>(a, p, s);
  }
  const int64_t ldc = (K + 15) / 16 * 16;
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  float* scale = reinterpret_cast<float*>(codes + M * ldc);
  if (int st = vf4_cast_fp8_block(x, dtype, M, K, ldx, 1, codes, ldc, scale, 1, M, stream)) return st;
  return vf4_gemm_fp8_block(codes, ldc, scale, 1, M, w, ldw, w_scale, ws_n, ws_k, M, N, K, bias, bias_dtype, out, ldo,
                            dtype, stream);
}

}  // extern "C"
