// The e4m3 linear: y = act(x w^T + bias) of rows and weights held as e4m3 with one
// power-of-two scale for each row and 128 columns of the reduction (fp8.cuh):
//   y[m][n] = sum_b 2^(ex[m][b] + ew[n][b]) sum_{k in b} qx[m][k] qw[n][k] + bias[n].
//
// The scales are applied by the tensor core (tcgen05.mma kind::mxf8f6f4 with ue8m0 block
// scales): the instruction scales every 32 products, and the four instructions of a block
// of 128 are given the same scale byte, so the accumulator in tensor memory holds the
// finished sum and no per-block rescale runs on the CUDA cores.
//
// Roles (640 threads, persistent, one CTA or one CTA pair per tile at a time; registers
// move from the first four warps to the epilogue's, setmaxnreg):
//   warp 0     TMA: per k-block of 128 bytes the x tile [128][128 B] and the w tile
//              (128B swizzle) into a ring; with every fourth k-block the scale tiles (512
//              bytes for 128 rows of four blocks, fp8_scale_offset's order);
//   warp 1     one thread copies new scale tiles into tensor memory (tcgen05.cp, 32 lanes
//              x 4 columns, one word = a row's four blocks) and issues four MMAs (K = 32)
//              a k-block, selecting the block's byte by the descriptor's scale ids;
//   warps 4-19 epilogue: tensor memory -> registers (64 columns a thread, row = lane) ->
//              bias, activation, quantisation -> 64-byte row pieces in a swizzled staging
//              buffer, stored (or, onto the residual, added) by TMA: the load-store unit,
//              73 % busy with the pieces' reads and stores when the warps made them, only
//              writes the buffer. Four warps an SM sub-partition hide each other's
//              latencies: eight warps of 128 columns took a quarter longer (M = 87680,
//              K = 1024, N = 4096 with GELU to f16).
//
// Bound: long reductions by the chip's power (8192 x 8192 x 8192: 440 us or 2.5 PFLOP/s, the
// MMAs at 92 % of their cycles but at 1.1 GHz), short ones by the MMAs (K = 1024: 4096 cycles a
// 256 x 256 tile) and the handover of a pair's one accumulator to the epilogue and back, about
// 1600 cycles: M = 87680, N = 4096 takes 315 us (2.3 PFLOP/s), M = 21920 85; K = 4096, N = 1024
// 74. With GELU the epilogue's own instructions (17 a value, two of them MUFU) are as long as
// the MMAs: 101 us at M = 21920, 104 quantised, 376 at M = 87680. A ring of five stages: four
// and six measured the same.
// Every wait is bounded (ptx.cuh); on a timeout the kernel records a status and exits.
#include <algorithm>
#include <atomic>
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "act.cuh"
#include "da3b.h"
#include "fp8.cuh"
#include "fp8.h"
#include "gemm.h"
#include "launch.h"
#include "ops.h"
#include "ptx.cuh"

namespace da3b {

namespace {

constexpr int kThreads = 640;
// Launched at 96 registers a thread (61 440 in all): the first warpgroup gives back down to
// 40, the epilogue's four warpgroups take 104.
constexpr int kRegsLaunch = 96, kRegsCtl = 40, kRegsEpi = 104;
static_assert(128 * kRegsCtl + 512 * kRegsEpi <= kThreads * kRegsLaunch, "register split exceeds the launch");
constexpr int kEpiWarps = 16;
constexpr int kStageOut = 2048;     // a warp's staging buffer, [32 rows][64 B], 64B swizzle
constexpr int kEpiTab = 3 * 256;    // a warp's bias and scale of 64 columns, 32 maxima (x 2)
constexpr int kSfBuffers = 8;  // scale buffers in tensor memory

// CG = 1: a CTA computes 128 x 128, two accumulators, the two halves of the epilogue warps
// take alternate tiles. CG = 2: a CTA pair computes 256 x 256 (128 x 256 in each CTA's
// tensor memory, half of the w tile in each CTA's ring), one accumulator that all epilogue
// warps read at once: the scales need tensor memory too, so a second 256-column accumulator
// does not fit.
template <int CG>
struct Cfg {
  static constexpr int kBN = 128 * CG;
  static constexpr int kABytes = 128 * 128;
  static constexpr int kBBytes = 128 * 128;
  static constexpr int kSfATiles = 1, kSfBTiles = kBN / 128;
  static constexpr int kSfBytes = 512 * (kSfATiles + kSfBTiles);
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = 5;
  static constexpr int kAcc = CG == 2 ? 1 : 2;
  static constexpr int kSfCols = 4 * (kSfATiles + kSfBTiles);
  static constexpr uint32_t kColSf = kAcc * kBN;
  static constexpr int kEpiBytes = kEpiWarps * (kStageOut + kEpiTab);
  static constexpr int kSmem = 1024 + kStages * (kStageBytes + kSfBytes) + kEpiBytes + 256;
  static_assert(kColSf + kSfBuffers * kSfCols <= 512, "tensor memory");
  // A scale buffer is reused kSfBuffers groups later, and a k-block's MMAs start only when
  // those of the k-block kStages before it are complete, so its readers are done.
  static_assert(kSfBuffers >= kStages, "scale buffers");
};

// Instruction descriptor of kind::mxf8f6f4: e4m3 x e4m3, ue8m0 scales, both operands
// K-major; sf = which byte of the scale words.
__host__ __device__ constexpr uint32_t idesc_mxf8(int M, int N, int sf) {
  return (static_cast<uint32_t>(sf) << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(M >> 4) << 24) | (static_cast<uint32_t>(sf) << 29);
}

template <int CG>
__device__ __forceinline__ void umma_mxf8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate) {
  if (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// One 512-byte scale tile from shared memory to 32 lanes x 4 columns, repeated in the four
// lane quarters. The source is 32 rows of 16 bytes: no swizzle, 128 bytes between groups of
// eight rows.
template <int CG>
__device__ __forceinline__ void copy_sf(uint32_t tmem, uint32_t saddr) {
  uint64_t d = static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(1) << 16;
  d |= static_cast<uint64_t>(128 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  if (CG == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
  else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}

// Erf-form GELU v Phi(v) of eight values, Phi(v) = 1 / (1 + 2^(-v Q(v^2))): Q is a
// degree-6 polynomial fitted (Lawson-weighted least squares towards the minimax) to the
// logit of the normal distribution function on |v| <= 6 so that |v Phi(v)| is off by at most
// 6.8e-8; beyond 6, v^2 is held at 36 and Phi is 0 or 1 to 1e-9. Ten multiply-adds and two
// MUFU operations a value; the four pairs run side by side, because a chain of about
// fifteen dependent operations a value otherwise leaves the pipes idle (the M = 87680,
// K = 1024, N = 4096 product with GELU took 1.7 times as long with one chain at a time). One
// reciprocal for two values (of the product of their denominators) was no faster.
__device__ __forceinline__ void gelu8(float* v) {
  float2 x[4], q[4];
  const float2 one = make_float2(1.f, 1.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 w = make_float2(v[2 * i], v[2 * i + 1]);
    x[i] = __fmul2_rn(w, w);
    x[i] = make_float2(fminf(x[i].x, 36.f), fminf(x[i].y, 36.f));
  }
  auto step = [&](float c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = __ffma2_rn(q[i], x[i], make_float2(c, c));
  };
#pragma unroll
  for (int i = 0; i < 4; ++i)
    q[i] = __ffma2_rn(make_float2(-5.209905840e-09f, -5.209905840e-09f), x[i], make_float2(3.850448707e-07f, 3.850448707e-07f));
  step(-1.145242732e-05f);
  step(1.593893976e-04f);
  step(9.559298633e-05f);
  step(-0.1048385799f);
  step(-2.302207232f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = __fmul2_rn(q[i], make_float2(v[2 * i], v[2 * i + 1]));
    const float2 d = __fadd2_rn(make_float2(ex2_approx(u.x), ex2_approx(u.y)), one);
    float rx, ry;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rx) : "f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(ry) : "f"(d.y));
    v[2 * i] *= rx;
    v[2 * i + 1] *= ry;
  }
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A warp's [32 rows][64 B] piece of the output: lane = row holds 16 words; rows [m0, m0 +
// 32), columns from n0 on. Into the warp's staging buffer (16-byte chunks XOR-swizzled by
// row, the 64B swizzle), then out by TMA, which clips it at the last row, and at the last
// column where that ends a 16-byte chunk (it writes whole chunks). Another last piece, and an
// output whose rows are not 16-byte aligned, is written from the buffer element by element.
// ESZ: bytes an element; RESID: out += value (f32).
template <int ESZ, bool RESID>
__device__ __forceinline__ void store_piece(const Fp8Linear& a, const CUtensorMap* map, uint8_t* stg,
                                            const uint32_t (&words)[16], int m0, int n0, bool tma, int lane) {
  if (n0 >= a.N) return;
  if (tma) {
    if (lane == 0) bulk_wait_read<0>();  // the last piece has left the buffer
    __syncwarp();
    tma = n0 + 64 / ESZ <= a.N || a.N % (16 / ESZ) == 0;
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<uint4*>(stg + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(words[4 * c], words[4 * c + 1], words[4 * c + 2], words[4 * c + 3]);
  if (tma) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (RESID) tma_reduce_add_2d(map, stg, n0, m0);
      else tma_store_2d(map, stg, n0, m0);
      bulk_commit();
    }
    return;
  }
  __syncwarp();
  // 32 consecutive elements a store
  const size_t pitch = static_cast<size_t>(a.ldo) * ESZ;
  const int rows = min(32, a.M - m0);
  uint8_t* out = static_cast<uint8_t*>(a.out) + m0 * pitch;
#pragma unroll 4
  for (int row = 0; row < rows; ++row) {
#pragma unroll
    for (int e = lane; e < 64 / ESZ; e += 32) {
      const int ne = n0 + e, b = e * ESZ;
      if (ne >= a.N) continue;
      const uint8_t* src = stg + row * 64 + (((b >> 4) ^ ((row >> 1) & 3)) << 4) + (b & 15);
      uint8_t* o = out + row * pitch + static_cast<size_t>(ne) * ESZ;
      if (ESZ == 4) {
        const float v = *reinterpret_cast<const float*>(src);
        *reinterpret_cast<float*>(o) = RESID ? *reinterpret_cast<const float*>(o) + v : v;
      } else if (ESZ == 2) {
        *reinterpret_cast<uint16_t*>(o) = *reinterpret_cast<const uint16_t*>(src);
      } else {
        *o = *src;
      }
    }
  }
  __syncwarp();
}

// Epilogue of a warp's 32 rows x 64 columns held as v (lane = row m0 + lane, column n0 + i).
// ctab: the warp's copies of bias and scale for these columns, [2][64], and the row maxima
// it shares with the warp that has the other 64 columns of the block, [2][32]: `other` is
// that warp's table, `pair` the barrier of the two, `uses` its phases so far. False if a wait
// ran out.
__device__ __forceinline__ bool epilogue64(const Fp8Linear& a, const CUtensorMap* map, float (&v)[64], int m0, int n0,
                                           uint8_t* stg, float* ctab, const float* other, uint64_t* pair, uint32_t& uses,
                                           bool tma, int lane, int* status) {
#pragma unroll
  for (int i = 0; i < 64; i += 4) {
    const float4 b = *reinterpret_cast<const float4*>(ctab + i);
    v[i] += b.x;
    v[i + 1] += b.y;
    v[i + 2] += b.z;
    v[i + 3] += b.w;
  }
  if (a.act == kActRelu) {
#pragma unroll
    for (int i = 0; i < 64; ++i) asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(v[i]));  // NaN stays NaN
  } else if (a.act != kActNone) {
#pragma unroll
    for (int i = 0; i < 64; i += 8) gelu8(v + i);
  }
  uint32_t words[16];
  if (a.kind == kFp8OutF16 || a.kind == kFp8OutBF16) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if (a.kind == kFp8OutF16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) words[i] = pack_f16(v[32 * p + 2 * i], v[32 * p + 2 * i + 1]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) words[i] = pack_bf16(v[32 * p + 2 * i], v[32 * p + 2 * i + 1]);
      }
      store_piece<2, false>(a, map, stg, words, m0, n0 + 32 * p, tma, lane);
    }
  } else if (a.kind == kFp8OutQ) {
    // this warp's 64 columns and its partner's are one block of the output's scales;
    // columns past N are zero (w has no rows there, and their bias is zero). Infinities are
    // looked for once the maximum is known: both warps of a pair then see one, and do it again.
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) amax = fmaxf(amax, fabsf(v[i]));
    auto swap = [&]() -> bool {
      const uint32_t flip = uses++ & 1;
      ctab[128 + 32 * flip + lane] = amax;
      __syncwarp();
      if (lane == 0) mbar_arrive(pair);
      if (!mbar_wait_warp(pair, flip, status, kStatusTimeoutAccum)) return false;
      amax = fmaxf(amax, other[128 + 32 * flip + lane]);
      return true;
    };
    if (!swap()) return false;
    if (__any_sync(0xffffffffu, amax > kFltMax)) {
      amax = 0.f;
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        amax = fmaxf(amax, finite_abs(v[i]));
        v[i] = fp8_nan_if_inf(v[i]);
      }
      if (!swap()) return false;
    }
    const uint32_t byte = fp8_scale_byte(amax);
    const float inv = fp8_inv_scale(byte);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      words[i] = fp8_pack4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv, v[4 * i + 3] * inv);
    if (m0 + lane < a.M && (n0 & 127) == 0)
      a.out_scales[fp8_scale_offset(m0 + lane, n0 >> 7, (a.M + 127) / 128)] = static_cast<uint8_t>(byte);
    store_piece<1, false>(a, map, stg, words, m0, n0, tma, lane);
  } else {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      if (a.kind == kFp8OutResid) {
#pragma unroll
        for (int i = 0; i < 16; ++i) words[i] = __float_as_uint(v[16 * p + i] * ctab[64 + 16 * p + i]);
        store_piece<4, true>(a, map, stg, words, m0, n0 + 16 * p, tma, lane);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) words[i] = __float_as_uint(v[16 * p + i]);
        store_piece<4, false>(a, map, stg, words, m0, n0 + 16 * p, tma, lane);
      }
    }
  }
  return true;
}

template <int CG>
__global__ void __launch_bounds__(kThreads, 1)
    k_fp8_gemm(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
               const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
               const __grid_constant__ CUtensorMap tmC, const __grid_constant__ Fp8Linear a, int tma, int* status) {
  using C = Cfg<CG>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + C::kStages * C::kABytes;
  uint8_t* sSf = sB + C::kStages * C::kBBytes;
  uint8_t* sEpi = sSf + C::kStages * C::kSfBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sEpi + C::kEpiBytes);
  uint64_t* empty = full + C::kStages;
  uint64_t* tfull = empty + C::kStages;   // [kAcc] accumulator complete
  uint64_t* tempty = tfull + C::kAcc;     // [kAcc] accumulator read by the epilogue
  uint64_t* pairs = tempty + C::kAcc;     // [8] row maxima of both warps of a block written
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pairs + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0;
  const int unit = static_cast<int>(blockIdx.x) / CG, units = static_cast<int>(gridDim.x) / CG;
  const int m_tiles = (a.M + 127) / 128, n_tiles = (a.N + C::kBN - 1) / C::kBN;
  const int num_tiles = (m_tiles + CG - 1) / CG * n_tiles;
  const int num_kb = (a.K + 127) / 128;
  const int row_tiles_n = (a.N + 127) / 128;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < C::kAcc; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], CG * kEpiWarps / C::kAcc);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&pairs[i], 2);
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmSA);
    prefetch_tmap(&tmSB);
  }
  if (warp == 1) {
    if (CG == 2) tmem_alloc2(tmem_slot, 512);
    else tmem_alloc(tmem_slot, 512);
  }
  tc_fence_before();
  if (CG == 2) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsCtl));
  // Producer and issuer loops run in the whole warp and one elected lane issues: addresses and
  // descriptors then stay in uniform registers, where the instructions want them. With one
  // lane in the loops every operand was moved there one by one, and that set the pace (M =
  // 87680, K = 1024, N = 4096: 343 us against 315, 8192 x 8192 x 8192: 484 against 440).
  if (warp == 0) {
    const bool one = elect_one();
    int stage = 0;
    uint32_t phase = 0, loads = 0;
    bool ok = true;
    for (int t = unit; t < num_tiles && ok; t += units) {
      const int mt = t / n_tiles * CG + static_cast<int>(rank), nt = t % n_tiles;
      const int n0 = nt * C::kBN + static_cast<int>(rank) * 128;
      for (int kb = 0; kb < num_kb; ++kb) {
        ok = mbar_wait_warp(&empty[stage], phase ^ 1u, status, kStatusTimeoutEmpty);
        if (!ok) break;
        ++loads;
        const bool sf = (kb & 3) == 0;
        uint8_t* da = sA + stage * C::kABytes;
        uint8_t* db = sB + stage * C::kBBytes;
        uint8_t* ds = sSf + stage * C::kSfBytes;
        if (one) {
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], CG * (C::kStageBytes + (sf ? C::kSfBytes : 0)));
          if (CG == 2) {
            const uint32_t fb = mapa_shared(smem_u32(&full[stage]), 0);
            tma2_load_2d(da, &tmA, fb, kb * 128, mt * 128);
            tma2_load_2d(db, &tmB, fb, kb * 128, n0);
            if (sf) {
              tma2_load_2d(ds, &tmSA, fb, 0, (kb >> 2) * m_tiles + mt);
              tma2_load_2d(ds + 512, &tmSB, fb, 0, (kb >> 2) * row_tiles_n + nt * C::kSfBTiles);
            }
          } else {
            tma_load_2d(da, &tmA, &full[stage], kb * 128, mt * 128);
            tma_load_2d(db, &tmB, &full[stage], kb * 128, n0);
            if (sf) {
              tma_load_2d(ds, &tmSA, &full[stage], 0, (kb >> 2) * m_tiles + mt);
              tma_load_2d(ds + 512, &tmSB, &full[stage], 0, (kb >> 2) * row_tiles_n + nt);
            }
          }
        }
        __syncwarp();
        if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok && rank == 0 && lane == 0) drain(full, C::kStages, loads, status);
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      const bool one = elect_one();
      const uint64_t ad0 = umma_desc_sw128(smem_u32(sA)), bd0 = umma_desc_sw128(smem_u32(sB));
      int stage = 0, it = 0;
      uint32_t phase = 0, group = 0;
      bool ok = true;
      for (int t = unit; t < num_tiles && ok; t += units, ++it) {
        const int acc = it % C::kAcc;
        ok = mbar_wait_warp(&tempty[acc], ((it / C::kAcc) & 1) ^ 1u, status, kStatusTimeoutAccumFree);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * C::kBN;
        uint32_t sf = 0;
        for (int kb = 0; kb < num_kb; ++kb) {
          ok = mbar_wait_warp(&full[stage], phase, status, kStatusTimeoutFull);
          if (!ok) break;
          tc_fence_after();
          if ((kb & 3) == 0) {
            sf = tmem + C::kColSf + (group++ % kSfBuffers) * C::kSfCols;
            const uint32_t ds = smem_u32(sSf + stage * C::kSfBytes);
            if (one) {
#pragma unroll
              for (int i = 0; i < C::kSfATiles + C::kSfBTiles; ++i) copy_sf<CG>(sf + 4 * i, ds + 512 * i);
            }
          }
          const uint64_t ad = ad0 + stage * (C::kABytes >> 4), bd = bd0 + stage * (C::kBBytes >> 4);
          const uint32_t id = idesc_mxf8(128 * CG, C::kBN, 0) | (static_cast<uint32_t>(kb & 3) * ((1u << 4) | (1u << 29)));
          if (one) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_mxf8<CG>(d, ad + 2 * k, bd + 2 * k, id, sf, sf + 4, (kb > 0 || k > 0) ? 1u : 0u);
            if (CG == 2) umma2_commit_mc(&empty[stage], 0x3);
            else umma_commit(&empty[stage]);
          }
          __syncwarp();
          if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
        }
        if (ok && one) {
          if (CG == 2) umma2_commit_mc(&tfull[acc], 0x3);
          else umma_commit(&tfull[acc]);
        }
        __syncwarp();
      }
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    const int q = warp & 3, part = (warp - 4) >> 2;  // lane quarter, 64-column part of the tile
    const int cols = (C::kAcc == 1 ? part : part & 1) * 64;
    uint8_t* stg = sEpi + (warp - 4) * kStageOut;
    uint8_t* tabs = sEpi + kEpiWarps * kStageOut;
    float* ctab = reinterpret_cast<float*>(tabs + (warp - 4) * kEpiTab);
    // the warp with the other half of a 128-column block: the next or last part
    const float* other = reinterpret_cast<const float*>(tabs + ((warp - 4) ^ 4) * kEpiTab);
    uint64_t* pair = &pairs[q + 4 * (part >> 1)];
    uint32_t uses = 0;
    int it = 0;
    for (int t = unit; t < num_tiles; t += units, ++it) {
      const int acc = it % C::kAcc;
      if (C::kAcc == 2 && acc != part >> 1) continue;  // the halves take alternate tiles
      const int mt = t / n_tiles * CG + static_cast<int>(rank), nt = t % n_tiles;
      const int m0 = mt * 128 + q * 32, n0 = nt * C::kBN + cols;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n = n0 + lane + 32 * i;
        ctab[lane + 32 * i] = a.bias && n < a.N ? a.bias[n] : 0.f;
        ctab[64 + lane + 32 * i] = a.scale && n < a.N ? a.scale[n] : 1.f;
      }
      __syncwarp();
      if (!mbar_wait_warp(&tfull[acc], (it / C::kAcc) & 1, status, kStatusTimeoutAccum)) break;
      tc_fence_after();
      const uint32_t src = tmem + (static_cast<uint32_t>(q * 32) << 16) + acc * C::kBN + cols;
      float v[64];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t r[32];
        tmem_ld32(src + 32 * i, r);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[32 * i + j] = __uint_as_float(r[j]);
      }
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      // the values are in registers: the next tile's MMAs may start
      if (lane == 0) {
        if (CG == 2) mbar_arrive_remote_relaxed(mapa_shared(smem_u32(&tempty[acc]), 0));
        else mbar_arrive(&tempty[acc]);
      }
      // whole 128-column blocks are in or out together, so both warps of a pair come here
      if (m0 < a.M && (n0 & ~127) < a.N &&
          !epilogue64(a, &tmC, v, m0, n0, stg, ctab, other, pair, uses, tma != 0, lane, status))
        break;
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();  // no CTA leaves while its peer may still signal its barriers
  if (warp == 1) {
    tc_fence_after();
    if (CG == 2) tmem_dealloc2(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int out_size(int kind) { return kind == kFp8OutQ ? 1 : (kind == kFp8OutF16 || kind == kFp8OutBF16) ? 2 : 4; }

int map_codes(CUtensorMap* m, const uint8_t* p, int rows, int K, int ld) {
  return make_tmap_2d_typed(m, p, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, K, ld, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Scale tiles as rows of 128 words, `tiles` of them a box.
int map_scales(CUtensorMap* m, const uint8_t* p, int rows, int K, int tiles) {
  const int64_t n = static_cast<int64_t>((K + 511) / 512) * ((rows + 127) / 128);
  if (n > 0x7fffffff) return -2;
  return make_tmap_2d_typed(m, p, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, static_cast<int>(n), 128, 128, 128, tiles,
                            CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <int CG>
int launch(const Fp8Linear& a, int* status, cudaStream_t s) {
  using C = Cfg<CG>;
  CUtensorMap ta, tb, tsa, tsb;
  if (map_codes(&ta, a.x, a.M, a.K, a.ldx) || map_codes(&tb, a.w, a.N, a.K, a.ldw) ||
      map_scales(&tsa, a.xs, a.M, a.K, C::kSfATiles) || map_scales(&tsb, a.ws, a.N, a.K, C::kSfBTiles))
    return -2;
  static std::atomic<uint64_t> attr_set{0};  // one bit per device; first calls may race
  int dev = 0;
  cudaGetDevice(&dev);
  if (!((attr_set.load() >> (dev & 63)) & 1)) {
    if (cudaFuncSetAttribute(k_fp8_gemm<CG>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess)
      return -3;
    // the register split waits for registers that the launch must have
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, k_fp8_gemm<CG>) != cudaSuccess ||
        fa.numRegs * kThreads < 128 * kRegsCtl + 512 * kRegsEpi)
      return -5;
    attr_set.fetch_or(uint64_t(1) << (dev & 63));
  }
  const long m_units = ((a.M + 127) / 128 + CG - 1) / CG;
  const long tiles = m_units * ((a.N + C::kBN - 1) / C::kBN);
  if (tiles > 0x7fffffffL) return -1;
  const int esz = out_size(a.kind);
  const int tma = aligned(a.out, 16) && (static_cast<size_t>(a.ldo) * esz) % 16 == 0;
  CUtensorMap tc = tsa;
  if (tma && make_tmap_2d_typed(&tc, a.out,
                                esz == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                : esz == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                           : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                                esz, a.M, a.N, a.ldo, 64 / esz, 32, CU_TENSOR_MAP_SWIZZLE_64B))
    return -2;
  const unsigned grid = static_cast<unsigned>(std::min<long>(tiles, sm_count(dev) / CG) * CG);
  return launch_pdl(k_fp8_gemm<CG>, dim3(grid), kThreads, C::kSmem, s, CG, ta, tb, tsa, tsb, tc, a, tma, status) ==
                 cudaSuccess
             ? 0
             : -4;
}

}  // namespace

int check_linear_fp8(const Fp8Linear& a) {
  if (a.K <= 0 || a.N <= 0 || a.M > kMostCount || a.N > kMostCount || a.K > kMostCount || a.ldx < a.K ||
      a.ldw < a.K || a.ldx % 16 || a.ldw % 16 || a.ldo < a.N ||
      !aligned(a.x, 16) || !aligned(a.w, 16) || !aligned(a.xs, 16) || !aligned(a.ws, 16) ||
      !aligned(a.out, out_size(a.kind)) || !aligned(a.bias, 4) || !aligned(a.scale, 4))
    return -1;
  if (a.kind == kFp8OutQ && (a.ldo % 16 || !aligned(a.out, 16) || !aligned(a.out_scales, 16))) return -1;
  return 0;
}

int linear_fp8(const Fp8Linear& a, int* status, cudaStream_t s) {
  // The tile shape with the shorter time (ns): waves of tiles times a tile's k-blocks of 128,
  // and the handover from one tile to the next, longer with a pair's one accumulator; pairs
  // also take longer to set up. Measured back to back in a graph, at N = 4096, K = 1024 and M =
  // 512, 1370, 2740, 5480, 21920: single CTAs 7.0, 12.0, 17.7, 30, 107 us, pairs 8.8, 12.3, 16.2,
  // 23, 87; at N = 1024, K = 4096 and M = 1370, 2740: 15.2 and 25, 17.7 and 17.3.
  int dev = 0;
  cudaGetDevice(&dev);
  const int64_t sms = sm_count(dev), kb = (a.K + 127) / 128;
  const int64_t tiles1 = (static_cast<int64_t>(a.M) + 127) / 128 * ((a.N + 127) / 128);
  const int64_t tiles2 = (static_cast<int64_t>(a.M) + 255) / 256 * ((a.N + 255) / 256);
  const int64_t time1 = 3800 + (tiles1 + sms - 1) / sms * (kb * 270 + 250);
  const int64_t time2 = 4500 + (tiles2 + sms / 2 - 1) / (sms / 2) * (kb * 330 + 1300);
  return time2 <= time1 ? launch<2>(a, status, s) : launch<1>(a, status, s);
}

}  // namespace da3b

using namespace da3b;

static int run_linear(const void* x, int M, int K, int ldx, const void* xs, const void* w, int N, int ldw,
                      const void* ws, const float* bias, const float* scale, int act, int kind, void* out, int ldo,
                      void* out_scales, void* stream) {
  if (!w || !ws || M < 0 || (M > 0 && (!x || !xs || !out)) || act < 0 || act > 3) return -100;
  const Fp8Linear a = {static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(xs), static_cast<const uint8_t*>(w),
                       static_cast<const uint8_t*>(ws), M, N, K, ldx, ldw, bias, scale, act, kind, out, ldo,
                       static_cast<uint8_t*>(out_scales)};
  if (check_linear_fp8(a)) return -1;
  if (M == 0) return 0;
  if (!usable_here({x, xs, w, ws, bias, scale, out, out_scales})) return -104;
  int* st = device_status_word();
  if (!st) return -101;
  return linear_fp8(a, st, static_cast<cudaStream_t>(stream));
}

extern "C" {

DA3B_API int da3b_linear_fp8(const void* x, int M, int K, int ldx, const void* x_scales, const void* w, int N, int ldw,
                             const void* w_scales, const float* bias, int act, void* out, int out_dtype, int ldo,
                             void* stream) {
  if (out_dtype < kF16 || out_dtype > kF32) return -100;
  return run_linear(x, M, K, ldx, x_scales, w, N, ldw, w_scales, bias, nullptr, act, out_dtype, out, ldo, nullptr,
                    stream);
}

DA3B_API int da3b_linear_fp8_q(const void* x, int M, int K, int ldx, const void* x_scales, const void* w, int N,
                               int ldw, const void* w_scales, const float* bias, int act, void* out_q, int ldo,
                               void* out_scales, void* stream) {
  if (!out_scales && M > 0) return -100;
  return run_linear(x, M, K, ldx, x_scales, w, N, ldw, w_scales, bias, nullptr, act, kFp8OutQ, out_q, ldo, out_scales,
                    stream);
}

DA3B_API int da3b_linear_fp8_resid_f32(const void* x, int M, int K, int ldx, const void* x_scales, const void* w,
                                       int N, int ldw, const void* w_scales, const float* bias, const float* scale,
                                       float* resid, int ldr, void* stream) {
  return run_linear(x, M, K, ldx, x_scales, w, N, ldw, w_scales, bias, scale, kActNone, kFp8OutResid, resid, ldr,
                    nullptr, stream);
}

}  // extern "C"
