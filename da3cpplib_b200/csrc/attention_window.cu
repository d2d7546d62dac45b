// Softmax attention over a window of keys and the first few keys of each sequence.
//
// Query i of a sequence with ql queries and kl keys stands at position p = kl - ql + i
// (the queries are the last ones of the keys) and sees the keys j < kl with
// j <= p + right and (j >= p - left or j < sinks). o = sum_j softmax_j(scale q.k_j) v_j; a
// query that sees nothing gets zeros, rows from ql on are not written.
#include <algorithm>
#include <atomic>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "attention_window.h"
#include "da3b.h"
#include "launch.h"
#include "ops.h"
#include "ptx.cuh"

namespace da3b {

namespace {

// ------------------------------------------------------------------ many queries
// Several tiles of 128 query rows a CTA (one CTA per SM) share every key tile: three with key
// tiles of 48 at head_dim 64, two with key tiles of 64 at 128. A query row is one (token,
// head): g query heads that share a key head lie side by side, 128 / g tokens a tile, so that
// shared heads read their keys once and a tile spans few positions (a window's ends are
// masked work).
//   warp 0     TMA: the Q tiles, then the key tiles that some row sees, K of a tile together
//              with V of the tile two before in a ring ([keys][64 dims] boxes, 128B swizzle);
//   warps 1..  one a query tile: O_t += P_t V (P_t from tensor memory; V is read as it lies,
//              its dims contiguous: an MN-major operand), then S_t = Q_t K^T two tiles on;
//   warps 4..  softmax, four a query tile: thread = row (its TMEM lane), the row's scores in
//              registers, one pass; P back to tensor memory.
// A CTA that is through its loads takes over the item of a CTA that has not been launched yet
// (cluster launch control), so that barriers and tensor memory are set up once, and the next
// item's queries, keys and scores are on their way while the softmax warps write this one's
// rows. The order stays the grid's, and no counter in memory has to be reset. Two prompts of
// 8192 tokens, 16 heads of 128, a window of 1024: 183 us with a CTA an item, 148 so (a window
// of 64: 82 and 44; 64 views of 1370 tokens, 16 heads of 64: 835 and 710).
// Tensor memory holds two S_t for each query tile, taken in turn, and P_t lies over its S_t:
// the scores of the next key tile are there when a softmax is done, and one barrier each way
// is enough. What bounds it is that softmax, a chain of its own: 16384 keys, 9 x 16 CTAs, take
// 942 ns a step of 48 keys at head_dim 64 (1064 ns a step of 64 at 128), 858 (904) without the
// products, 660 (968) without the exponentials, and 540 (536) without both, which is what
// the waits, the trip from and to tensor memory and the maximum take (since the first tile's
// maximum lost its branch, 833 ns at head_dim 64). Several query tiles
// fill each other's waits; tensor memory has no room for more of them. Full attention of 4096
// tokens runs at 743 and 1130 TFLOP/s. Taken otherwise: P_t over a single S_t (746 us against
// 793 in that measure with four query tiles, but 114 against 86 for a new view of 1297
// tokens, whose items then fill 96 SMs), S_t and P_t in columns of their own (802 us, 90), two
// softmax threads a row (1057 us), one issuing warp for all query tiles (its waits, about
// 100 cycles each, leave the tensor pipe idle).
// The maximum of a row is raised only when a tile exceeds it by more than 2^8; O_t is then
// rescaled in tensor memory. Sums are f32 of the unrounded probabilities.
// Masks are applied to the tiles that a window's end, the sinks' end or the last key cuts.
// V rows of such tiles that no row of the CTA sees are zeroed in shared memory (0 * NaN).

constexpr float kRaise = 8.0f;          // log2 by which a tile may exceed the row's maximum

template <int D>
struct WinCfg {
  static constexpr int kNT = D == 64 ? 3 : 2;    // query tiles
  static constexpr int kKT = D == 64 ? 48 : 64;  // keys a tile
  static constexpr int kThreads = 128 + 128 * kNT;
  // registers move from the first warpgroup to the softmax's (setmaxnreg); the split may not
  // exceed what the launch holds
  static constexpr int kRegsLaunch = kNT == 3 ? 128 : 168, kRegsCtl = kNT == 3 ? 80 : 72, kRegsSoft = kNT == 3 ? 144 : 216;
  static_assert(128 * kRegsCtl + 128 * kNT * kRegsSoft <= kThreads * kRegsLaunch, "register split");
  static constexpr int kQTile = 128 * D * 2, kTile = kKT * D * 2;  // bytes of a Q and of a K or V tile
  static constexpr int kStage = 2 * kTile;          // a V tile and a K tile
  static constexpr int kRing = D == 64 ? 10 : 5, kRingBytes = kRing * kStage;
  static constexpr int kSmem = 1024 + kNT * kQTile + kRingBytes + 640;
  static constexpr uint32_t kColO = 2 * kNT * kKT;  // behind two S_t each
  static_assert(kColO + kNT * D <= 512, "tensor memory");
  // a CTA's share of a split item: O rows, then (m, l), over the Q tiles and the ring
  static constexpr int kShareO = kNT * 128 * D * 4;
  static_assert(kShareO + kNT * 128 * 8 <= kNT * kQTile + kRingBytes, "a share fits");
};

__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float fmax_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x by the hardware approximation, free for the compiler to schedule.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x of two values on the FMA pipe (the MUFU pipe takes one exponential a score
// otherwise, and bounds the kernel): x = j + f with j = round(x) (adding 1.5 * 2^23 + 127
// leaves j + 127 in the low mantissa bits), f in [-0.5, 0.5]; 2^f by a cubic fitted to
// relative error (max 7.5e-5, below the rounding of P to 16 bits), times 2^j, whose bits are
// j + 127 in the exponent field. (Adding j to the cubic's own exponent field would turn NaN
// into a number.) x is held at -127, where those bits and so the result are zero: a masked score
// has no weight at all, whatever value it would meet in V.
__device__ __forceinline__ float2 exp2_cubic(float2 x) {
  constexpr float kShift = 12582912.0f + 127.0f;
  constexpr float c3 = 0.05517166853f, c2 = 0.24261112511f, c1 = 0.69326096773f, c0 = 0.99992805719f;
  x = make_float2(fmax_nan(x.x, -127.0f), fmax_nan(x.y, -127.0f));
  const float2 t = __fadd2_rn(x, make_float2(kShift, kShift));
  const float2 j = __fadd2_rn(t, make_float2(-kShift, -kShift));
  const float2 f = __fadd2_rn(x, make_float2(-j.x, -j.y));
  float2 p = __ffma2_rn(make_float2(c3, c3), f, make_float2(c2, c2));
  p = __ffma2_rn(p, f, make_float2(c1, c1));
  p = __ffma2_rn(p, f, make_float2(c0, c0));
  return __fmul2_rn(p, make_float2(__uint_as_float(__float_as_uint(t.x) << 23),
                                   __uint_as_float(__float_as_uint(t.y) << 23)));
}

// N columns (a multiple of 16) of this thread's lane of tensor memory, there after
// tmem_wait_ld and landed.
template <int N>
__device__ __forceinline__ void load_cols(uint32_t taddr, float (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N / 32; ++i)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(s[32 * i + 0]), "=f"(s[32 * i + 1]), "=f"(s[32 * i + 2]), "=f"(s[32 * i + 3]), "=f"(s[32 * i +
          4]), "=f"(s[32 * i + 5]), "=f"(s[32 * i + 6]), "=f"(s[32 * i + 7]), "=f"(s[32 * i + 8]), "=f"(s[32 *
          i + 9]), "=f"(s[32 * i + 10]), "=f"(s[32 * i + 11]), "=f"(s[32 * i + 12]), "=f"(s[32 * i + 13]),
          "=f"(s[32 * i + 14]), "=f"(s[32 * i + 15]), "=f"(s[32 * i + 16]), "=f"(s[32 * i + 17]), "=f"(s[32 *
          i + 18]), "=f"(s[32 * i + 19]), "=f"(s[32 * i + 20]), "=f"(s[32 * i + 21]), "=f"(s[32 * i + 22]),
          "=f"(s[32 * i + 23]), "=f"(s[32 * i + 24]), "=f"(s[32 * i + 25]), "=f"(s[32 * i + 26]), "=f"(s[32 *
          i + 27]), "=f"(s[32 * i + 28]), "=f"(s[32 * i + 29]), "=f"(s[32 * i + 30]), "=f"(s[32 * i + 31])
        : "r"(taddr + 32 * i));
  if constexpr (N % 32 != 0)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=f"(s[N - 16 + 0]), "=f"(s[N - 16 + 1]), "=f"(s[N - 16 + 2]), "=f"(s[N - 16 + 3]), "=f"(s[N - 16 +
          4]), "=f"(s[N - 16 + 5]), "=f"(s[N - 16 + 6]), "=f"(s[N - 16 + 7]), "=f"(s[N - 16 + 8]), "=f"(s[N -
          16 + 9]), "=f"(s[N - 16 + 10]), "=f"(s[N - 16 + 11]), "=f"(s[N - 16 + 12]), "=f"(s[N - 16 + 13]),
          "=f"(s[N - 16 + 14]), "=f"(s[N - 16 + 15])
        : "r"(taddr + N - 16));
}
// N words (a multiple of 8) into this thread's lane, there after tmem_wait_st.
template <int N>
__device__ __forceinline__ void store_words(uint32_t taddr, const uint32_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N / 32; ++i) {
    uint32_t x[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] = w[32 * i + j];
    tmem_st32(taddr + 32 * i, x);
  }
  constexpr int r = N / 32 * 32;
  if constexpr (N % 32 >= 16) {
    uint32_t x[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = w[r + j];
    tmem_st16(taddr + r, x);
  }
  if constexpr (N % 16 != 0)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr + N - 8),
                 "r"(w[N - 8]), "r"(w[N - 7]), "r"(w[N - 6]), "r"(w[N - 5]), "r"(w[N - 4]), "r"(w[N - 3]), "r"(w[N - 2]),
                 "r"(w[N - 1])
                 : "memory");
}

// The lowest n bits (none for n <= 0, all for n >= 32). Masks are taken from such words:
// compared column by column against a row's bounds, a cut tile took thousands of cycles.
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Keeps every use of loaded values behind the wait before it.
template <int N>
__device__ __forceinline__ void landed(float (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(s[i]));
}

// 32 columns of O; zeros where no product was made. Warp-collective.
__device__ __forceinline__ void take_o(uint32_t taddr, bool any, uint32_t (&w)[32]) {
  if (any) {
    tmem_ld32(taddr, w);
    tmem_wait_ld();
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) w[i] = 0u;
  }
}

// Transposes 4 x 4 chunks over four neighbouring lanes: lane j's u[i] becomes lane i's u[j].
__device__ __forceinline__ void turn4(uint4 (&u)[4], int lane) {
  auto swap = [&](uint4& x, uint4& y, int by) {
    const bool up = lane & by;
    uint4 give = up ? x : y;
    give.x = __shfl_xor_sync(0xffffffffu, give.x, by);
    give.y = __shfl_xor_sync(0xffffffffu, give.y, by);
    give.z = __shfl_xor_sync(0xffffffffu, give.z, by);
    give.w = __shfl_xor_sync(0xffffffffu, give.w, by);
    if (up) x = give;
    else y = give;
  };
  swap(u[0], u[1], 1);
  swap(u[2], u[3], 1);
  swap(u[0], u[2], 2);
  swap(u[1], u[3], 2);
}

// Shared-memory descriptor of an MN-major operand tile in 128B-swizzled rows of 64 values:
// 1024 bytes between groups of eight k rows, lbo bytes between 64-wide column chunks.
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t saddr, uint32_t lbo) {
  uint64_t d = static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(lbo >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Work that is left in the grid: asks for the launch of a CTA that has not begun to be
// cancelled, so that this one takes its item (16 bytes at answer, one phase of bar). Not
// asked again once an answer was no.
__device__ __forceinline__ void take_launch(uint4* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
// blockIdx.x of the cancelled CTA, -1 for none.
__device__ __forceinline__ int launch_taken(const uint4* answer) {
  int x;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 h, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "mov.b32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n\t}\n"
      : "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return x;
}

// What the rows of one query tile see: tokens [i0, i0 + n) of a sequence at positions from
// p on. Keys are counted in columns (Columns below) once shifted.
struct Span {
  int n;                 // tokens inside the sequence (0: the tile has no rows)
  int hi_min, hi_max;    // last visible key of its first and last row
  int lo_min, lo_max;    // first key of their windows
  __device__ Span(int i0, int tokens, int ql, int kl, int left, int right) {
    n = min(max(ql - i0, 0), tokens);
    const int p = kl - ql + i0, pl = p + max(n - 1, 0);
    hi_min = min(kl - 1, p + right);
    hi_max = min(kl - 1, pl + right);
    lo_min = max(0, p - left);
    lo_max = max(0, pl - left);
  }
  __device__ void shift(int by) {
    hi_min += by;
    hi_max += by;
    lo_min += by;
    lo_max += by;
  }
};

// The same in key tiles of KT columns: which a query tile sees, and sees whole.
template <int KT>
struct Seen {
  int first, last, front;           // some row sees tiles [first, last] and [0, front), up to last
  int whole0, whole1, whole_front;  // every row sees all of [whole0, whole1] and [0, whole_front), up to whole1
  __device__ Seen(const Span& sp, int sinks) {
    first = sp.lo_min / KT;
    last = sp.n > 0 && sp.hi_max >= 0 ? sp.hi_max / KT : -1;
    front = sinks / KT + (sinks % KT != 0);
    whole0 = sp.lo_max / KT + (sp.lo_max % KT != 0);
    whole1 = sp.hi_min >= 0 ? (sp.hi_min + 1) / KT - 1 : -1;
    whole_front = sinks / KT;
  }
  __device__ bool some(int tile) const { return tile <= last && (tile >= first || tile < front); }
  __device__ bool whole(int tile) const { return tile <= whole1 && (tile >= whole0 || tile < whole_front); }
};

// The keys of a CTA as one run of columns: the sinks, up to a multiple of eight, then the
// windows' keys from the oldest on, so that neither starts a tile of its own: four sinks and
// a window of 1024 for 64 tokens are 18 tiles of 64 instead of 19. One tile may hold both; it
// is loaded in boxes of eight rows.
struct Columns {
  int front;  // columns of the sinks (0: the columns are keys from `base` on)
  int base;   // key of column `front`
  __device__ Columns(int sinks, int lo) {
    front = sinks > lo - 128 ? 0 : (sinks + 7) & ~7;
    base = sinks > 0 && front == 0 ? 0 : lo;
  }
  __device__ int key(int v) const { return v < front ? v : base + v - front; }
  __device__ int shift() const { return front - base; }  // key + shift = column
  __device__ bool mixed(int v0, int keys) const { return v0 < front && front < v0 + keys; }
};

// One unit of work: up to qt query tiles of a group of heads of a sequence, and of their key
// tiles the share that one CTA of a cluster of nsplit takes. Items are numbered so that a
// sequence's last tokens come first: where the left side is not limited they have the most
// keys.
template <int KT>
struct alignas(16) Item {
  int b, h0, hk, ql, kl, i0;
  int nt;        // query tiles with rows (-1: not an item, there is no more work)
  int lo, hi;    // columns that the windows reach
  int n0, n_all; // first key tile and their number
  Columns cols;
  __device__ Item(const AttnWindow& a, int item, int split, int nsplit, int g, int tokens, int qt, int tiles)
      : b(item / tiles / (a.heads / g)),
        h0(item / tiles % (a.heads / g) * g),
        hk(h0 / (a.heads / a.kv_heads)),
        ql(a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len),
        kl(a.k_lens ? min(max(a.k_lens[b], 0), a.k_len) : a.k_len),
        i0((tiles - 1 - item % tiles) * qt * tokens),
        cols(a.sinks, Span(i0, tokens, ql, kl, a.left, a.right).lo_min) {
    nt = i0 < ql ? min(qt, (ql - i0 + tokens - 1) / tokens) : 0;
    const int hi_key = nt > 0 ? Span(i0 + (nt - 1) * tokens, tokens, ql, kl, a.left, a.right).hi_max : -1;
    hi = hi_key + cols.shift();
    lo = Span(i0, tokens, ql, kl, a.left, a.right).lo_min + cols.shift();
    const int n_cols = hi_key < 0 ? 0 : hi / KT + 1;
    n0 = static_cast<int>(static_cast<int64_t>(split) * n_cols / nsplit);
    n_all = static_cast<int>(static_cast<int64_t>(split + 1) * n_cols / nsplit) - n0;
  }
  __device__ Span span(const AttnWindow& a, int tokens, int t) const {
    Span sp(i0 + t * tokens, t < nt ? tokens : 0, ql, kl, a.left, a.right);
    sp.shift(cols.shift());
    return sp;
  }
  __device__ int col0(int n) const { return (n0 + n) * KT; }
};

template <int D, bool BF16>
__global__ void __launch_bounds__(WinCfg<D>::kThreads, 1)
    k_attn_tiles(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmK8,
                 const __grid_constant__ CUtensorMap tmV8, const __grid_constant__ AttnWindow a, int g, int tokens,
                 int qt, int tiles, int nsplit, int* status) {
  using C = WinCfg<D>;
  constexpr int NT = C::kNT, KT = C::kKT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                       // [NT]
  // the ring: load i brings V of tile i - 2 and K of tile i, where there are such tiles
  uint8_t* sKV = sQ + NT * C::kQTile;       // [kRing] V, K
  Item<KT>* items = reinterpret_cast<Item<KT>*>(sKV + C::kRingBytes);  // [2] the current one and the next
  uint4* answer = reinterpret_cast<uint4*>(items + 2);  // to the request for another item
  uint64_t* answered = reinterpret_cast<uint64_t*>(answer + 1);
  uint64_t* item_full = answered + 1;       // [2]
  uint64_t* item_free = item_full + 2;      // [2] done with by every warp that works
  uint64_t* q_full = item_free + 2;
  uint64_t* q_free = q_full + 1;            // the item's last scores are complete (every issuing warp)
  uint64_t* kv_full = q_free + 1;           // [kRing]
  uint64_t* kv_empty = kv_full + C::kRing;  // [kRing] (every issuing warp)
  // one barrier for the even and one for the odd ones of the tiles that query tile t sees:
  uint64_t* s_full = kv_empty + C::kRing;   // [NT][2] S_t complete (and the product two before)
  uint64_t* p_ready = s_full + 2 * NT;      // [NT][2] P_t written, O_t rescaled, V rows zeroed (4 warps)
  uint64_t* pv_done = p_ready + 2 * NT;     // [NT][2] P_t V complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + 2 * NT);
  uint32_t* gave_up = tmem_slot + 1;        // not 0: a wait of this CTA ran out

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a cluster of nsplit CTAs shares an item's key tiles
  const int split = static_cast<int>(blockIdx.x) % nsplit, item0 = static_cast<int>(blockIdx.x) / nsplit;
  pdl_wait();

  if (threadIdx.x == 0) {
    *gave_up = 0;
    mbar_init(q_full, 1);
    mbar_init(q_free, NT);
    mbar_init(answered, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_free[i], 5 * NT);
    }
    for (int s = 0; s < C::kRing; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], NT);
    }
    for (int t = 0; t < 2 * NT; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_ready[t], 4);
      mbar_init(&pv_done[t], 1);
    }
    fence_mbar_init();
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsCtl));
    if (warp == 0) {
      if (lane == 0) {
        const uint32_t q_bytes = static_cast<uint32_t>(g * tokens) * 128;  // of one 64-wide box
        int st = 0;
        uint32_t par = 1, loads = 0, nq = 0;
        bool ok = true;
        int item = item0;
        for (uint32_t k = 0;; ++k) {
          ok = mbar_wait(&item_free[k & 1], ((k >> 1) & 1) ^ 1u, status, kStatusTimeoutEmpty);
          if (!ok) break;
          if (item < 0) items[k & 1].nt = -1;
          else items[k & 1] = Item<KT>(a, item, split, nsplit, g, tokens, qt, tiles);
          mbar_arrive(&item_full[k & 1]);
          if (item < 0) break;
          const Item<KT> it = items[k & 1];
          auto load_tile = [&](uint8_t* dst, const CUtensorMap& whole, const CUtensorMap& eight, uint64_t* bar, int v0) {
            for (int c = 0; c < D / 64; ++c) {
              if (!it.cols.mixed(v0, KT)) {
                tma_load_4d(dst + c * KT * 128, &whole, bar, c * 64, it.hk, it.cols.key(v0), it.b);
              } else {
                for (int j = 0; j < KT; j += 8)
                  tma_load_4d(dst + (c * KT + j) * 128, &eight, bar, c * 64, it.hk, it.cols.key(v0 + j), it.b);
              }
            }
          };
          if (it.n_all > 0) {
            ok = mbar_wait(q_free, (nq & 1) ^ 1u, status, kStatusTimeoutEmpty);
            if (ok) {
              mbar_arrive_expect_tx(q_full, q_bytes * (D / 64) * it.nt);
              for (int t = 0; t < it.nt; ++t)
                for (int c = 0; c < D / 64; ++c)
                  tma_load_4d(sQ + t * C::kQTile + c * 16384, &tmQ, q_full, c * 64, it.h0, it.i0 + t * tokens, it.b);
              ++nq;
            }
            for (int i = 0; i < it.n_all + 2 && ok; ++i) {
              ok = mbar_wait(&kv_empty[st], par, status, kStatusTimeoutEmpty);
              if (!ok) break;
              uint8_t* dst = sKV + st * C::kStage;
              const bool k_tile = i < it.n_all, v_tile = i >= 2;
              mbar_arrive_expect_tx(&kv_full[st], (k_tile ? C::kTile : 0) + (v_tile ? C::kTile : 0));
              if (k_tile) load_tile(dst + C::kTile, tmK, tmK8, &kv_full[st], it.col0(i));
              if (v_tile) load_tile(dst, tmV, tmV8, &kv_full[st], it.col0(i - 2));
              ++loads;
              if (++st == C::kRing) { st = 0; par ^= 1u; }
            }
          }
          if (!ok || nsplit > 1) break;
          // Ask for another item, not before this one's last tile is under way: work that is
          // asked for early is not there for a CTA that runs out of it.
          mbar_arrive_expect_tx(answered, 16);
          take_launch(answer, answered);
          ok = mbar_wait(answered, k & 1, status, kStatusTimeoutFull);
          if (!ok) {  // as drain: the answer is written to this CTA's memory
            for (int i = 0; i < 8 && !mbar_wait(answered, k & 1, status, kStatusTimeoutFull); ++i) {}
            break;
          }
          item = launch_taken(answer);
          fence_proxy_async_smem();  // read before another answer is written there
        }
        if (!ok) {
          drain(kv_full, C::kRing, loads, status);
          if (nq > 0) mbar_wait(q_full, (nq - 1) & 1, status, kStatusTimeoutFull);
          *gave_up = 1;
        }
      }
      __syncwarp();
    } else if (warp <= NT) {
      // The whole warp runs this loop and one elected lane issues: addresses and descriptors
      // then stay in uniform registers, where the instructions want them. (With one lane in
      // the loop every product's operands were moved there one by one, and that set the
      // pace.)
      constexpr uint32_t fmt = BF16 ? (1u << 7) | (1u << 10) : 0u;
      constexpr uint32_t id_s = umma_idesc_f16(128, KT) | fmt;
      constexpr uint32_t id_o = umma_idesc_f16(128, D) | fmt | (1u << 16);  // B is MN-major
      const bool one = elect_one();
      const int t = warp - 1;
      const uint64_t qd = umma_desc_sw128(smem_u32(sQ) + t * C::kQTile);
      const uint64_t vd0 = desc_mn_sw128(smem_u32(sKV), KT * 128), kd0 = umma_desc_sw128(smem_u32(sKV) + C::kTile);
      const uint32_t tS = tmem + 2 * t * KT, tO = tmem + C::kColO + t * D;
      uint32_t ns = 0, np = 0;  // S and P V products issued
      auto issue_s = [&](int st) {
        const uint64_t kd = kd0 + st * (C::kStage >> 4);
        const uint32_t d = tS + (ns & 1) * KT;
        if (one) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_f16(d, qd + c * 1024 + 2 * kk, kd + c * (KT * 8) + 2 * kk, id_s, (c > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&s_full[2 * t + (ns & 1)]);
        }
        __syncwarp();
        ++ns;
      };
      bool ok = true;
      int st = 0;
      uint32_t par = 0, nq = 0;
      for (uint32_t k = 0; ok; ++k) {
        ok = mbar_wait_warp(&item_full[k & 1], (k >> 1) & 1, status, kStatusTimeoutFull);
        const Item<KT> it = items[k & 1];
        if (!ok || it.nt < 0) break;
        const Seen<KT> see(it.span(a, tokens, t), a.sinks);
        const uint32_t np0 = np;
        if (it.n_all > 0) ok = mbar_wait_warp(q_full, nq++ & 1, status, kStatusTimeoutFull);
        for (int i = 0; i < it.n_all + 2 && it.n_all > 0 && ok; ++i) {
          ok = mbar_wait_warp(&kv_full[st], par, status, kStatusTimeoutFull);
          if (ok && i >= 2 && see.some(it.n0 + i - 2)) {
            ok = mbar_wait_warp(&p_ready[2 * t + (np & 1)], (np >> 1) & 1, status, kStatusTimeoutFull);
            if (ok) {
              tc_fence_after();
              const uint64_t vd = vd0 + st * (C::kStage >> 4);
              const uint32_t p = tS + (np & 1) * KT;
              if (one) {
#pragma unroll
                for (int kk = 0; kk < KT / 16; ++kk)
                  umma_f16_tmem_a(tO, p + 8 * kk, vd + 128 * kk, id_o, (np != np0 || kk > 0) ? 1u : 0u);
                umma_commit(&pv_done[2 * t + (np & 1)]);
              }
              __syncwarp();
              ++np;
            }
          }
          // behind the product that read the P_t in its place
          if (ok && i < it.n_all && see.some(it.n0 + i)) {
            tc_fence_after();
            issue_s(st);
          }
          if (ok && one) {
            umma_commit(&kv_empty[st]);
            if (i == it.n_all - 1) umma_commit(q_free);
          }
          __syncwarp();
          if (++st == C::kRing) { st = 0; par ^= 1u; }
        }
        if (nsplit > 1) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_free[k & 1]);
      }
      if (!ok) *gave_up = 1;
      // every load of the item has landed; the softmax warps write their shares over them
      if (nsplit > 1) asm volatile("bar.sync 1, %0;" ::"n"(160 * NT) : "memory");
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoft));
    const int t = (warp - 4) >> 2, q = warp & 3, r = q * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t tS0 = tmem + 2 * t * KT + lanes, tO = tmem + C::kColO + t * D + lanes;
    const float c = a.scale * 1.4426950408889634f;
    int cnt = 0, st = C::kRing - 1;
    uint32_t par = 1;
    bool ok = true;
    auto advance = [&]() {
      if (++st == C::kRing) { st = 0; par ^= 1u; }
    };
    for (uint32_t k = 0;; ++k) {
      ok = mbar_wait_warp(&item_full[k & 1], (k >> 1) & 1, status, kStatusTimeoutFull);
      if (nsplit == 1 && (!ok || items[k & 1].nt < 0)) break;
      const int cnt0 = cnt;
      float m = -INFINITY, l = 0.f;
      if (ok) {
        const Item<KT> it = items[k & 1];
        const Seen<KT> see(it.span(a, tokens, t), a.sinks);
        const int n0 = it.n0, n_all = it.n_all, lo = it.lo, hi = it.hi;
        // tiles with keys that no row of the CTA sees, and the tiles that need no look: seen whole
        // by this query tile, and by its windows alone
        const int fix0 = lo > a.sinks ? a.sinks / KT : 1, fix1 = lo > a.sinks ? (lo - 1) / KT : 0;
        const int fix2 = (hi + 1) % KT != 0 ? hi / KT : -1;
        const int plain0 = max(see.whole0, fix1 + 1);
        const int plain1 = min(min(see.whole1, see.last), fix2 < 0 ? see.whole1 : fix2 - 1);
        const int p = it.kl - it.ql + it.i0 + t * tokens + r / g;   // this row's position, and its columns
        const int row_hi = min(it.kl - 1, p + a.right) + it.cols.shift(), row_lo = p - a.left + it.cols.shift();
        if (n_all > 0) {  // the loads bring V two behind K
          advance();
          advance();
        }
        for (int n = 0; n < n_all && ok; ++n) {
          advance();  // the stage of this tile's V
          const bool plain = n0 + n >= plain0 && n0 + n <= plain1;
          if (!plain && !see.some(n0 + n)) continue;
          const int v0 = (n0 + n) * KT;
          const uint32_t tS = tS0 + (cnt & 1) * KT;  // S_t, then P_t
          ok = mbar_wait_warp(&s_full[2 * t + (cnt & 1)], (cnt >> 1) & 1, status, kStatusTimeoutAccum);
          if (!ok) break;
          tc_fence_after();
          float s[KT];
          load_cols<KT>(tS, s);
          // keys that no row of the CTA sees: their V rows count as zero, whatever they hold
          if (!plain && (n0 + n == fix2 || (n0 + n >= fix0 && n0 + n <= fix1))) {
            ok = mbar_wait_warp(&kv_full[st], par, status, kStatusTimeoutFull);
            if (!ok) break;
            const int v = v0 + r;
            if (r < KT && (v > hi || (v < lo && v >= a.sinks))) {
              uint4* row = reinterpret_cast<uint4*>(sKV + st * C::kStage + r * 128);
#pragma unroll
              for (int i = 0; i < D / 8; ++i) row[(i >> 3) * (KT * 8) + (i & 7)] = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
          }
          tmem_wait_ld();
          landed<KT>(s);
          if (!plain && !see.whole(n0 + n)) {
            // visible columns of this row: [x0, x1] and [0, x2) of the tile, up to x1
            const int x1 = row_hi - v0, x0 = row_lo - v0, x2 = a.sinks - v0;
#pragma unroll
            for (int w = 0; w < (KT + 31) / 32; ++w) {
              const uint32_t bits = below(x1 + 1 - 32 * w) & (~below(x0 - 32 * w) | below(x2 - 32 * w));
#pragma unroll
              for (int i = 0; i < 32 && 32 * w + i < KT; ++i)
                s[32 * w + i] = bits >> i & 1u ? s[32 * w + i] : -INFINITY;
            }
          }
          float m8[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) m8[i] = fmaxf(s[i], s[KT - 8 + i]);
#pragma unroll
          for (int i = 8; i < KT - 8; i += 16)
#pragma unroll
            for (int j = 0; j < 8; ++j) m8[j] = fmax3(m8[j], s[i + j], s[i + 8 + j]);
          const float mt = fmaxf(fmax3(fmax3(m8[0], m8[1], m8[2]), fmax3(m8[3], m8[4], m8[5]), m8[6]), m8[7]);
          const bool raise = (mt - m) * c > kRaise;  // the first finite one, too; -inf - -inf: no
          const float alpha = raise ? ex2((m - mt) * c) : 1.f;
          if (raise) m = mt;
          const float mc = m == -INFINITY ? 0.f : m * c;
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          uint32_t pk[KT / 2];
#pragma unroll
          for (int i = 0; i < KT / 2; ++i) {
            const float2 x = __ffma2_rn(make_float2(s[2 * i], s[2 * i + 1]), make_float2(c, c), make_float2(-mc, -mc));
            const float2 e = (i & 3) == 0 ? exp2_cubic(x) : make_float2(ex2(x.x), ex2(x.y));
            sum[i & 1] = __fadd2_rn(sum[i & 1], e);
            pk[i] = pack2<BF16>(e.x, e.y);
          }
          const float2 s2 = __fadd2_rn(sum[0], sum[1]);
          // O_t is rescaled behind the last tile's product, where there is one (l is 0 before
          // the first tile only). The product before that is complete: S_t of this tile was
          // issued after it, so no phase of the barrier is missed.
          if (__any_sync(0xffffffffu, raise && l != 0.f)) {
            ok = mbar_wait_warp(&pv_done[2 * t + ((cnt - 1) & 1)], ((cnt - 1) >> 1) & 1, status, kStatusTimeoutAccum);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < D; i += 16) {
              uint32_t w[16];
              tmem_ld16(tO + i, w);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(__uint_as_float(w[j]) * alpha);
              tmem_st16(tO + i, w);
            }
            l *= alpha;
          }
          l += s2.x + s2.y;
          store_words<KT / 2>(tS, pk);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_ready[2 * t + (cnt & 1)]);
          ++cnt;
        }
      }
      if (ok && cnt > cnt0) {
        ok = mbar_wait_warp(&pv_done[2 * t + ((cnt - 1) & 1)], ((cnt - 1) >> 1) & 1, status, kStatusTimeoutAccum);
        tc_fence_after();
      }
      ok = __all_sync(0xffffffffu, ok);
      if (nsplit == 1) {
        // O / l. A row that saw no key still has m = -inf and is zero; one of NaN scores has
        // m = -inf too, but l is NaN.
        const float inv = m == -INFINITY && l == l ? 0.f : 1.f / l;
        const Item<KT> it = items[k & 1];
        const bool mine = ok && r < it.span(a, tokens, t).n * g;
        const int64_t off = it.b * a.os.seq + static_cast<int64_t>(it.i0 + t * tokens + r / g) * a.os.tok +
                            static_cast<int64_t>(it.h0 + r % g) * a.os.head;
#pragma unroll 1
        for (int ch = 0; ch < D / 32; ++ch) {
          uint32_t w[32];
          take_o(tO + 32 * ch, cnt > cnt0, w);
          uint4 u[4];  // 16-byte chunks of this lane's row
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t* uw = reinterpret_cast<uint32_t*>(&u[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              uw[j] = pack2<BF16>(__uint_as_float(w[8 * i + 2 * j]) * inv, __uint_as_float(w[8 * i + 2 * j + 1]) * inv);
          }
          // four lanes exchange so that they hold a row's four chunks, one row after the other
          turn4(u, lane);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int from = (lane & 28) + i;
            const int64_t o = __shfl_sync(0xffffffffu, off, from);
            if (__shfl_sync(0xffffffffu, mine, from))
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + o + 32 * ch + 8 * (lane & 3)) = u[i];
          }
        }
        tc_fence_before();  // O_t has been read before the next item's first P_t is ready
      } else {
        // this CTA's share of the row, over the Q tiles and the ring: O, 16-byte chunks
        // XOR-swizzled by row, then (m, l). They are idle once every product is complete, which
        // the softmax warps know, and every load, which the issuing warps know: a tile between
        // the sinks and the windows is loaded although no row sees it, and no product waits
        // for one at the end of the share.
        asm volatile("bar.sync 1, %0;" ::"n"(160 * NT) : "memory");
        float4* part = reinterpret_cast<float4*>(smem) + (t * 128 + r) * (D / 4);
#pragma unroll 1
        for (int ch = 0; ch < D / 32; ++ch) {
          uint32_t w[32];
          take_o(tO + 32 * ch, cnt > cnt0, w);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            part[(8 * ch + i) ^ (r & 7)] = make_float4(__uint_as_float(w[4 * i]), __uint_as_float(w[4 * i + 1]),
                                                       __uint_as_float(w[4 * i + 2]), __uint_as_float(w[4 * i + 3]));
        }
        reinterpret_cast<float2*>(smem + C::kShareO)[t * 128 + r] = make_float2(m, l);
      }
      if (!ok || nsplit > 1) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_free[k & 1]);
    }
    if (!ok) *gave_up = 1;
  }
  if (nsplit > 1) {
    // Join the shares in rank order (the result does not depend on who finished first):
    // with M the largest m, O = sum 2^((m_s - M) c) O_s / sum 2^((m_s - M) c) l_s. A warp
    // takes four rows at a time, eight lanes each. Nothing is joined once a wait of any CTA of
    // the cluster ran out: its share is not one, and its item may never have been written.
    cluster_sync();
    uint32_t any_gave_up = 0;
    for (int i = 0; i < nsplit; ++i) any_gave_up |= __float_as_uint(ld_dsmem_f1(mapa_shared(smem_u32(gave_up), i)));
    if (warp >= 4 && any_gave_up == 0) {
      const Item<KT> it = items[0];
      const float c = a.scale * 1.4426950408889634f;
      const uint32_t part = smem_u32(smem), ml = part + C::kShareO;
      const int sub = lane & 7;
      const int last = ((it.nt - 1) * 128) + min(tokens, it.ql - it.i0 - (it.nt - 1) * tokens) * g;
      for (int row = (split * 4 * NT + warp - 4) * 4 + (lane >> 3); row < last; row += nsplit * 16 * NT) {
        const int t = row >> 7, r = row & 127;
        if (r >= tokens * g) continue;
        float2 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < nsplit) x[i] = ld_dsmem_f2(mapa_shared(ml + row * 8, i));
        float mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < nsplit) mx = fmaxf(mx, x[i].x);
        float4 o[D / 32];
#pragma unroll
        for (int j = 0; j < D / 32; ++j) o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i >= nsplit) break;
          // a share that saw no key has no weight; a NaN sum is kept
          const float f = x[i].y != x[i].y ? 1.f : (x[i].x == -INFINITY ? 0.f : ex2((x[i].x - mx) * c));
          sum += f * x[i].y;
          const uint32_t src = mapa_shared(part + row * (D * 4), i);
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const float4 v = ld_dsmem_f4(src + (((sub + 8 * j) ^ (r & 7)) << 4));
            o[j].x += f * v.x;
            o[j].y += f * v.y;
            o[j].z += f * v.z;
            o[j].w += f * v.w;
          }
        }
        const float inv = mx == -INFINITY && sum == sum ? 0.f : 1.f / sum;
        const int64_t off = it.b * a.os.seq + static_cast<int64_t>(it.i0 + t * tokens + r / g) * a.os.tok +
                            static_cast<int64_t>(it.h0 + r % g) * a.os.head + 4 * sub;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + off + 32 * j) =
              make_uint2(pack2<BF16>(o[j].x * inv, o[j].y * inv), pack2<BF16>(o[j].z * inv, o[j].w * inv));
      }
    }
    cluster_sync();  // no CTA leaves while another may still read its share
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// 4-D tensor map (head_dim, heads, tokens, sequences) of a 16-bit tensor: boxes of 64 dims x
// box_heads x box_tokens, 128B swizzle, zero fill out of range.
int map_4d(CUtensorMap* m, const void* p, const Strides& st, int bf16, int D, int heads, int len, int nseq, int box_heads,
           int box_tokens) {
  const int64_t dims[4] = {D, heads, len, nseq};
  const int64_t strides[3] = {st.head * 2, st.tok * 2, st.seq * 2};
  const int box[4] = {64, box_heads, box_tokens, 1};
  return make_tmap_4d(m, p, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, dims, strides, box);
}

// Clusters of ns CTAs of the tiled kernel that the device holds at once (asked once each).
template <int D, bool BF16>
int clusters_at_once(int ns, int dev) {
  using C = WinCfg<D>;
  static std::atomic<int> known[64][9];
  int n = known[dev & 63][ns].load(std::memory_order_relaxed);
  if (ns == 1) return sm_count(dev);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ns));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ns);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, k_attn_tiles<D, BF16>, &cfg) != cudaSuccess || n <= 0) n = -1;
    known[dev & 63][ns].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <int D, bool BF16>
int launch_tiles(const AttnWindow& a, int* status, cudaStream_t s) {
  using C = WinCfg<D>;
  // query heads side by side in a tile: the largest divisor of the sharing that fits
  const int share = a.heads / a.kv_heads;
  int g = 1;
  for (int d = 2; d <= 32 && d <= share; ++d)
    if (share % d == 0) g = d;
  const int tokens = 128 / g;
  CUtensorMap tq, tk, tv, tk8, tv8;
  if (map_4d(&tk8, a.k, a.ks, a.bf16, D, a.kv_heads, a.k_len, a.nseq, 1, 8) ||
      map_4d(&tv8, a.v, a.vs, a.bf16, D, a.kv_heads, a.k_len, a.nseq, 1, 8) ||
      map_4d(&tq, a.q, a.qs, a.bf16, D, a.heads, a.q_len, a.nseq, g, tokens) ||
      map_4d(&tk, a.k, a.ks, a.bf16, D, a.kv_heads, a.k_len, a.nseq, 1, C::kKT) ||
      map_4d(&tv, a.v, a.vs, a.bf16, D, a.kv_heads, a.k_len, a.nseq, 1, C::kKT))
    return -2;
  static std::atomic<uint64_t> attr_set{0};  // one bit per device; first calls may race
  int dev = 0;
  cudaGetDevice(&dev);
  if (!((attr_set.load() >> (dev & 63)) & 1)) {
    if (cudaFuncSetAttribute(k_attn_tiles<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess)
      return -3;
    // the register split waits for registers that the launch must have
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, k_attn_tiles<D, BF16>) != cudaSuccess ||
        fa.numRegs * C::kThreads < 128 * C::kRegsCtl + 128 * C::kNT * C::kRegsSoft)
      return -5;
    attr_set.fetch_or(uint64_t(1) << (dev & 63));
  }
  // Query tiles an item, and a split of its key tiles over a cluster: whatever makes the call
  // shortest. CTAs run one an SM, so a call takes its rounds of items times an item's time,
  // with the times measured (ns a key tile for 1, 2, .. query tiles; about 4 us to set a CTA
  // up, 1.3 for another item, 5 to join shares). A view of 1297 tokens and 16 heads over 7800
  // keys: 64 items of three query tiles, each split in two, take 80 us; unsplit 149, 96 unsplit
  // items of two query tiles 133.
  constexpr int64_t kTileNs[2][3] = {{560, 770, 865}, {720, 1000, 0}};
  constexpr int64_t kSetupNs = 4000, kNextNs = 1300, kJoinNs = 5000;
  int nsplit = 1, qt = C::kNT;
  int64_t best = 0;
  for (int n = C::kNT; n >= 1; --n) {
    const int64_t items = static_cast<int64_t>((a.q_len + n * tokens - 1) / (n * tokens)) * (a.heads / g) * a.nseq;
    const int64_t reach = std::min<int64_t>(a.k_len, static_cast<int64_t>(a.left) + n * tokens + std::min(a.right, a.q_len));
    const int64_t keys = (std::min<int64_t>(a.k_len, reach + a.sinks) + C::kKT - 1) / C::kKT;  // key tiles
    for (int ns = 1; ns <= 8 && (ns == 1 || keys >= 4 * ns); ++ns) {
      const int64_t at_once = clusters_at_once<D, BF16>(ns, dev);
      if (at_once <= 0) continue;
      const int64_t rounds = (items + at_once - 1) / at_once, tile = kTileNs[D == 128][n - 1];
      const int64_t cost = ns == 1 ? kSetupNs + rounds * (keys * tile + kNextNs)
                                   : rounds * ((keys + ns - 1) / ns * tile + kSetupNs + kJoinNs);
      if (best == 0 || cost < best) {
        best = cost;
        nsplit = ns;
        qt = n;
      }
    }
  }
  const int tiles = (a.q_len + qt * tokens - 1) / (qt * tokens);
  const int64_t items = static_cast<int64_t>(tiles) * (a.heads / g) * a.nseq;
  if (items * nsplit > 0x7fffffff) return -1;
  return launch_pdl(k_attn_tiles<D, BF16>, dim3(static_cast<unsigned>(items * nsplit)), C::kThreads, C::kSmem, s,
                    static_cast<unsigned>(nsplit), tq, tk, tv, tk8, tv8, a, g, tokens, qt, tiles, nsplit, status) ==
                 cudaSuccess
             ? 0
             : -4;
}

// ------------------------------------------------------------------ few queries
// At most 16 query rows ((token, head) pairs of a key head): every visible K and V byte is
// read once and that bounds the kernel. A CTA takes one (sequence, key head), or a share of
// its keys when there are too few of those to fill the SMs: the CTAs of a cluster then join
// their sums through distributed shared memory. Key tiles of 64 arrive by TMA in a ring; each
// of four warps takes 16 keys of a tile with m16n8k16 products (the rows padded to 16; the
// tensor work is far below the memory's time, so the small warp-level form is enough) and
// keeps its own running maximum, sum and output, joined at the end. Measured: 32 tokens over
// windows of 4096 keys, 8 key heads of 128 dims (462 MB): 73 us, 6.3 TB/s or 0.96 of a copy; one
// token of 16 heads of 64 dims over 6485 keys (27 MB): 12.5 us, most of it launch, the first
// loads' latency and the join of the eight shares.
constexpr int kFewRows = 16, kFewKeys = 64, kFewWarps = 4, kFewThreads = 32 * (kFewWarps + 1);

template <int D>
struct FewCfg {
  static constexpr int kTile = kFewKeys * D * 2;           // bytes of a K or V tile
  static constexpr int kStages = D == 64 ? 6 : 3;          // about 96 KB in flight, two CTAs an SM
  static constexpr int kPartFloats = kFewRows * (D + 2);   // O rows, then maxima and sums
  static constexpr int kSmem = 1024 + kStages * 2 * kTile + 128;
  static_assert((kFewWarps + 1) * kPartFloats * 4 <= kStages * 2 * kTile, "partial sums fit the ring");
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kFewThreads, 2)
    k_attn_few(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
               const __grid_constant__ AttnWindow a, int nsplit, int* status) {
  using C = FewCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kStages * 2 * C::kTile);
  uint64_t* empty = full + C::kStages;
  uint32_t* gave_up = reinterpret_cast<uint32_t*>(empty + C::kStages);  // not 0: a wait of this CTA ran out

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = static_cast<int>(blockIdx.x) % nsplit, item = static_cast<int>(blockIdx.x) / nsplit;
  const int hk = item % a.kv_heads, b = item / a.kv_heads;
  const int share = a.heads / a.kv_heads;
  pdl_wait();
  const int ql = a.q_lens ? min(max(a.q_lens[b], 0), a.q_len) : a.q_len;
  const int kl = a.k_lens ? min(max(a.k_lens[b], 0), a.k_len) : a.k_len;
  const int rows = ql * share;
  // keys some row sees: [lo, hi] and [0, s0); tiles of the latter first
  const int hi = min(kl - 1, kl - 1 + a.right), lo = max(0, kl - ql - a.left);
  const int s0 = min(a.sinks, lo);
  const int n_sink = (s0 + kFewKeys - 1) / kFewKeys;
  const int n_all = rows == 0 || hi < 0 ? 0 : n_sink + (hi - lo + kFewKeys) / kFewKeys;
  const int n_begin = static_cast<int>(static_cast<int64_t>(split) * n_all / nsplit);
  const int n_end = static_cast<int>(static_cast<int64_t>(split + 1) * n_all / nsplit);
  auto key0 = [&](int n) { return n < n_sink ? n * kFewKeys : lo + (n - n_sink) * kFewKeys; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kFewWarps);
    }
    fence_mbar_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  __syncthreads();

  float o[D / 8][4];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
  bool ok = true;

  if (warp == kFewWarps) {
    if (lane == 0) {
      for (int n = n_begin; n < n_end; ++n) {
        const int it = n - n_begin, st = it % C::kStages;
        if (!mbar_wait(&empty[st], ((it / C::kStages) & 1) ^ 1u, status, kStatusTimeoutEmpty)) {
          drain(full, C::kStages, it, status);
          break;
        }
        mbar_arrive_expect_tx(&full[st], 2 * C::kTile);
        uint8_t* k = smem + st * 2 * C::kTile;
        for (int c = 0; c < D / 64; ++c) tma_load_4d(k + c * 8192, &tmK, &full[st], c * 64, hk, key0(n), b);
        for (int c = 0; c < D / 64; ++c) tma_load_4d(k + C::kTile + c * 8192, &tmV, &full[st], c * 64, hk, key0(n), b);
      }
    }
    __syncwarp();
  } else {
    const float c = a.scale * 1.4426950408889634f;
    // Q fragments: rows lane / 4 and + 8, dims 16 i + 2 (lane % 4) and + 8
    uint32_t q[D / 16][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = lane / 4 + 8 * j;
      const uint16_t* row = static_cast<const uint16_t*>(a.q) + b * a.qs.seq + static_cast<int64_t>(r / share) * a.qs.tok +
                            static_cast<int64_t>(hk * share + r % share) * a.qs.head;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          q[i][j + 2 * h] = r < rows ? *reinterpret_cast<const uint32_t*>(row + 16 * i + 8 * h + 2 * (lane % 4)) : 0u;
    }
    const int p0 = kl - ql + (lane / 4) / share, p1 = kl - ql + (lane / 4 + 8) / share;  // the rows' positions
    const int row_hi[2] = {min(kl - 1, p0 + a.right), min(kl - 1, p1 + a.right)}, row_lo[2] = {p0 - a.left, p1 - a.left};
    for (int n = n_begin; n < n_end; ++n) {
      const int it = n - n_begin, st = it % C::kStages, k0 = key0(n);
      ok = mbar_wait_warp(&full[st], (it / C::kStages) & 1, status, kStatusTimeoutFull);
      if (!ok) break;
      const uint32_t sK = smem_u32(smem + st * 2 * C::kTile), sV = sK + C::kTile;
      const int key_w = k0 + 16 * warp;  // this warp's first key
      // S: 16 rows x 16 keys
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      {
        const int r = 16 * warp + (lane & 7) + ((lane >> 4) << 3), ch = (lane >> 3) & 1;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t kf[4];
          ldmatrix4(sK + (i >> 2) * 8192 + r * 128 + (((2 * (i & 3) + ch) ^ (r & 7)) << 4), kf);
          mma16816<BF16>(s[0], q[i], kf[0], kf[1]);
          mma16816<BF16>(s[1], q[i], kf[2], kf[3]);
        }
      }
      // keys that no row sees: masked, and their V rows zeroed (0 * NaN)
      const bool sink_tile = n < n_sink;
      const int key_end = sink_tile ? min(s0, hi + 1) : hi + 1;
      if (key_w + 16 > key_end) {
        const int dead = max(0, key_end - key_w);  // first dead key of the warp's 16
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int chunk = lane + 32 * i, r = chunk / (D / 8), cc = chunk % (D / 8);
          if (r >= dead)
            *reinterpret_cast<uint4*>(smem + st * 2 * C::kTile + C::kTile + (cc >> 3) * 8192 + (16 * warp + r) * 128 +
                                      (cc & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      // mask by row where the tile is not seen whole by every row
      if (sink_tile || key_w + 15 > kl - ql + a.right || key_w + 16 > key_end || key_w < kl - 1 - a.left) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key_w + 8 * j + 2 * (lane % 4) + (e & 1), rr = e >> 1;
            const bool sees = key < key_end && key <= row_hi[rr] && (key >= row_lo[rr] || key < a.sinks);
            if (!sees) s[j][e] = -INFINITY;
          }
      }
      float mt[2];
#pragma unroll
      for (int rr = 0; rr < 2; ++rr) {
        mt[rr] = fmaxf(fmaxf(s[0][2 * rr], s[0][2 * rr + 1]), fmaxf(s[1][2 * rr], s[1][2 * rr + 1]));
        mt[rr] = fmaxf(mt[rr], __shfl_xor_sync(0xffffffffu, mt[rr], 1));
        mt[rr] = fmaxf(mt[rr], __shfl_xor_sync(0xffffffffu, mt[rr], 2));
      }
      if (__any_sync(0xffffffffu, mt[0] > m[0] || mt[1] > m[1])) {
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const float mn = fmaxf(m[rr], mt[rr]);
          const float alpha = m[rr] == mn ? 1.f : ex2((m[rr] - mn) * c);
          m[rr] = mn;
          l[rr] *= alpha;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            o[i][2 * rr] *= alpha;
            o[i][2 * rr + 1] *= alpha;
          }
        }
      }
      uint32_t pf[4];
#pragma unroll
      for (int rr = 0; rr < 2; ++rr) {
        const float mc = m[rr] == -INFINITY ? 0.f : m[rr] * c;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float e0 = ex2(fmaf(s[j][2 * rr], c, -mc)), e1 = ex2(fmaf(s[j][2 * rr + 1], c, -mc));
          l[rr] += e0 + e1;
          pf[rr + 2 * j] = pack2<BF16>(e0, e1);
        }
      }
      {
        const int r = 16 * warp + (lane & 15), ch = lane >> 4;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t vf[4];
          ldmatrix4_trans(sV + (i >> 2) * 8192 + r * 128 + (((2 * (i & 3) + ch) ^ (r & 7)) << 4), vf);
          mma16816<BF16>(o[2 * i], pf, vf[0], vf[1]);
          mma16816<BF16>(o[2 * i + 1], pf, vf[2], vf[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
      l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 1);
      l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 2);
    }
  }

  // Join the warps: each leaves O, maxima and sums in the ring (every tile has been read).
  // part[w]: [16][D], then [16] maxima, [16] sums; part[kFewWarps] is the CTA's.
  uint32_t bad = __syncthreads_or(!ok);
  if (threadIdx.x == 0) *gave_up = bad;
  float* part = reinterpret_cast<float*>(smem);
  if (warp < kFewWarps) {
    float* w = part + warp * C::kPartFloats;
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int rr = 0; rr < 2; ++rr)
        *reinterpret_cast<float2*>(w + (lane / 4 + 8 * rr) * D + 8 * i + 2 * (lane % 4)) =
            make_float2(o[i][2 * rr], o[i][2 * rr + 1]);
    if (lane % 4 == 0) {
#pragma unroll
      for (int rr = 0; rr < 2; ++rr) {
        w[kFewRows * D + lane / 4 + 8 * rr] = m[rr];
        w[kFewRows * D + kFewRows + lane / 4 + 8 * rr] = l[rr];
      }
    }
  }
  __syncthreads();
  const float c = a.scale * 1.4426950408889634f;
  // weights of n partial sums with maxima m_i, in order: 2^((m_i - max) c), 0 for one that
  // saw no key; max over finite scores only where there is one
  auto weight = [&](float mi, float mx) { return mi == -INFINITY ? 0.f : ex2((mi - mx) * c); };
  float* mine = part + kFewWarps * C::kPartFloats;
  for (int e = threadIdx.x; e < kFewRows * D / 2; e += kFewThreads) {
    const int r = e / (D / 2), d = e % (D / 2) * 2;
    float mx = -INFINITY, sum = 0.f;
    float2 v = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) mx = fmaxf(mx, part[w * C::kPartFloats + kFewRows * D + r]);
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float* pw = part + w * C::kPartFloats;
      const float lw = pw[kFewRows * D + kFewRows + r];
      // a NaN sum (NaN scores only: the maximum passed them by) is kept
      const float f = lw == lw ? weight(pw[kFewRows * D + r], mx) : 1.f;
      sum += f * lw;
      const float2 x = *reinterpret_cast<const float2*>(pw + r * D + d);
      v.x += f * x.x;
      v.y += f * x.y;
    }
    *reinterpret_cast<float2*>(mine + r * D + d) = v;
    if (d == 0) {
      mine[kFewRows * D + r] = mx;
      mine[kFewRows * D + kFewRows + r] = sum;
    }
  }
  if (nsplit > 1) cluster_sync();
  else __syncthreads();
  // Join the CTAs of the cluster in rank order; each writes its share of the elements, unless a
  // wait of any of them ran out.
  if (nsplit > 1)
    for (int i = 0; i < nsplit; ++i) bad |= __float_as_uint(ld_dsmem_f1(mapa_shared(smem_u32(gave_up), i)));
  if (bad == 0) {
    const uint32_t base = smem_u32(mine);
    const int pairs = rows * D / 2;
    for (int e = split * kFewThreads + static_cast<int>(threadIdx.x); e < pairs; e += nsplit * kFewThreads) {
      const int r = e / (D / 2), d = e % (D / 2) * 2;
      float mx = -INFINITY, sum = 0.f;
      float2 v = make_float2(0.f, 0.f);
      if (nsplit == 1) {
        mx = mine[kFewRows * D + r];
        sum = mine[kFewRows * D + kFewRows + r];
        v = *reinterpret_cast<const float2*>(mine + r * D + d);
      } else {
        for (int i = 0; i < nsplit; ++i) mx = fmaxf(mx, ld_dsmem_f1(mapa_shared(base + 4 * (kFewRows * D + r), i)));
        for (int i = 0; i < nsplit; ++i) {
          const float li = ld_dsmem_f1(mapa_shared(base + 4 * (kFewRows * D + kFewRows + r), i));
          const float mi = ld_dsmem_f1(mapa_shared(base + 4 * (kFewRows * D + r), i));
          const float2 x = ld_dsmem_f2(mapa_shared(base + 4 * (r * D + d), i));
          const float f = li == li ? weight(mi, mx) : 1.f;
          sum += f * li;
          v.x += f * x.x;
          v.y += f * x.y;
        }
      }
      const float inv = mx == -INFINITY && sum == sum ? 0.f : 1.f / sum;  // no key seen: zeros
      const int64_t off = b * a.os.seq + static_cast<int64_t>(r / share) * a.os.tok +
                          static_cast<int64_t>(hk * share + r % share) * a.os.head + d;
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + off) = pack2<BF16>(v.x * inv, v.y * inv);
    }
  }
  if (nsplit > 1) cluster_sync();  // no CTA leaves while another may still read its sums
}

template <int D, bool BF16>
int launch_few(const AttnWindow& a, int* status, cudaStream_t s) {
  using C = FewCfg<D>;
  CUtensorMap tk, tv;
  if (map_4d(&tk, a.k, a.ks, a.bf16, D, a.kv_heads, a.k_len, a.nseq, 1, kFewKeys) ||
      map_4d(&tv, a.v, a.vs, a.bf16, D, a.kv_heads, a.k_len, a.nseq, 1, kFewKeys))
    return -2;
  static std::atomic<uint64_t> attr_set{0};  // one bit per device; first calls may race
  int dev = 0;
  cudaGetDevice(&dev);
  if (!((attr_set.load() >> (dev & 63)) & 1)) {
    if (cudaFuncSetAttribute(k_attn_few<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess)
      return -3;
    attr_set.fetch_or(uint64_t(1) << (dev & 63));
  }
  // Split the keys while the SMs' two slots each are not full and a share keeps four tiles
  // (of the longest window that the sizes allow; lengths are on the device).
  const int64_t items = static_cast<int64_t>(a.nseq) * a.kv_heads;
  const int64_t window = static_cast<int64_t>(a.left) + a.q_len + a.sinks;
  const int64_t tiles = (std::min<int64_t>(a.k_len, window) + kFewKeys - 1) / kFewKeys;
  const int64_t slots = 2 * static_cast<int64_t>(sm_count(dev));
  const int nsplit = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({8, slots / items, tiles / 4})));
  if (items * nsplit > 0x7fffffff) return -1;
  return launch_pdl(k_attn_few<D, BF16>, dim3(static_cast<unsigned>(items * nsplit)), kFewThreads, C::kSmem, s,
                    static_cast<unsigned>(nsplit), tk, tv, a, nsplit, status) == cudaSuccess
             ? 0
             : -4;
}

// No keys at all (k_len 0; a tensor map cannot be empty): zeros in the rows that count.
__global__ void k_attn_none(const AttnWindow a) {
  pdl_wait();
  const int64_t per_row = a.head_dim / 8;
  const int64_t n = static_cast<int64_t>(a.nseq) * a.q_len * a.heads * per_row;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < n;
       e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = e / per_row;
    const int h = static_cast<int>(row % a.heads), i = static_cast<int>(row / a.heads % a.q_len);
    const int b = static_cast<int>(row / a.heads / a.q_len);
    if (a.q_lens && i >= a.q_lens[b]) continue;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + b * a.os.seq + i * a.os.tok + h * a.os.head +
                              e % per_row * 8) = make_uint4(0u, 0u, 0u, 0u);
  }
}

}  // namespace

template <int D, bool BF16>
static int run(const AttnWindow& a, int* status, cudaStream_t s) {
  // few rows for each key head: the memory-bound kernel (its tensor work is padded to 16 rows,
  // the tiled kernel's to 128 a query tile). 32 single tokens, 8 key heads of 128 dims, windows
  // of 4096: 16 rows a key head here 87 us, 17 rows there 120; 16 key heads of 64 dims over 6485
  // keys: 16 queries here 14 us, 17 there 21.
  if (static_cast<int64_t>(a.q_len) * (a.heads / a.kv_heads) <= kFewRows) return launch_few<D, BF16>(a, status, s);
  return launch_tiles<D, BF16>(a, status, s);
}

int attention_window(const AttnWindow& a, int* status, cudaStream_t s) {
  if (a.k_len == 0) return launch_pdl(k_attn_none, dim3(256), 256, 0, s, 1, a) == cudaSuccess ? 0 : -4;
  if (a.bf16) return a.head_dim == 64 ? run<64, true>(a, status, s) : run<128, true>(a, status, s);
  return a.head_dim == 64 ? run<64, false>(a, status, s) : run<128, false>(a, status, s);
}

}  // namespace da3b

using namespace da3b;

// Strides of a tensor of the given sizes: multiples of 8 elements, positive (a stride of
// a size of one is never used, and set to one token or head so that nothing depends on it).
static bool take_strides(const int64_t* in, int nseq, int len, int heads, int D, Strides* st) {
  *st = {in[0], in[1], in[2]};
  if (heads == 1) st->head = D;
  if (len == 1) st->tok = static_cast<int64_t>(heads) * D;
  if (nseq == 1) st->seq = static_cast<int64_t>(len) * heads * D;
  const int64_t most = int64_t(1) << 38;  // tensor maps hold strides below 2^40 bytes
  for (int64_t v : {st->seq, st->tok, st->head})
    if (v < D || v % 8 || v >= most) return false;
  return true;
}

extern "C" {

DA3B_API int da3b_attention_window(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                   const void* v, const int64_t* v_strides, void* out, const int64_t* out_strides,
                                   int dtype, int nseq, int q_len, int k_len, int heads, int kv_heads, int head_dim,
                                   const int* q_lens, const int* k_lens, int left, int right, int sinks, float scale,
                                   void* stream) {
  if ((dtype != 0 && dtype != 1) || nseq < 0 || q_len < 0 || k_len < 0 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads || (head_dim != 64 && head_dim != 128) || sinks < 0 || !(scale >= 0.f) || isinf(scale))
    return -100;
  if (q_len > kWindowAll || k_len > kWindowAll) return -1;
  if (nseq == 0 || q_len == 0) return 0;
  if (!q || !out || !q_strides || !k_strides || !v_strides || !out_strides || (k_len > 0 && (!k || !v))) return -100;
  AttnWindow a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.bf16 = dtype;
  a.nseq = nseq;
  a.q_len = q_len;
  a.k_len = k_len;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.head_dim = head_dim;
  a.q_lens = q_lens;
  a.k_lens = k_lens;
  a.left = left < 0 || left > kWindowAll ? kWindowAll : left;
  a.right = right < 0 || right > kWindowAll ? kWindowAll : right;
  a.sinks = sinks;
  // At 0 a masked score (-inf) times it would be NaN. Times the smallest float any f32 score is
  // below 2^-20, and every weight 1.
  a.scale = fmaxf(scale, FLT_TRUE_MIN);
  if (!take_strides(q_strides, nseq, q_len, heads, head_dim, &a.qs) ||
      (k_len > 0 && (!take_strides(k_strides, nseq, k_len, kv_heads, head_dim, &a.ks) ||
                     !take_strides(v_strides, nseq, k_len, kv_heads, head_dim, &a.vs))) ||
      !take_strides(out_strides, nseq, q_len, heads, head_dim, &a.os))
    return -1;
  for (const void* p : {q, k, v, static_cast<const void*>(out)})
    if (reinterpret_cast<uintptr_t>(p) & 15) return -1;
  for (const int* p : {q_lens, k_lens})
    if (reinterpret_cast<uintptr_t>(p) & 3) return -1;
  // 32-bit work counts inside
  if (static_cast<double>(nseq) * heads * q_len > 2147483647.0 * 8) return -1;
  if (!usable_here({q, k_len > 0 ? k : nullptr, k_len > 0 ? v : nullptr, out, q_lens, k_lens})) return -104;
  int* st = device_status_word();
  if (!st) return -101;
  return attention_window(a, st, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
