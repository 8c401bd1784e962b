// Backward of the training attention under a sliding window with sinks (abkv_window_attention_backward) on
// 5th-generation tensor cores (tcgen05 + TMEM) for sm_100a.
//
// Row i sees keys j <= i with j > i - window or j < n_sink.  With P = exp(scale q k^T - lse) on the visible
// pairs (lse from the forward), dP = dO V^T and Di = rowsum(dO * O):
//   dS = P (dP - Di)      dV = sum P^T dO      dK = scale sum dS^T Q      dQ = scale dS K
//
// Two kernels instead of one.  A key-stationary kernel (dK, dV: four products a tile) and a query-stationary one
// (dQ: three) recompute S and dP once each -- seven products a tile instead of five -- but every sum stays in TMEM:
// no fp32 accumulator of dQ in memory (its zeroing, a 64 KiB reduction per tile pair, its conversion) and no order-
// dependent additions, so all gradients repeat bit for bit.  Measured at 2 x 32 heads (8 KV heads) x 4096 rows x
// 128 dims: window 1024, row sums 29 us, dK/dV 265 us, dQ 200 us; no window, dK/dV 486 us, dQ 378 us (0.9 PFLOP/s
// of the visible pairs' products with the window, 1.1 without, of 1.63 for a library product).  A tile takes a dQ
// CTA about 4000 clocks against 1536 of products: the hand-overs between the issuer and the threads (about 200
// clocks each way) and the threads' element-wise work in between bound both kernels, not a pipe.
//
// Both work on 128 x 128 tiles (S and dP products with N = 128: with N = 64 the operands' shared-memory reads,
// not the tensor core, set the pace).  18 warps: 0 the TMA producer, 1 the issuer of tcgen05.mma and owner of the
// TMEM, 2..17 threads of TMEM lanes -- warp group cg = (warp - 2) / 4 takes columns [32 cg, 32 cg + 32) of
// every tile, the warp's lane quarter 32 of its rows, and puts its bf16 operands (16 columns) over the scores it has
// read itself, so no warp waits for another: the products take each 16-row step's operand where it lies.  The
// element-wise half of a tile (16,384 exponentials, 1024 clocks) runs beside the products of its neighbours:
//   dK/dV:  S(0) dP(0) | dV(u) S(u+1) | dK(u) dP(u+1) | ...    threads: P(u) then dS(u)
//   dQ:     S(0) dP(0) S(1) | dP(u+1) | dQ(u) S(u+2) | ...     threads: P(u), dP(u) in registers, dS(u) over S(u)
// Every mbarrier wait is bounded and records ABKV_DEVERR_TIMEOUT on expiry.
#include <algorithm>
#include <cstring>

#include "tcgen05.cuh"

namespace abkv {
namespace {
using namespace tc;

constexpr int kT = 128;          // tile rows (keys and queries)
constexpr int kThreads = 576;    // 18 warps
constexpr int kWorkers = 16;     // warps of TMEM lanes, one arrival each
constexpr int kLong = 3, kShort = 2;  // ring depth of the operand used twice, and of the one released early
constexpr uint32_t kIdescS = idesc_bf16_m128(kT, false);
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct Lay {
  static constexpr int kAtoms = D / 64;
  static constexpr int kTile = kT * D * 2;         // [128][D] bf16: D / 64 atom columns of [128 rows][128 B]
  static constexpr int kAtom = kTile / kAtoms;
  static constexpr int kOffA = 0;                  // stationary operands (K, V or Q, dO)
  static constexpr int kOffB = kTile;
  static constexpr int kOffLong = 2 * kTile;       // Q (dK/dV kernel) or K (dQ kernel)
  static constexpr int kOffShort = kOffLong + kLong * kTile;  // dO or V
  static constexpr int kOffStat = kOffShort + kShort * kTile;  // [2 tiles][4 column groups][lse2, di][32]
  static constexpr int kOffBar = kOffStat + 2 * 4 * 2 * 32 * 4;
  static constexpr int kSmem = kOffBar + 512;      // the base is 1024-byte aligned (checked by the kernels)
  static constexpr int kRedStride = D + 4;         // fp32 rows of the cluster reduction (in the rings)
  static constexpr uint32_t kIdescAcc = idesc_bf16_m128(D, true);
};
static_assert(Lay<128>::kSmem <= 227 * 1024, "shared memory");
static_assert(2 * kT * Lay<128>::kRedStride * 4 <= (kLong + kShort) * Lay<128>::kTile, "cluster reduction");
static_assert(2 * kT * Lay<64>::kRedStride * 4 <= (kLong + kShort) * Lay<64>::kTile, "cluster reduction");

// barriers: stationary operands, long ring full / empty, short ring full / empty, S full (two in the dQ kernel), dP
// full, P ready (dQ: dP read), dS ready (two in the dQ kernel), accumulators complete / drained, statistics [column
// group][buffer], stationary operands released, work item full / empty (two deep), then the TMEM address and the
// items.  One barrier per buffer wherever an arrival may be a pair ahead of a wait (a parity wait cannot tell phases 2
// apart): the statistics' writer runs ahead of their readers, and dS(u+1) may be ready before the issuer, which put
// dP(u+1) under way before it, has looked at dS(u).
constexpr int kBarA = 0, kBarLF = 1, kBarLE = kBarLF + kLong, kBarSF = kBarLE + kLong, kBarSE = kBarSF + kShort,
              kBarS = kBarSE + kShort, kBarDP = kBarS + 2, kBarP = kBarDP + 1, kBarDS = kBarP + 1,
              kBarAcc = kBarDS + 2, kBarDrain = kBarAcc + 1, kBarStat = kBarDrain + 1, kBarAE = kBarStat + 8,
              kBarIF = kBarAE + 1, kBarIE = kBarIF + 2, kBarTmem = kBarIE + 2, kBarItem = kBarTmem + 1;
static_assert((kBarItem + 1) * 8 <= 512, "barrier area");

struct alignas(64) WinBwdParams {
  CUtensorMap tm_q, tm_k, tm_v, tm_do;
  const float* lse;  // [B][H][S], natural log
  const float* di;   // [B][H][S]
  __nv_bfloat16 *dq, *dk, *dv;
  int64_t dq_sb, dq_sh, dq_ss, dk_sb, dk_sh, dk_ss, dv_sb, dv_sh, dv_ss;
  int32_t* err;
  int32_t* work;     // next work item of the dK/dV launch (zeroed by the row-sum kernel)
  int B, H, Hkv, G, S, n_tiles, window, n_sink;
  int cluster, tile0, tiles;  // dK/dV launch: CTAs per key tile; its key tiles
  int first;                  // the launch that waits for the row sums
  float scale, scale_log2;
};

__device__ __forceinline__ uint32_t below(int n) {  // bits [0, n)
  return n >= 32 ? 0xFFFFFFFFu : (n <= 0 ? 0u : ((1u << n) - 1u));
}

template <int D>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, int row, int head, int b, uint64_t* bar) {
#pragma unroll
  for (int a = 0; a < Lay<D>::kAtoms; ++a) tma_load_4d(dst + a * Lay<D>::kAtom, map, 64 * a, row, head, b, bar);
}

// Position in a ring of N slots and the parity of its use.
template <int N>
struct Pos {
  int i = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void step() {
    if (++i == N) {
      i = 0;
      ph ^= 1u;
    }
  }
};

// D(128 x 128) = A B^T over head_dim, both K-major tiles in shared memory (descriptors).
template <int D>
__device__ __forceinline__ void issue_scores(uint32_t tmem, uint64_t da, uint64_t db) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint32_t off = (kk >> 2) * Lay<D>::kAtom + (kk & 3) * 32;
    umma(tmem, desc_advance(da, off), desc_advance(db, off), kIdescS, kk > 0 ? 1u : 0u);
  }
}
// D(128 x head_dim) += A B: A bf16 in TMEM (128 x 128, 32 of its columns in 16 words every 32 words), B a [128][D]
// tile read MN-major (descriptor).
template <int D>
__device__ __forceinline__ void issue_accumulate(uint32_t tmem, uint32_t a, uint64_t db, bool first) {
#pragma unroll
  for (int kk = 0; kk < kT / 16; ++kk)
    umma_tmem_a(tmem, a + (kk >> 1) * 32 + (kk & 1) * 8, desc_advance(db, kk * 2048), Lay<D>::kIdescAcc,
                (!first || kk > 0) ? 1u : 0u);
}

__device__ __forceinline__ void alloc_tmem(uint32_t* s_tmem) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(s_tmem)), "r"(512u));
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
}

// (a - b) * c on pairs.
__device__ __forceinline__ void sub_mul_pair(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0,
                                             float c1) {
  asm("{\n .reg .b64 x, y, z, r;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " sub.rn.f32x2 r, x, y;\n mul.rn.f32x2 r, r, z;\n mov.b64 {%0, %1}, r;\n}\n"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}

// w = bf16 roundings of the pair a, b; returns those of what they leave out.
__device__ __forceinline__ uint32_t pack_rest(uint32_t w, float a, float b) {
  return pack_bf16x2(a - __uint_as_float(w << 16), b - __uint_as_float(w & 0xFFFF0000u));
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::: "memory");
}
__device__ __forceinline__ float4 peer_ld4(uint32_t local, int rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(local), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
  return v;
}

// ---------------------------------------------------------------------------
// dK and dV.  A work item is a 128-key tile of one KV head: all (query tile, head) pairs that see it.  Without
// clusters a CTA per SM takes items from a counter, longest first, and the next item's operands and first scores are
// under way while the finished accumulators are read out.  With p.cluster > 1 (idle SMs, or the sinks' tiles, which
// every query tile sees) a cluster takes one item, its CTAs share the pairs and add their parts, in rank order,
// through shared memory.
template <int D, bool kRest>
__global__ void __launch_bounds__(kThreads, 1) window_dkdv_kernel(const __grid_constant__ WinBwdParams p) {
  using LY = Lay<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // the 128B swizzle needs it; the same answer in every thread of the launch
    if (threadIdx.x == 0) set_error(p.err, ABKV_DEVERR_RANGE);
    return;
  }
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + LY::kOffBar);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bar + kBarTmem);
  volatile int32_t* s_item = reinterpret_cast<volatile int32_t*>(bar + kBarItem);  // [2]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % p.cluster;
  const int heads = p.Hkv * p.B, n_items = heads * p.tiles;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kBarTmem; ++i)
      mbar_init(&bar[i], (i == kBarP || i == kBarDS || i == kBarDrain) ? kWorkers
                                                                       : (i >= kBarIE && i < kBarIE + 2 ? kWorkers + 1 : 1));
  }
  if (warp == 1) alloc_tmem(s_tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // The row sums are complete before the first launch goes on, and the others start after all of its CTAs have: they
  // need nothing of one another.
  if (p.first) asm volatile("griddepcontrol.wait;\n" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const uint32_t tmem = *s_tmem;  // S^T [0,128), dP^T [128,256), dV [256,..), dK [384,..)
  bool dead = false;

  // Work item `it` of this CTA (every role asks in turn): false when there is none.
  struct Item {
    int kt, hk, b, n;
  };
  auto decode = [&](int i, Item& x) {
    x.kt = p.tile0 + i / heads;  // longest first
    const int r = i % heads;
    x.hk = r % p.Hkv;
    x.b = r / p.Hkv;
    // query tiles kt .. last see the key tile (its last key k: queries < k + window); the sinks' tiles: all
    int last = p.n_tiles - 1;
    if (x.kt * kT >= p.n_sink) last = min(last, (min(x.kt * kT + kT, p.S) - 1 + p.window - 1) / kT);
    const int pairs = (last - x.kt + 1) * p.G;
    x.n = pairs > rank ? (pairs - rank - 1) / p.cluster + 1 : 0;  // this CTA's
  };
  auto next_item = [&](int it, Item& x) -> bool {
    if (p.cluster > 1) {
      if (it > 0) return false;
      decode(blockIdx.x / p.cluster, x);
      return true;
    }
    const int slot = it & 1;
    if (!wait_or_abort(&bar[kBarIF + slot], (uint32_t)((it >> 1) & 1), dead, p.err)) return false;
    const int i = s_item[slot];
    if (i < 0) return false;
    decode(i, x);
    return true;
  };
  auto done_item = [&](int it) {  // by one thread of a role: it has decoded the item
    if (p.cluster == 1) mbar_arrive_one(&bar[kBarIE + (it & 1)]);
  };
  auto pair_at = [&](const Item& x, int u, int& qt, int& h) {
    const int i = rank + u * p.cluster;
    qt = x.kt + i / p.G;
    h = x.hk * p.G + i % p.G;
  };

  if (warp == 0) {
    if (elect_one()) {
      Item x;
      Pos<kLong> l;
      Pos<kShort> sh;
      for (int it = 0; !dead; ++it) {
        if (p.cluster > 1) {
          if (!next_item(it, x)) break;
        } else {
          // take the next item and hand it to the other roles
          const int slot = it & 1;
          if (!wait_or_abort(&bar[kBarIE + slot], (uint32_t)(((it >> 1) & 1) ^ 1), dead, p.err)) break;
          const int i = atomicAdd(p.work, 1);
          s_item[slot] = i < n_items ? i : -1;
          mbar_arrive_one(&bar[kBarIF + slot]);
          if (i >= n_items) break;
          decode(i, x);
        }
        if (x.n == 0) continue;
        // the previous item's last products over K and V have run
        if (!wait_or_abort(&bar[kBarAE], (uint32_t)((it & 1) ^ 1), dead, p.err)) break;
        mbar_expect_tx(&bar[kBarA], 2 * LY::kTile);
        load_tile<D>(smem + LY::kOffA, &p.tm_k, x.kt * kT, x.hk, x.b, &bar[kBarA]);
        load_tile<D>(smem + LY::kOffB, &p.tm_v, x.kt * kT, x.hk, x.b, &bar[kBarA]);
        for (int u = 0; u < x.n; ++u) {
          int qt, h;
          pair_at(x, u, qt, h);
          if (!wait_or_abort(&bar[kBarLE + l.i], l.ph ^ 1u, dead, p.err)) break;
          mbar_expect_tx(&bar[kBarLF + l.i], LY::kTile);
          load_tile<D>(smem + LY::kOffLong + l.i * LY::kTile, &p.tm_q, qt * kT, h, x.b, &bar[kBarLF + l.i]);
          l.step();
          if (!wait_or_abort(&bar[kBarSE + sh.i], sh.ph ^ 1u, dead, p.err)) break;
          mbar_expect_tx(&bar[kBarSF + sh.i], LY::kTile);
          load_tile<D>(smem + LY::kOffShort + sh.i * LY::kTile, &p.tm_do, qt * kT, h, x.b, &bar[kBarSF + sh.i]);
          sh.step();
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint64_t kStep = LY::kTile >> 4;  // a ring slot on, in a descriptor
      const uint64_t dk = desc_kmajor_sw128(smem_u32(smem + LY::kOffA));
      const uint64_t dv = desc_kmajor_sw128(smem_u32(smem + LY::kOffB));
      const uint64_t q_k = desc_kmajor_sw128(smem_u32(smem + LY::kOffLong));
      const uint64_t do_k = desc_kmajor_sw128(smem_u32(smem + LY::kOffShort));
      const uint64_t q_mn = desc_mnmajor_sw128(smem_u32(smem + LY::kOffLong), LY::kAtom);
      const uint64_t do_mn = desc_mnmajor_sw128(smem_u32(smem + LY::kOffShort), LY::kAtom);
      Pos<kLong> qf, qe;    // next Q to read for scores; Q of the current pair
      Pos<kShort> df, de;   // likewise dO
      uint32_t par = 0, it_par = 0;
      auto scores = [&]() -> bool {  // S^T of the next pair
        if (!wait_or_abort(&bar[kBarLF + qf.i], qf.ph, dead, p.err)) return false;
        tc_fence_after();
        issue_scores<D>(tmem, dk, q_k + qf.i * kStep);
        umma_commit(&bar[kBarS]);
        qf.step();
        return true;
      };
      auto dscores = [&]() -> bool {  // dP^T of the next pair
        if (!wait_or_abort(&bar[kBarSF + df.i], df.ph, dead, p.err)) return false;
        tc_fence_after();
        issue_scores<D>(tmem + 128, dv, do_k + df.i * kStep);
        umma_commit(&bar[kBarDP]);
        df.step();
        return true;
      };
      Item x;
      for (int it = 0; next_item(it, x); ++it) {
        done_item(it);
        if (x.n == 0) continue;
        if (!wait_or_abort(&bar[kBarA], it_par, dead, p.err) || !scores() || !dscores()) break;
        if (x.n == 1) umma_commit(&bar[kBarAE]);
        for (int u = 0; u < x.n; ++u, par ^= 1u) {
          // P^T is ready: dV, then the next scores over it (one thread's MMAs run in issue order)
          if (!wait_or_abort(&bar[kBarP], par, dead, p.err)) break;
          // the first product of an item overwrites dV and dK: the previous ones have been read out
          if (u == 0 && it > 0 && !wait_or_abort(&bar[kBarDrain], it_par ^ 1u, dead, p.err)) break;
          tc_fence_after();
          issue_accumulate<D>(tmem + 256, tmem, do_mn + de.i * kStep, u == 0);
          umma_commit(&bar[kBarSE + de.i]);  // dO's last use
          de.step();
          if (u + 1 < x.n && !scores()) break;
          if (!wait_or_abort(&bar[kBarDS], par, dead, p.err)) break;
          tc_fence_after();
          issue_accumulate<D>(tmem + 384, tmem + 128, q_mn + qe.i * kStep, u == 0);
          if (kRest) issue_accumulate<D>(tmem + 384, tmem + 128 + 16, q_mn + qe.i * kStep, false);
          umma_commit(&bar[kBarLE + qe.i]);
          qe.step();
          if (u + 1 < x.n && !dscores()) break;
          if (u + 2 == x.n) umma_commit(&bar[kBarAE]);  // the item's last scores are issued: K and V are free then
        }
        if (dead) break;
        umma_commit(&bar[kBarAcc]);
        it_par ^= 1u;
      }
    }
  } else {
    const int sw = warp - 2, cg = sw >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    // the four warps of a column group share its queries' statistics: quarter 0 writes them, two tiles deep
    float* stat = reinterpret_cast<float*>(smem + LY::kOffStat) + cg * 64;
    const float sl2 = p.scale_log2;
    const bool stager = quarter == 0;
    Item x;
    int g = 0;
    for (int it = 0;; ++it) {
      const bool more = next_item(it, x);
      if (!__all_sync(0xffffffffu, more)) break;
      __syncwarp();
      if (lane == 0) done_item(it);
      const int key = x.kt * kT + row;
      const bool sink = key < p.n_sink;
      // lane c holds the statistics of the next pair's query 32 cg + c
      float n_lse = 0.f, n_di = 0.f;
      auto fetch = [&](int u) {
        int qt, h;
        pair_at(x, u, qt, h);
        const int q = qt * kT + 32 * cg + lane;
        const int64_t r = ((int64_t)x.b * p.H + h) * p.S + q;
        n_lse = q < p.S ? __ldg(p.lse + r) * -kLog2e : 0.f;  // staged negated: an addend of the exponent
        n_di = q < p.S ? __ldcg(p.di + r) : 0.f;
      };
      const int g_item = g;
      auto stage = [&](int u) {  // statistics of pair u into its buffer, then fetch those of pair u + 1
        const int buf = (g_item + u) & 1;
        stat[buf * 256 + lane] = n_lse;
        stat[buf * 256 + 32 + lane] = n_di;
        __syncwarp();
        if (lane == 0) mbar_arrive_one(&bar[kBarStat + 2 * cg + buf]);
        if (u + 1 < x.n) fetch(u + 1);
      };
      if (stager && x.n > 0) {
        fetch(0);
        stage(0);
      }
      for (int u = 0; u < x.n; ++u, ++g) {
        const uint32_t par = (uint32_t)(g & 1);
        int qt, h;
        pair_at(x, u, qt, h);
        const float *s_lse = stat + (g & 1) * 256, *s_di = s_lse + 32;
        // visible queries of this key among the warp's 32: q >= key, q < key + window (or a sink), q < S
        const int q0 = qt * kT + 32 * cg;
        const int e = sink ? p.S : min(p.S, key + p.window);
        const uint32_t mask = below(e - q0) & ~below(key - q0);
        const bool full = __all_sync(0xffffffffu, mask == 0xFFFFFFFFu);
        bool ok = __all_sync(0xffffffffu, wait_or_abort(&bar[kBarStat + 2 * cg + (g & 1)], (uint32_t)((g >> 1) & 1), dead,
                                                            p.err) &&
                                              wait_or_abort(&bar[kBarS], par, dead, p.err));
        if (!ok) dead = true;
        tc_fence_after();
        float pv[32];
        uint32_t w[16];
        if (ok) {
          tmem_ld32(tmem + lane_base + 32 * cg, pv);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 l = *reinterpret_cast<const float4*>(s_lse + c);
            ffma2(pv[c], pv[c + 1], pv[c], pv[c + 1], sl2, l.x, l.y);
            ffma2(pv[c + 2], pv[c + 3], pv[c + 2], pv[c + 3], sl2, l.z, l.w);
#pragma unroll
            for (int j = 0; j < 4; ++j) pv[c + j] = fast_exp2(pv[c + j]);
          }
          if (!full) {
#pragma unroll
            for (int c = 0; c < 32; ++c) pv[c] = (mask >> c) & 1u ? pv[c] : 0.f;
          }
#pragma unroll
          for (int c = 0; c < 16; ++c) w[c] = pack_bf16x2(pv[2 * c], pv[2 * c + 1]);
          if (q0 == 0) pv[0] = 0.f;  // query 0 sees one key: P = 1, dS = 0 exactly (also where every query does: scale)
          tmem_st16(tmem + lane_base + 32 * cg, w);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_one(&bar[kBarP]);
        ok = __all_sync(0xffffffffu, wait_or_abort(&bar[kBarDP], par, dead, p.err));
        if (!ok) dead = true;
        // dP(u) followed every warp's dS(u - 1): nobody reads the other statistics buffer any more
        if (stager && u + 1 < x.n) stage(u + 1);
        tc_fence_after();
        if (ok) {
          float dp[32];
          tmem_ld32(tmem + lane_base + 128 + 32 * cg, dp);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 d = *reinterpret_cast<const float4*>(s_di + c);
            sub_mul_pair(dp[c], dp[c + 1], dp[c], dp[c + 1], d.x, d.y, pv[c], pv[c + 1]);
            sub_mul_pair(dp[c + 2], dp[c + 3], dp[c + 2], dp[c + 3], d.z, d.w, pv[c + 2], pv[c + 3]);
            w[c / 2] = pack_bf16x2(dp[c], dp[c + 1]);
            w[c / 2 + 1] = pack_bf16x2(dp[c + 2], dp[c + 3]);
            if (kRest) {
              dp[c / 2] = __uint_as_float(pack_rest(w[c / 2], dp[c], dp[c + 1]));
              dp[c / 2 + 1] = __uint_as_float(pack_rest(w[c / 2 + 1], dp[c + 2], dp[c + 3]));
            }
          }
          tmem_st16(tmem + lane_base + 128 + 32 * cg, w);
          if (kRest) {
#pragma unroll
            for (int c = 0; c < 16; ++c) w[c] = __float_as_uint(dp[c]);
            tmem_st16(tmem + lane_base + 128 + 16 + 32 * cg, w);
          }
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_one(&bar[kBarDS]);
      }
      if (x.n > 0) {
        if (!__all_sync(0xffffffffu, wait_or_abort(&bar[kBarAcc], (uint32_t)(it & 1), dead, p.err))) dead = true;
        tc_fence_after();
      }
      // dV (cg 0, 1) and dK (cg 2, 3): this warp's D / 2 columns of its rows
      const bool is_dk = cg >= 2;
      const int c0 = (cg & 1) * (D / 2);
      const uint32_t col = (is_dk ? 384u : 256u) + c0;
      const float gs = is_dk ? p.scale : 1.f;
      float* red = reinterpret_cast<float*>(smem + LY::kOffLong) + ((is_dk ? kT : 0) + row) * LY::kRedStride;
      __nv_bfloat16* out = is_dk ? p.dk + (int64_t)x.b * p.dk_sb + (int64_t)x.hk * p.dk_sh + (int64_t)key * p.dk_ss
                                 : p.dv + (int64_t)x.b * p.dv_sb + (int64_t)x.hk * p.dv_sh + (int64_t)key * p.dv_ss;
#pragma unroll
      for (int c = 0; c < D / 2; c += 32) {
        float t[32];
        if (x.n > 0) {
          tmem_ld32(tmem + lane_base + col + c, t);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) t[j] = 0.f;
        }
        if (c + 32 == D / 2) {  // the accumulators are in registers
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_one(&bar[kBarDrain]);
        }
        if (p.cluster > 1) {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<float4*>(red + c0 + c + j) = make_float4(t[j], t[j + 1], t[j + 2], t[j + 3]);
        } else if (key < p.S && !dead) {
#pragma unroll
          for (int v8 = 0; v8 < 4; ++v8) {
            uint4 pk;
            pk.x = pack_bf16x2(t[v8 * 8 + 0] * gs, t[v8 * 8 + 1] * gs);
            pk.y = pack_bf16x2(t[v8 * 8 + 2] * gs, t[v8 * 8 + 3] * gs);
            pk.z = pack_bf16x2(t[v8 * 8 + 4] * gs, t[v8 * 8 + 5] * gs);
            pk.w = pack_bf16x2(t[v8 * 8 + 6] * gs, t[v8 * 8 + 7] * gs);
            *reinterpret_cast<uint4*>(out + c0 + c + v8 * 8) = pk;
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u));
  if (p.cluster > 1) {
    Item x;
    decode(blockIdx.x / p.cluster, x);
    cluster_barrier();
    // this CTA's share of the rows of [dV; dK], eight dims a thread, the parts in rank order
    const int rows = 2 * kT / p.cluster;
    const uint32_t base = smem_u32(smem + LY::kOffLong);
    for (int i = threadIdx.x; i < rows * (D / 8); i += kThreads) {
      const int rr = rank * rows + i / (D / 8), d0 = (i % (D / 8)) * 8;
      const bool is_dk = rr >= kT;
      const int key = x.kt * kT + (is_dk ? rr - kT : rr);
      if (key >= p.S) continue;
      float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int c = 0; c < p.cluster; ++c) {
        const uint32_t at = base + (rr * LY::kRedStride + d0) * 4;
        const float4 y = peer_ld4(at, c), z = peer_ld4(at + 16, c);
        a[0] += y.x; a[1] += y.y; a[2] += y.z; a[3] += y.w;
        a[4] += z.x; a[5] += z.y; a[6] += z.z; a[7] += z.w;
      }
      const float gs = is_dk ? p.scale : 1.f;
      uint4 pk;
      pk.x = pack_bf16x2(a[0] * gs, a[1] * gs);
      pk.y = pack_bf16x2(a[2] * gs, a[3] * gs);
      pk.z = pack_bf16x2(a[4] * gs, a[5] * gs);
      pk.w = pack_bf16x2(a[6] * gs, a[7] * gs);
      __nv_bfloat16* out = is_dk ? p.dk + (int64_t)x.b * p.dk_sb + (int64_t)x.hk * p.dk_sh + (int64_t)key * p.dk_ss
                                 : p.dv + (int64_t)x.b * p.dv_sb + (int64_t)x.hk * p.dv_sh + (int64_t)key * p.dv_ss;
      *reinterpret_cast<uint4*>(out + d0) = pk;
    }
    cluster_barrier();  // no CTA leaves while another reads its part
  }
  // a launch of this kernel that ran beside another one is not over before it
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
}

// ---------------------------------------------------------------------------
// kRest in either kernel: dS = bf16 part + bf16 rest, one product each; the rest takes the 16 words of TMEM that the bf16
// part leaves of its 32.
//
// dQ.  A work item is a 128-query tile of one head: it walks the key tiles that the tile sees (the sinks', then the
// window's).  A CTA per SM takes items round robin, the longest first; the next item's operands are loaded and its
// first scores computed while the finished dQ is read out.
template <int D, bool kRest>
__global__ void __launch_bounds__(kThreads, 1) window_dq_kernel(const __grid_constant__ WinBwdParams p) {
  using LY = Lay<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {  // the 128B swizzle needs it; the same answer in every thread of the launch
    if (threadIdx.x == 0) set_error(p.err, ABKV_DEVERR_RANGE);
    return;
  }
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + LY::kOffBar);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bar + kBarTmem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.H * p.B, n_items = heads * p.n_tiles;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kBarTmem; ++i)
      mbar_init(&bar[i], (i == kBarDS || i == kBarDS + 1 || i == kBarP || i == kBarDrain) ? kWorkers : 1);
  }
  if (warp == 1) alloc_tmem(s_tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;  // S [0,128) [128,256), dP [256,384), dQ [384,..)
  bool dead = false;
  struct Item {
    int qt, h, b, ns, shift, n;
  };
  auto decode = [&](int i) -> Item {
    Item x;
    x.qt = p.n_tiles - 1 - i / heads;
    const int r = i % heads;
    x.h = r % p.H;
    x.b = r / p.H;
    // keys [n_sink, w_lo) are hidden from the whole tile; visited tile u is key tile u < ns ? u : u + shift
    const int w_lo = max(0, x.qt * kT - p.window + 1);
    x.ns = (min(p.n_sink, w_lo) + kT - 1) / kT;
    x.shift = max(w_lo / kT - x.ns, 0);
    x.n = x.qt + 1 - x.shift;
    return x;
  };

  if (warp == 0) {
    if (elect_one()) {
      Pos<kLong> l;
      Pos<kShort> sh;
      int it = 0;
      for (int i = blockIdx.x; i < n_items && !dead; i += gridDim.x, ++it) {
        const Item x = decode(i);
        const int hk = x.h / p.G;
        for (int u = 0; u < x.n; ++u) {
          const int row = (u < x.ns ? u : u + x.shift) * kT;
          if (!wait_or_abort(&bar[kBarLE + l.i], l.ph ^ 1u, dead, p.err)) break;
          mbar_expect_tx(&bar[kBarLF + l.i], LY::kTile);
          load_tile<D>(smem + LY::kOffLong + l.i * LY::kTile, &p.tm_k, row, hk, x.b, &bar[kBarLF + l.i]);
          l.step();
          if (!wait_or_abort(&bar[kBarSE + sh.i], sh.ph ^ 1u, dead, p.err)) break;
          mbar_expect_tx(&bar[kBarSF + sh.i], LY::kTile);
          load_tile<D>(smem + LY::kOffShort + sh.i * LY::kTile, &p.tm_v, row, hk, x.b, &bar[kBarSF + sh.i]);
          sh.step();
          if (u == 0) {  // the item's Q and dO once the previous item's last scores have run
            if (!wait_or_abort(&bar[kBarAE], (uint32_t)((it & 1) ^ 1), dead, p.err)) break;
            mbar_expect_tx(&bar[kBarA], 2 * LY::kTile);
            load_tile<D>(smem + LY::kOffA, &p.tm_q, x.qt * kT, x.h, x.b, &bar[kBarA]);
            load_tile<D>(smem + LY::kOffB, &p.tm_do, x.qt * kT, x.h, x.b, &bar[kBarA]);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint64_t kStep = LY::kTile >> 4;
      const uint64_t dq = desc_kmajor_sw128(smem_u32(smem + LY::kOffA));
      const uint64_t ddo = desc_kmajor_sw128(smem_u32(smem + LY::kOffB));
      const uint64_t k_k = desc_kmajor_sw128(smem_u32(smem + LY::kOffLong));
      const uint64_t v_k = desc_kmajor_sw128(smem_u32(smem + LY::kOffShort));
      const uint64_t k_mn = desc_mnmajor_sw128(smem_u32(smem + LY::kOffLong), LY::kAtom);
      Pos<kLong> kf, ke;  // next K to read for scores; K of the current tile
      Pos<kShort> vf;
      uint32_t sbuf = 0, it_par = 0;
      auto scores = [&]() -> bool {  // S of the next tile into its buffer, over the dS that dQ has read
        if (!wait_or_abort(&bar[kBarLF + kf.i], kf.ph, dead, p.err)) return false;
        tc_fence_after();
        issue_scores<D>(tmem + 128 * sbuf, dq, k_k + kf.i * kStep);
        umma_commit(&bar[kBarS + sbuf]);
        kf.step();
        sbuf ^= 1u;
        return true;
      };
      auto dscores = [&]() -> bool {  // dP of the next tile
        if (!wait_or_abort(&bar[kBarSF + vf.i], vf.ph, dead, p.err)) return false;
        tc_fence_after();
        issue_scores<D>(tmem + 256, ddo, v_k + vf.i * kStep);
        umma_commit(&bar[kBarDP]);
        umma_commit(&bar[kBarSE + vf.i]);  // V's only use
        vf.step();
        return true;
      };
      int it = 0;
      uint32_t g = 0;  // tiles so far; tile g's S buffer, which dS takes over, is g & 1
      for (int i = blockIdx.x; i < n_items && !dead; i += gridDim.x, ++it) {
        const Item x = decode(i);
        if (!wait_or_abort(&bar[kBarA], it_par, dead, p.err) || !scores()) break;
        // the last dP of the previous item has been read
        if (it > 0 && !wait_or_abort(&bar[kBarP], (g & 1u) ^ 1u, dead, p.err)) break;
        if (!dscores()) break;
        if (x.n == 1) umma_commit(&bar[kBarAE]);
        if (x.n > 1 && !scores()) break;
        for (int u = 0; u < x.n; ++u, ++g) {
          const uint32_t buf = g & 1u;
          // dP has been read: the next one, beside the forming of dS
          if (u + 1 < x.n && (!wait_or_abort(&bar[kBarP], buf, dead, p.err) || !dscores())) break;
          if (u + 2 == x.n) umma_commit(&bar[kBarAE]);  // the item's last scores are issued: Q and dO are free then
          if (!wait_or_abort(&bar[kBarDS + buf], (g >> 1) & 1u, dead, p.err)) break;
          // the first product of an item overwrites dQ: the previous one has been read out
          if (u == 0 && it > 0 && !wait_or_abort(&bar[kBarDrain], it_par ^ 1u, dead, p.err)) break;
          tc_fence_after();
          issue_accumulate<D>(tmem + 384, tmem + 128 * buf, k_mn + ke.i * kStep, u == 0);
          if (kRest) issue_accumulate<D>(tmem + 384, tmem + 128 * buf + 16, k_mn + ke.i * kStep, false);
          umma_commit(&bar[kBarLE + ke.i]);
          ke.step();
          if (u + 2 < x.n && !scores()) break;
        }
        if (dead) break;
        umma_commit(&bar[kBarAcc]);
        it_par ^= 1u;
      }
    }
  } else {
    const int sw = warp - 2, cg = sw >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const float sl2 = p.scale_log2;
    int g = 0, it = 0;
    for (int i = blockIdx.x; i < n_items; i += gridDim.x, ++it) {
      const Item x = decode(i);
      const int q = x.qt * kT + row;
      const int64_t r = ((int64_t)x.b * p.H + x.h) * p.S + q;
      const bool in = q < p.S;
      const bool live = in && q > 0;  // query 0 sees one key: P = 1, dS = 0 exactly
      const float nl = in ? -__ldg(p.lse + r) * kLog2e : 0.f, di = in ? __ldcg(p.di + r) : 0.f;
      for (int u = 0; u < x.n; ++u, ++g) {
        const int k0 = (u < x.ns ? u : u + x.shift) * kT + 32 * cg;
        // visible keys of this row among the warp's 32: k <= q without [n_sink, q - window + 1)
        const uint32_t mask = live ? below(q + 1 - k0) & (below(p.n_sink - k0) | ~below(q - p.window + 1 - k0)) : 0u;
        const bool full = __all_sync(0xffffffffu, mask == 0xFFFFFFFFu);
        bool ok = __all_sync(0xffffffffu, wait_or_abort(&bar[kBarS + (g & 1)], (uint32_t)((g >> 1) & 1), dead, p.err));
        if (!ok) dead = true;
        tc_fence_after();
        float pv[32];
        if (ok) {
          tmem_ld32(tmem + lane_base + 128 * (g & 1) + 32 * cg, pv);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            ffma2(pv[c], pv[c + 1], pv[c], pv[c + 1], sl2, nl);
            pv[c] = fast_exp2(pv[c]);
            pv[c + 1] = fast_exp2(pv[c + 1]);
          }
          if (!full) {
#pragma unroll
            for (int c = 0; c < 32; ++c) pv[c] = (mask >> c) & 1u ? pv[c] : 0.f;
          }
        }
        ok = __all_sync(0xffffffffu, wait_or_abort(&bar[kBarDP], (uint32_t)(g & 1), dead, p.err));
        if (!ok) dead = true;
        tc_fence_after();
        if (ok) {
          float dp[32];
          uint32_t w[16];
          tmem_ld32(tmem + lane_base + 256 + 32 * cg, dp);
          tmem_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_one(&bar[kBarP]);  // dP is in registers
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            sub_mul_pair(dp[c], dp[c + 1], dp[c], dp[c + 1], di, di, pv[c], pv[c + 1]);
            w[c / 2] = pack_bf16x2(dp[c], dp[c + 1]);
            if (kRest) dp[c / 2] = __uint_as_float(pack_rest(w[c / 2], dp[c], dp[c + 1]));
          }
          tmem_st16(tmem + lane_base + 128 * (g & 1) + 32 * cg, w);
          if (kRest) {
#pragma unroll
            for (int c = 0; c < 16; ++c) w[c] = __float_as_uint(dp[c]);
            tmem_st16(tmem + lane_base + 128 * (g & 1) + 16 + 32 * cg, w);
          }
          tmem_wait_st();
        } else if (lane == 0) {
          mbar_arrive_one(&bar[kBarP]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_one(&bar[kBarDS + (g & 1)]);
      }
      if (!__all_sync(0xffffffffu, wait_or_abort(&bar[kBarAcc], (uint32_t)(it & 1), dead, p.err))) dead = true;
      tc_fence_after();
      // this warp's D / 4 columns of its rows
      __nv_bfloat16* out = p.dq + (int64_t)x.b * p.dq_sb + (int64_t)x.h * p.dq_sh + (int64_t)q * p.dq_ss + cg * (D / 4);
      float t[32];
      tmem_ld32(tmem + lane_base + 384 + cg * (D / 4), t);  // D 64: the upper 16 columns are not this warp's
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_one(&bar[kBarDrain]);
      if (in && !dead) {
#pragma unroll
        for (int v8 = 0; v8 < D / 32; ++v8) {
          uint4 pk;
          pk.x = pack_bf16x2(t[v8 * 8 + 0] * p.scale, t[v8 * 8 + 1] * p.scale);
          pk.y = pack_bf16x2(t[v8 * 8 + 2] * p.scale, t[v8 * 8 + 3] * p.scale);
          pk.z = pack_bf16x2(t[v8 * 8 + 4] * p.scale, t[v8 * 8 + 5] * p.scale);
          pk.w = pack_bf16x2(t[v8 * 8 + 6] * p.scale, t[v8 * 8 + 7] * p.scale);
          *reinterpret_cast<uint4*>(out + v8 * 8) = pk;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u));
  // this kernel started beside the dK/dV kernel and must not be over before it: what follows reads both
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
}

// Di = rowsum(dO * O) in fp32: D / 8 lanes per row, eight dims a lane.  O is the forward's bf16 output with,
// optionally, the next eight bits of its mantissa (out_lo): Di enters every dS of its row alike, and with
// O rounded to bf16 it would be the largest error of dQ and dK after dS's own rounding.
template <int D>
__global__ void __launch_bounds__(256) window_rowdot_kernel(const __nv_bfloat16* __restrict__ o, int64_t o_sb,
                                                            int64_t o_sh, int64_t o_ss, const int8_t* __restrict__ lo,
                                                            const __nv_bfloat16* __restrict__ dout, int64_t d_sb,
                                                            int64_t d_sh, int64_t d_ss, float* di, int32_t* work, int B,
                                                            int H, int S) {
  constexpr int kL = D / 8;
  if (blockIdx.x == 0 && threadIdx.x == 0) *work = 0;  // the dK/dV launch's item counter
  // at most 2^31 rows (the entry checks), counted in 32 bits: 64-bit divisions took longer than the loads
  const uint32_t r = blockIdx.x * (256u / kL) + threadIdx.x / kL;
  const int d0 = (int)(threadIdx.x % kL) * 8;
  const bool live = r < (uint32_t)B * H * S;
  // rows in memory order of [B][S][H]: neighbouring rows of a warp are neighbours there
  const uint32_t bs = r / (uint32_t)H;
  const int h = (int)(r - bs * H), b = (int)(bs / (uint32_t)S), q = (int)(bs - (uint32_t)b * S);
  const int64_t rr = ((int64_t)b * H + h) * S + q;
  float acc = 0.f;
  if (live) {
    const uint4 x = ld_stream_v4(o + b * o_sb + h * o_sh + q * o_ss + d0);
    const uint4 y = ld_stream_v4(dout + b * d_sb + h * d_sh + q * d_ss + d0);
    uint2 l = make_uint2(0, 0);
    if (lo) l = __ldcs(reinterpret_cast<const uint2*>(lo + rr * D + d0));
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t xb = k & 1 ? xs[k / 2] & 0xFFFF0000u : xs[k / 2] << 16;
      const uint32_t yb = k & 1 ? ys[k / 2] & 0xFFFF0000u : ys[k / 2] << 16;
      const int32_t low = (int32_t)(int8_t)((k < 4 ? l.x : l.y) >> (8 * (k & 3)));
      acc = fmaf(__int_as_float((int32_t)xb + (low << 8)), __uint_as_float(yb), acc);
    }
  }
#pragma unroll
  for (int s = kL / 2; s; s >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, s);
  if (live && d0 == 0) di[rr] = acc;
}

constexpr size_t kWsHeader = 256;
constexpr int kSms = 148;
// dS is rounded to bf16 for the products of dQ and dK: one more error beside the rounding of the result, together sqrt(2)
// of the latter alone (1.43 rms measured for rows of 128 keys and more, 1.46 for the first 128 rows of a sequence; up to
// 1.7 for single outputs over 60 random shapes).  A launch none of whose rows sees more than kRestKeys keys adds a second product
// with what the rounding left out (kRest: 1.04 rms, 1.25 at most).  It costs 33.0 -> 33.1 us at 333 rows of 8 heads, 377 ->
// 441 us at 2 x 4096 rows of 32 heads with a window of 256, and would cost 497 -> 594 us with one of 1024.  The choice is
// the launch's: the first rows of a longer one see as few keys and get one part, like its other rows.  Made by query tile it
// gave those rows' dq 1.04 and dk 1.05, and took a step of 2 x 4096 rows with a window of 1024 from 652 to 665 us (as
// launches of their own) or 669 (as a branch): the second part's registers, for 4% of the tiles.
constexpr int kRestKeys = 512;

template <int D, bool kRest>
int launch(WinBwdParams& prm, const void* out, const int64_t* os, const int8_t* lo, const void* dout,
           const int64_t* ds, float* di, cudaStream_t s) {
  const int64_t threads = (int64_t)prm.B * prm.H * prm.S * (D / 8);
  window_rowdot_kernel<D><<<(unsigned)((threads + 255) / 256), 256, 0, s>>>(
      static_cast<const __nv_bfloat16*>(out), os[0], os[1], os[2], lo, static_cast<const __nv_bfloat16*>(dout), ds[0],
      ds[1], ds[2], di, prm.work, prm.B, prm.H, prm.S);
  if (cudaFuncSetAttribute(window_dkdv_kernel<D, kRest>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<D>::kSmem) !=
          cudaSuccess ||
      cudaFuncSetAttribute(window_dq_kernel<D, kRest>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<D>::kSmem) !=
          cudaSuccess)
    return ABKV_ERR_CUDA;
  // Each kernel may be set up while the one before it drains; the last ones run beside one another.
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Lay<D>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  cfg.attrs = attr;
  auto dkdv = [&](int tile0, int tiles, int cluster, bool first) -> bool {
    prm.tile0 = tile0;
    prm.tiles = tiles;
    prm.cluster = cluster;
    prm.first = first ? 1 : 0;
    const int64_t items = (int64_t)prm.Hkv * prm.B * tiles;
    attr[1].val.clusterDim = {(unsigned)cluster, 1, 1};
    cfg.gridDim = dim3((unsigned)(cluster > 1 ? items * cluster : std::min<int64_t>(items, kSms)));
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, window_dkdv_kernel<D, kRest>, prm) == cudaSuccess;
  };
  // Key tiles as (sinks', others), pairs per tile and in all.
  const int64_t heads = (int64_t)prm.Hkv * prm.B;
  const int sink_tiles = std::min(prm.n_tiles, (prm.n_sink + kT - 1) / kT);
  const int64_t most = (int64_t)prm.n_tiles * prm.G;
  const int64_t usual = (int64_t)std::min(prm.n_tiles, (prm.window + kT - 2) / kT + 1) * prm.G;
  const int64_t share = heads * (sink_tiles * most + (prm.n_tiles - sink_tiles) * usual) / kSms;  // pairs per SM
  if (heads * prm.n_tiles * 2 <= kSms) {
    // few key tiles: a cluster of CTAs for each, up to one CTA per SM
    const int64_t pairs = sink_tiles ? most : usual;
    int cs = 1;
    while (cs < 8 && pairs >= 2 * cs && heads * prm.n_tiles * 2 * cs <= kSms) cs *= 2;
    if (!dkdv(0, prm.n_tiles, cs, true)) return ABKV_ERR_CUDA;
  } else if (sink_tiles && sink_tiles < prm.n_tiles && 10 * most > 11 * share) {
    // the sinks' tiles would outlast the rest: clusters for them, beside the others
    int cs = 2;
    while (cs < 8 && most > cs * std::max(usual, share / 2)) cs *= 2;
    if (!dkdv(0, sink_tiles, cs, true) || !dkdv(sink_tiles, prm.n_tiles - sink_tiles, 1, false)) return ABKV_ERR_CUDA;
  } else {
    if (!dkdv(0, prm.n_tiles, 1, true)) return ABKV_ERR_CUDA;
  }
  cfg.gridDim = dim3((unsigned)std::min<int64_t>((int64_t)prm.H * prm.B * prm.n_tiles, kSms));
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, window_dq_kernel<D, kRest>, prm) != cudaSuccess) return ABKV_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? ABKV_OK : ABKV_ERR_CUDA;
}

}  // namespace
}  // namespace abkv

using namespace abkv;

extern "C" size_t abkv_window_attention_backward_workspace_size(int B, int H, int S, int head_dim) {
  if (B <= 0 || H <= 0 || S <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
  return kWsHeader + ((size_t)B * H * S * 4 + 255) / 256 * 256;
}

extern "C" int abkv_window_attention_backward(
    const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
    const int64_t* v_strides, const void* out, const int64_t* out_strides, const void* out_lo, const void* dout,
    const int64_t* dout_strides, const float* lse, void* dq, const int64_t* dq_strides, void* dk,
    const int64_t* dk_strides, void* dv, const int64_t* dv_strides, int B, int H, int Hkv, int S, int head_dim,
    float scale, int window, int num_sinks, void* workspace, size_t workspace_bytes, void* stream) {
  const void* ptrs[9] = {q, k, v, out, dout, dq, dk, dv, lse};
  for (const void* x : ptrs)
    if (!x) return ABKV_ERR_INVALID_ARG;
  const int64_t* strs[8] = {q_strides, k_strides, v_strides, out_strides, dout_strides, dq_strides, dk_strides,
                            dv_strides};
  for (const int64_t* x : strs)
    if (!x) return ABKV_ERR_INVALID_ARG;
  if (B <= 0 || H <= 0 || Hkv <= 0 || S <= 0 || H % Hkv != 0 || !(scale > 0.f) || window <= 0 || num_sinks < 0)
    return ABKV_ERR_INVALID_ARG;
  if ((head_dim != 64 && head_dim != 128) || H > 128 || B > 65535 || S > (1 << 17)) return ABKV_ERR_UNSUPPORTED;
  if ((int64_t)B * H * S > INT32_MAX) return ABKV_ERR_UNSUPPORTED;
  for (int i = 0; i < 8; ++i)
    if (reinterpret_cast<uintptr_t>(ptrs[i]) & 15) return ABKV_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(out_lo) & 15) return ABKV_ERR_INVALID_ARG;
  for (int i = 3; i < 8; ++i)
    if (strs[i][0] % 8 || strs[i][1] % 8 || strs[i][2] % 8) return ABKV_ERR_INVALID_ARG;
  const size_t need = abkv_window_attention_backward_workspace_size(B, H, S, head_dim);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return ABKV_ERR_WORKSPACE;
  WinBwdParams prm;
  std::memset(&prm, 0, sizeof(prm));
  int st = tc::encode_bhsd(&prm.tm_q, q, B, H, S, head_dim, q_strides, kT);
  if (st == ABKV_OK) st = tc::encode_bhsd(&prm.tm_do, dout, B, H, S, head_dim, dout_strides, kT);
  if (st == ABKV_OK) st = tc::encode_bhsd(&prm.tm_k, k, B, Hkv, S, head_dim, k_strides, kT);
  if (st == ABKV_OK) st = tc::encode_bhsd(&prm.tm_v, v, B, Hkv, S, head_dim, v_strides, kT);
  if (st != ABKV_OK) return st;
  float* di = reinterpret_cast<float*>(static_cast<char*>(workspace) + kWsHeader);
  prm.lse = lse;
  prm.di = di;
  prm.dq = static_cast<__nv_bfloat16*>(dq);
  prm.dk = static_cast<__nv_bfloat16*>(dk);
  prm.dv = static_cast<__nv_bfloat16*>(dv);
  prm.dq_sb = dq_strides[0];
  prm.dq_sh = dq_strides[1];
  prm.dq_ss = dq_strides[2];
  prm.dk_sb = dk_strides[0];
  prm.dk_sh = dk_strides[1];
  prm.dk_ss = dk_strides[2];
  prm.dv_sb = dv_strides[0];
  prm.dv_sh = dv_strides[1];
  prm.dv_ss = dv_strides[2];
  prm.err = static_cast<int32_t*>(workspace);
  prm.work = static_cast<int32_t*>(workspace) + 32;  // inside the header
  prm.B = B;
  prm.H = H;
  prm.Hkv = Hkv;
  prm.G = H / Hkv;
  prm.S = S;
  prm.n_tiles = (S + kT - 1) / kT;
  // where every query sees its own key alone the scores have no gradient: exactly, not as the difference of two sums
  prm.scale = window == 1 && num_sinks == 0 ? 0.f : scale;
  prm.scale_log2 = scale * kLog2e;
  // a window past S hides nothing, sinks past S are every key: keep the tile arithmetic in 32 bits
  prm.window = window < S ? window : S;
  prm.n_sink = num_sinks < S ? num_sinks : S;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int8_t* lo = static_cast<const int8_t*>(out_lo);
  // Rows that see few keys: dS in two bf16 parts (kRestKeys).
  const bool rest = std::min<int64_t>(S, (int64_t)window + num_sinks) <= kRestKeys;
  auto run = head_dim == 64 ? (rest ? launch<64, true> : launch<64, false>)
                            : (rest ? launch<128, true> : launch<128, false>);
  return run(prm, out, out_strides, lo, dout, dout_strides, di, s);
}
