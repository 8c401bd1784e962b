// Attention weights of prompt rows over the paged KV cache, summed per cache row, on 5th-generation
// tensor cores (tcgen05 + TMEM) for sm_100a.
//
// For KV head h of a request of n rows, cache row j, and the request's counted query rows i (its last
// `observe` rows, or all) at positions p_i = n - qlen + i:
//   w[j] += sum over i and the query heads g of h, where j <= p_i and (no window or j > p_i - window or
//           j < sinks), of exp(scale q_ig . k_j - lse_ig)
// with lse the log-sum-exp that the attention of these rows returned, so one pass over the keys is
// enough and nothing is rescaled.
//
// A tile of S^T = K Q^T (128 cache rows x 128 query columns) per step: the accumulator's lanes are
// cache rows, so the sum over queries is a sum over a thread's own registers, no reduction across lanes
// and no second product.  The 128 columns are 4 units of 32 consecutive query rows of one head (so a
// group of 4 heads x 32 observed rows is one full tile).  19 warps:
//   warp 0      the items' descriptors (request, tile, units), passed on through a ring in shared memory, and
//               their K tiles (eight 16-row page slices) by cp.async.bulk.tensor, 128B swizzle
//   warp 18     Q tiles (four 32-row boxes); where every counted row of a request fits one
//               tile, it is loaded once for all cache tiles of a (request, head) run, and the six ring slots go to K
//               (4) rather than Q (4 otherwise)
//   warp 1      TMEM owner (4 S^T buffers) and issuer of tcgen05.mma
//   warps 2..17 thread = one cache row of every fourth step: x = S scale log2(e) - lse log2(e), 2^x, sum
// The exponentials bound it: 128 x 128 of them take 1024 clocks of the SM's 16 a clock, the tile's MMAs 512
// (head_dim 128); a step takes about 1800, as four warps an SM quarter do not hide each other's loads and
// hand-overs.  Measured: 2 x 4050 rows, 32 heads, all counted 219 us (117 of exponentials); the last 32 rows
// of 4 requests over 8065 rows 24 us.  Tried and no faster: half of the exponentials, or a quarter, as
// polynomials on the FMA pipe (238 and 222 us), scores in halves of 64 columns with an issuer for every
// second step (246 us), the next 32 columns loaded ahead (343 us, out of registers).
// Work items are (cache tile, KV head, request); a CTA per SM takes them round robin to and fro, the cache
// tiles that the most rows see first -- or, where Q stays resident, a contiguous run.
// The sum's order is fixed (steps, then the four warp groups), so results repeat bit for bit.
// With one accumulator row for all heads, per-head sums go through the workspace and are added in head order.
// Every mbarrier wait is bounded and records ABKV_DEVERR_TIMEOUT on expiry.
#include <algorithm>
#include <cstring>

#include "tcgen05.cuh"

namespace abkv {
namespace {
using namespace tc;

constexpr int kM = 128, kN = 128, kD = 128;  // cache rows, query columns, head_dim
constexpr int kUnit = 32;                    // query rows of a unit
constexpr int kThreads = 608;
constexpr int kWarpQ = 18;
constexpr int kStages = 6, kSBufs = 4;  // 32 KiB ring slots, shared out between K and Q
__host__ __device__ constexpr int k_stages(bool resident) { return resident ? 4 : 2; }
__host__ __device__ constexpr int q_stages(bool resident) { return kStages - k_stages(resident); }
constexpr int kMaxK = 4, kMaxQ = 4;
constexpr uint32_t kIdescS = idesc_bf16_m128(kN, false);
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTileBytes = kM * kD * 2;  // 2 atoms of [128 rows][128 B]
constexpr int kOffK = 0;
constexpr int kOffLse = kOffK + kStages * kTileBytes;   // 16 warps x [128] floats
constexpr int kOffAcc = kOffLse + 16 * kN * 4;          // [2 items][4 groups][128 rows] partial sums
constexpr int kMaxPref = 1024;
constexpr int kOffPref = kOffAcc + 2 * 4 * kM * 4;      // [R + 1] running tile counts
constexpr int kItemGroup = 4, kItemGroups = 4;          // items are described four at a time, four groups ahead
constexpr int kOffItems = kOffPref + (kMaxPref + 4) * 4;
constexpr int kOffBar = kOffItems + kItemGroup * kItemGroups * 48;
static_assert(kOffItems % 16 == 0 && kOffBar % 8 == 0, "descriptors and barriers");
constexpr int kBarKFull = 0, kBarKEmpty = kBarKFull + kMaxK, kBarQFull = kBarKEmpty + kMaxK,
              kBarQEmpty = kBarQFull + kMaxQ, kBarSFull = kBarQEmpty + kMaxQ, kBarSEmpty = kBarSFull + kSBufs,
              kBarAccFull = kBarSEmpty + kSBufs, kBarAccEmpty = kBarAccFull + 2, kBarItemFull = kBarAccEmpty + 2,
              kBarItemEmpty = kBarItemFull + kItemGroups, kBarTmem = kBarItemEmpty + kItemGroups;
constexpr int kSmemBytes = kOffBar + 8 * (kBarTmem + 1) + 1024;
static_assert(kSmemBytes <= 227 * 1024, "shared memory");

struct alignas(64) PromptParams {
  CUtensorMap tm_q, tm_k;  // q [T][H][D] in boxes of 32 rows; K/V planes of the paged cache
  const float* lse;        // [T][H]
  const int32_t* bt;
  const int32_t* seq_lens;
  const int32_t* q_start;
  float* w;      // [R][units][w_rows], or the per-head sums of the workspace
  float* w_out;  // [R][1][...]: set when w is the workspace
  int64_t w_sb, w_su, out_sb;
  int32_t* err;
  int64_t bt_stride, num_blocks;
  int page, fa_layout, T, H, Hkv, G, R, w_rows, max_tiles, n_items, observe, window, n_sink;
  int max_query_len;
  float scale_log2;
};

// One request as every role sees it.
struct Req {
  int q0, nq, n, p0;  // first counted query row, counted rows, cache rows, position of the first counted row
};

// Most counted rows of a request that the launch is laid out for.
__device__ __forceinline__ int most_rows(const PromptParams& p) {
  return p.observe > 0 ? min(p.observe, p.max_query_len) : p.max_query_len;
}

__device__ __forceinline__ Req load_req(const PromptParams& p, int r, bool report) {
  Req x;
  const int a = __ldg(p.q_start + r), e = __ldg(p.q_start + r + 1);
  const int qlen = e - a;
  x.q0 = x.nq = x.n = x.p0 = 0;
  if (a < 0 || qlen < 0 || e > p.T) {
    if (report) set_error(p.err, ABKV_DEVERR_RANGE);
    return x;
  }
  const int n = __ldg(p.seq_lens + r);
  const int64_t cap = p.bt_stride * (int64_t)p.page;
  if (n < qlen || (int64_t)n > cap || n > p.w_rows) {
    if (report) set_error(p.err, ABKV_DEVERR_SEQ_OOB);
    return x;  // nothing of the request is counted
  }
  x.nq = min(qlen, most_rows(p));
  if (report && qlen > p.max_query_len && x.nq < (p.observe > 0 ? min(qlen, p.observe) : qlen))
    set_error(p.err, ABKV_DEVERR_RANGE);  // max_query_len understated: only the last rows are counted
  x.q0 = e - x.nq;
  x.n = n;
  x.p0 = n - x.nq;
  return x;
}

// A 16-row slice hidden from every counted row is not looked up: its page may be freed.
__device__ __forceinline__ bool hidden_slice(const PromptParams& p, const Req& x, int row0) {
  return p.window > 0 && row0 >= p.n_sink && row0 + 16 <= x.p0 - p.window + 1;
}

// Work of one item: the contiguous range [u0, u1) of units (unit = chunk * G + head) whose rows see a row
// of cache tile kt; empty when there is none.
__device__ __forceinline__ void item_units(const PromptParams& p, const Req& x, int kt, bool resident, int& u0,
                                           int& u1) {
  const int k0 = kt * kM;
  u0 = u1 = 0;
  if (x.nq == 0 || k0 >= x.n) return;
  const int chunks = (x.nq + kUnit - 1) / kUnit;
  // chunk c holds positions p0 + 32 c .. : the first whose last row reaches the tile, the last whose
  // first row's window still does
  const int k1 = min(k0 + kM, x.n) - 1;
  int c0 = k0 <= x.p0 ? 0 : (k0 - x.p0) / kUnit;  // its last row is at or past k0
  int c1 = chunks;
  if (p.window > 0 && k0 >= p.n_sink) {
    // p - window < k1 for the chunk's first row p = p0 + 32 c
    const int64_t lim = (int64_t)k1 + p.window - x.p0;  // 32 c < lim
    c1 = lim <= 0 ? 0 : (int)min((int64_t)chunks, (lim + kUnit - 1) / kUnit);
  }
  if (c0 >= c1) return;
  u0 = resident ? 0 : c0 * p.G;
  u1 = resident ? chunks * p.G : c1 * p.G;
}

// Item sequence of a CTA; resident: every request's counted rows fit one Q tile (by the host's bound on them).
struct Items {
  int first, n;         // items k = 0 .. n - 1 of this CTA
  const int32_t* pref;  // resident: [R + 1] visible cache tiles of the requests before, in shared memory
};
// The visible cache tiles of a request: tile v of `count` is cache tile v < ns ? v : v + shift.
struct Tiles {
  int ns, shift, count;
};
__device__ __forceinline__ Tiles req_tiles(const PromptParams& p, const Req& x) {
  Tiles t;
  const int lo = p.window > 0 ? max(0, x.p0 - p.window + 1) : 0;
  t.ns = (min(p.n_sink, lo) + kM - 1) / kM;
  t.shift = max(lo / kM - t.ns, 0);
  t.count = x.nq > 0 ? (x.n + kM - 1) / kM - t.shift : 0;
  return t;
}
// k-th item of this CTA -> false past the end.  Resident: every item is one tile of work, a contiguous run of the
// requests' visible tiles, (request, head) outermost.  Else the cache tiles in order (under causality the first see
// the most rows), dealt out to and fro so that the CTAs' shares of long and short items come out alike.
__device__ __forceinline__ bool item_at(const PromptParams& p, const Items& it, int k, int& r, int& hk, int& kt) {
  if (it.pref) {
    int i = it.first + k;
    if (k >= it.n) return false;
    int lo = 0, hi = p.R;  // pref[lo] * Hkv <= i < pref[hi] * Hkv
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (it.pref[mid] * p.Hkv <= i)
        lo = mid;
      else
        hi = mid;
    }
    r = lo;
    i -= it.pref[r] * p.Hkv;
    const int count = it.pref[r + 1] - it.pref[r];
    hk = i / count;
    const Tiles t = req_tiles(p, load_req(p, r, false));
    const int v = i - hk * count;
    kt = v < t.ns ? v : v + t.shift;
    return true;
  }
  const int rh = p.R * p.Hkv;
  const int i = k * (int)gridDim.x + ((k & 1) ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x);
  if (i >= p.n_items) return false;
  kt = i / rh;
  const int g = i - kt * rh;
  r = g / p.Hkv;
  hk = g - r * p.Hkv;
  return true;
}

// What every role has to know of an item; units [u0, u1) may be empty.
struct alignas(16) Desc {
  int r, hk, kt, u0;
  int u1, q0, nq, n;  // n: the request's rows, cut before the tile's first bad page
  int p0, pad[3];
};
static_assert(sizeof(Desc) == 48, "ring of descriptors");

__global__ void __launch_bounds__(kThreads, 1) prompt_weights_kernel(const __grid_constant__ PromptParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bar + kBarTmem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool resident = (int64_t)((most_rows(p) + kUnit - 1) / kUnit) * p.G <= kN / kUnit && p.R <= kMaxPref;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kBarTmem; ++i) {
      int n = 1;
      if ((i >= kBarSEmpty && i < kBarSEmpty + kSBufs) || (i >= kBarAccEmpty && i < kBarAccEmpty + 2))
        n = 4;  // the four warps of a group
      else if (i >= kBarAccFull && i < kBarAccFull + 2)
        n = 16;
      else if (i >= kBarItemEmpty)
        n = 16 + 2;  // the groups' warps, the issuer, the Q producer
      mbar_init(&bar[i], n);
    }
  }
  int32_t* s_pref = reinterpret_cast<int32_t*>(smem + kOffPref);
  if (resident && warp == 2) {  // running count of the requests' visible tiles
    int run = 0;
    for (int r0 = 0; r0 < p.R; r0 += 32) {
      int v = 0;
      if (r0 + lane < p.R) v = req_tiles(p, load_req(p, r0 + lane, blockIdx.x == 0)).count;
      int incl = v;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
      }
      if (r0 + lane < p.R) s_pref[r0 + lane + 1] = run + incl;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) s_pref[0] = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(s_tmem)),
                 "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  bool dead = false;
  Items it;
  it.pref = nullptr;
  it.first = 0;
  it.n = (p.n_items + (int)gridDim.x - 1) / (int)gridDim.x;  // the last one may be past the end
  if (resident) {
    const int total = s_pref[p.R] * p.Hkv, per = (total + (int)gridDim.x - 1) / (int)gridDim.x;
    it.pref = s_pref;
    it.first = blockIdx.x * per;
    it.n = max(0, min(per, total - it.first));
  }
  // ring lengths are 2 or 4: slot and phase of a running count
  const int kKStages = k_stages(resident), kQStages = q_stages(resident);
  const int k_shift = kKStages >> 1, q_shift = kQStages >> 1;
  const Desc* const s_items = reinterpret_cast<const Desc*>(smem + kOffItems);
  auto items_ready = [&](int grp) -> bool {
    return wait_or_abort(&bar[kBarItemFull + (grp & (kItemGroups - 1))], (uint32_t)(grp / kItemGroups) & 1u, dead, p.err);
  };
  uint8_t* const s_k = smem + kOffK;
  uint8_t* const s_q = smem + kOffK + kKStages * kTileBytes;

  if (warp == 0) {
    // ---------------- K producer: four items at a time, lane = 8 x item + 16-row slice, so that the
    // look-ups of four items (request, page) are under way together ----------------
    int kc = 0;
    for (int base = 0; base < it.n && !dead; base += 4) {
      const int k = base + (lane >> 3), slice = lane & 7;
      int pg = -1, off = 0;
      bool bad = false;
      Desc d;
      d.r = d.hk = d.kt = d.u0 = d.u1 = d.q0 = d.nq = d.n = d.p0 = 0;
      if (k < it.n && item_at(p, it, k, d.r, d.hk, d.kt)) {
        const Req x = load_req(p, d.r, !resident && d.kt == 0 && d.hk == 0 && slice == 0);
        item_units(p, x, d.kt, resident, d.u0, d.u1);
        d.q0 = x.q0;
        d.nq = x.nq;
        d.n = x.n;
        d.p0 = x.p0;
        const int row0 = d.kt * kM + 16 * slice;
        if (d.u0 < d.u1 && row0 < x.n) {
          if (!hidden_slice(p, x, row0)) {
            pg = __ldg(p.bt + (int64_t)d.r * p.bt_stride + row0 / p.page);
            off = row0 % p.page;
            if (pg < 0 || (int64_t)pg >= p.num_blocks) {
              set_error(p.err, ABKV_DEVERR_PAGE_OOB);
              pg = -1;
              bad = true;
            }
          }
        }
      }
      const uint32_t valid = __ballot_sync(0xffffffffu, pg >= 0), work = __ballot_sync(0xffffffffu, d.u0 < d.u1);
      // Scores of a slice without its page are of what the ring held before.  Its rows must not collect them, and the rows
      // behind it in the tile go without as well: a limit that the writers read anyway (checking each row's own slice
      // there took 2 to 6% of the kernel's time).
      const uint32_t bad8 = __ballot_sync(0xffffffffu, bad) >> (lane & 24) & 0xFFu;
      if (bad8) d.n = min(d.n, d.kt * kM + 16 * (__ffs(bad8) - 1));
      const int grp = base / kItemGroup, gs = grp & (kItemGroups - 1);
      if (!__all_sync(0xffffffffu, wait_or_abort(&bar[kBarItemEmpty + gs], ((uint32_t)(grp / kItemGroups) & 1u) ^ 1u,
                                                 dead, p.err))) {
        dead = true;
        break;
      }
      if (slice == 0) *reinterpret_cast<Desc*>(smem + kOffItems + (gs * kItemGroup + (lane >> 3)) * 48) = d;
      __syncwarp();
      if (lane == 0) mbar_arrive_one(&bar[kBarItemFull + gs]);
      for (int j = 0; j < 4; ++j) {
        if (!((work >> (8 * j)) & 1u)) continue;
        const int st = kc & (kKStages - 1);
        bool ok = true;
        if (lane == 0) {
          ok = wait_or_abort(&bar[kBarKEmpty + st], (uint32_t)(((kc >> k_shift) & 1) ^ 1), dead, p.err);
          if (ok) mbar_expect_tx(&bar[kBarKFull + st], (uint32_t)__popc((valid >> (8 * j)) & 0xFFu) * 2u * 2048u);
        }
        if (!__shfl_sync(0xffffffffu, ok, 0)) {
          dead = true;
          break;
        }
        if ((lane >> 3) == j && pg >= 0) {
          uint8_t* kb = s_k + st * kTileBytes + slice * 2048;
          const int plane = p.fa_layout ? pg : 2 * pg;
          tma_load_4d(kb, &p.tm_k, 0, d.hk, off, plane, &bar[kBarKFull + st]);
          tma_load_4d(kb + kTileBytes / 2, &p.tm_k, 64, d.hk, off, plane, &bar[kBarKFull + st]);
        }
        ++kc;
      }
    }
  } else if (warp == kWarpQ) {
    // ---------------- Q producer ----------------
    if (elect_one()) {
      int qc = 0, last_g = -1;
      for (int base = 0, grp = 0; base < it.n && !dead; base += kItemGroup, ++grp) {
        if (!items_ready(grp)) break;
        for (int j = 0; j < kItemGroup && !dead; ++j) {
          const Desc x = s_items[(grp & (kItemGroups - 1)) * kItemGroup + j];
          if (x.u0 >= x.u1) continue;
          if (resident && last_g == x.r * p.Hkv + x.hk) continue;  // this tile is loaded
          last_g = x.r * p.Hkv + x.hk;
          int chunk = x.u0 / p.G, g = x.u0 - chunk * p.G;
          for (int u = x.u0; u < x.u1; u += 4, ++qc) {
            const int st = qc & (kQStages - 1), nu = min(4, x.u1 - u);
            if (!wait_or_abort(&bar[kBarQEmpty + st], (uint32_t)(((qc >> q_shift) & 1) ^ 1), dead, p.err)) break;
            mbar_expect_tx(&bar[kBarQFull + st], (uint32_t)nu * 2u * 4096u);
            for (int c = 0; c < nu; ++c) {
              uint8_t* qb = s_q + st * kTileBytes + c * 4096;
              const int h = x.hk * p.G + g, t = x.q0 + chunk * kUnit;
              tma_load_4d(qb, &p.tm_q, 0, h, t, 0, &bar[kBarQFull + st]);
              tma_load_4d(qb + kTileBytes / 2, &p.tm_q, 64, h, t, 0, &bar[kBarQFull + st]);
              if (++g == p.G) {
                g = 0;
                ++chunk;
              }
            }
          }
        }
        mbar_arrive_one(&bar[kBarItemEmpty + (grp & (kItemGroups - 1))]);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (elect_one()) {
      const uint64_t dk0 = desc_kmajor_sw128(smem_u32(s_k)), dq0 = desc_kmajor_sw128(smem_u32(s_q));
      constexpr uint64_t kStep = kTileBytes >> 4;  // descriptors count 16 bytes
      int kc = 0, qc = 0, sc = 0, last_g = -1;
      for (int base = 0, grp = 0; base < it.n && !dead; base += kItemGroup, ++grp) {
        if (!items_ready(grp)) break;
        for (int j = 0; j < kItemGroup && !dead; ++j) {
          const Desc x = s_items[(grp & (kItemGroups - 1)) * kItemGroup + j];
          if (x.u0 >= x.u1) continue;
          const int ks = kc & (kKStages - 1), g = x.r * p.Hkv + x.hk;
          const bool fresh = !resident || last_g != g;
          if (resident && fresh && last_g >= 0) {
            umma_commit(&bar[kBarQEmpty + (qc & (kQStages - 1))]);  // the previous run's Q tile
            ++qc;
          }
          last_g = g;
          if (!wait_or_abort(&bar[kBarKFull + ks], (uint32_t)((kc >> k_shift) & 1), dead, p.err)) break;
          const uint64_t dk = dk0 + ks * kStep;
          for (int u = x.u0; u < x.u1; u += 4) {
            const int qs = qc & (kQStages - 1), sb = sc & (kSBufs - 1);
            if (fresh && !wait_or_abort(&bar[kBarQFull + qs], (uint32_t)((qc >> q_shift) & 1), dead, p.err)) break;
            if (!wait_or_abort(&bar[kBarSEmpty + sb], (uint32_t)(((sc / kSBufs) & 1) ^ 1), dead, p.err)) break;
            tc_fence_after();
            const uint64_t dq = dq0 + qs * kStep;
#pragma unroll
            for (int kk = 0; kk < kD / 16; ++kk) {
              const uint32_t off = (kk >> 2) * (kTileBytes / 2) + (kk & 3) * 32;
              umma(tmem + 128 * sb, desc_advance(dk, off), desc_advance(dq, off), kIdescS, kk > 0 ? 1u : 0u);
            }
            umma_commit(&bar[kBarSFull + sb]);
            ++sc;
            if (!resident) {
              umma_commit(&bar[kBarQEmpty + qs]);
              ++qc;
            }
          }
          umma_commit(&bar[kBarKEmpty + ks]);
          ++kc;
        }
        mbar_arrive_one(&bar[kBarItemEmpty + (grp & (kItemGroups - 1))]);
      }
    }
  } else {
    // ---------------- exponentials and sums: lane = cache row; group cg of four warps (one per lane quarter)
    // takes every fourth step, all of its 128 columns, so that four steps are under way at a time ----------------
    const int sw = warp - 2, cg = sw >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    float* s_lse = reinterpret_cast<float*>(smem + kOffLse) + sw * kN;  // this warp's: a step's 128 rows
    float* s_acc = reinterpret_cast<float*>(smem + kOffAcc);
    const float sl2 = p.scale_log2;
    const int ahead = 16 / p.G;  // whole chunks from a group's step to its next
    int sc = 0, ic = 0;
    for (int base = 0, grp = 0; base < it.n && !dead; base += kItemGroup, ++grp) {
      if (!__all_sync(0xffffffffu, items_ready(grp))) {
        dead = true;
        break;
      }
      for (int i = 0; i < kItemGroup && !dead; ++i) {
        const Desc& x = s_items[(grp & (kItemGroups - 1)) * kItemGroup + i];
        const int u0 = x.u0, u1 = x.u1;
        if (u0 >= u1) continue;
        if (resident && (sc & 3) != cg) {  // one step, another group's
          ++sc;
          continue;
        }
        const int key = x.kt * kM + row;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        // log-sum-exp of a step's rows, lane = row of each of its four units
        float n_lse[4];
        int mine = u0 + 4 * ((cg - sc) & 3);  // the group's first step of the item
        int f_chunk = mine / p.G, f_h = mine - f_chunk * p.G;  // chunk and head of unit `mine`
        auto fetch = [&]() {
          int chunk = f_chunk, h = f_h;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int t = min(x.q0 + chunk * kUnit + lane, p.T - 1);
            n_lse[j] = mine + j < u1 ? __ldg(p.lse + (int64_t)t * p.H + x.hk * p.G + h) : 0.f;
            if (++h == p.G) {
              h = 0;
              ++chunk;
            }
          }
        };
        if (mine < u1) fetch();
        for (int u = u0; u < u1; u += 4, ++sc) {
          if (u != mine) continue;
          const int sb = sc % kSBufs;
          __syncwarp();  // every lane is past its reads of the previous step's values
#pragma unroll
          for (int j = 0; j < 4; ++j) s_lse[32 * j + lane] = n_lse[j] * -kLog2e;
          __syncwarp();
          int chunk = f_chunk, h = f_h;
          mine += 16;
          f_chunk += ahead;
          f_h += 16 - ahead * p.G;
          if (f_h >= p.G) {
            f_h -= p.G;
            ++f_chunk;
          }
          if (mine < u1) fetch();
          const bool ok = __all_sync(0xffffffffu,
                                     wait_or_abort(&bar[kBarSFull + sb], (uint32_t)((sc / kSBufs) & 1), dead, p.err));
          if (!ok) dead = true;
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (ok && u + j < u1) {
              float s[32];
              tmem_ld32(tmem + lane_base + 128 * sb + 32 * j, s);
              tmem_wait_ld();
              // visible columns [a, e): rows at or past the key, inside its window, and counted
              const int pc = x.p0 + chunk * kUnit;
              const int a = max(key - pc, 0);
              int e = min(kUnit, x.nq - chunk * kUnit);
              if (p.window > 0 && key >= p.n_sink) e = (int)min((int64_t)e, (int64_t)key + p.window - pc);
              const uint32_t mask = (a >= e || e <= 0) ? 0u : (0xFFFFFFFFu >> (32 - e)) & (0xFFFFFFFFu << a);
              const bool full = __all_sync(0xffffffffu, mask == 0xFFFFFFFFu);
              const float* l4 = s_lse + 32 * j;
              if (full) {
#pragma unroll
                for (int c = 0; c < 32; c += 4) {
                  const float4 l = *reinterpret_cast<const float4*>(l4 + c);
                  float x0, x1, x2, x3;
                  ffma2(x0, x1, s[c], s[c + 1], sl2, l.x, l.y);
                  ffma2(x2, x3, s[c + 2], s[c + 3], sl2, l.z, l.w);
                  fadd2(acc[0], acc[1], fast_exp2(x0), fast_exp2(x1));
                  fadd2(acc[2], acc[3], fast_exp2(x2), fast_exp2(x3));
                }
              } else if (__any_sync(0xffffffffu, mask != 0u)) {
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                  const float v = fast_exp2(fmaf(s[c], sl2, l4[c]));
                  acc[c & 3] += (mask >> c) & 1u ? v : 0.f;
                }
              }
            }
            if (++h == p.G) {
              h = 0;
              ++chunk;
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_one(&bar[kBarSEmpty + sb]);
        }
        float add = (acc[0] + acc[1]) + (acc[2] + acc[3]);
        bool writer = true;
        if (!resident) {
          // the four groups' parts of a cache row, added in group order by one group (in turn)
          const int b = ic & 1;
          const uint32_t ph = (uint32_t)(ic >> 1) & 1u;
          float* sa = s_acc + b * 4 * kM;
          if (!__all_sync(0xffffffffu, wait_or_abort(&bar[kBarAccEmpty + b], ph ^ 1u, dead, p.err))) dead = true;
          if (!dead) sa[cg * kM + row] = add;
          __syncwarp();
          if (lane == 0) mbar_arrive_one(&bar[kBarAccFull + b]);
          writer = (ic & 3) == cg;
          if (writer) {
            if (!__all_sync(0xffffffffu, wait_or_abort(&bar[kBarAccFull + b], ph, dead, p.err))) dead = true;
            add = (sa[row] + sa[kM + row]) + (sa[2 * kM + row] + sa[3 * kM + row]);
            __syncwarp();
            if (lane == 0) mbar_arrive_one(&bar[kBarAccEmpty + b]);
          }
          ++ic;
        }
        if (writer && key < x.n && !dead) {
          float* w = p.w + (int64_t)x.r * p.w_sb + (int64_t)x.hk * p.w_su + key;
          // one addition per element and launch: without waiting for the old value
          if (p.w_out)
            *w = add;
          else
            atomicAdd(w, add);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_one(&bar[kBarItemEmpty + (grp & (kItemGroups - 1))]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u));
  }
}

// One accumulator row for all heads: w_out[r][row] += the per-head sums in head order.
__global__ void prompt_weights_heads_kernel(const __grid_constant__ PromptParams p) {
  const int r = blockIdx.y;
  const Req x = load_req(p, r, false);
  const int row = blockIdx.x * blockDim.x + threadIdx.x;
  if (row >= x.n || x.nq == 0) return;
  // nor were the rows from a tile's first bad page on
  for (int row0 = row / kM * kM; row0 <= row; row0 += 16) {
    if (hidden_slice(p, x, row0)) continue;
    const int pg = __ldg(p.bt + (int64_t)r * p.bt_stride + row0 / p.page);
    if (pg < 0 || (int64_t)pg >= p.num_blocks) return;
  }
  float acc = 0.f;
  for (int h = 0; h < p.Hkv; ++h) {
    // a tile no counted row sees was not written
    int u0, u1;
    item_units(p, x, row / kM, false, u0, u1);
    if (u0 < u1) acc += __ldcg(p.w + (int64_t)r * p.w_sb + (int64_t)h * p.w_su + row);
  }
  p.w_out[(int64_t)r * p.out_sb + row] += acc;
}

}  // namespace
}  // namespace abkv

using namespace abkv;

extern "C" size_t abkv_prompt_weights_workspace_size(int R, int num_kv_heads, int64_t max_rows, int weight_units) {
  if (R <= 0 || num_kv_heads <= 0 || max_rows <= 0 || weight_units <= 0) return 0;
  return 256 + (weight_units == 1 && num_kv_heads > 1 ? (size_t)R * num_kv_heads * max_rows * 4 : 0);
}

extern "C" int abkv_prompt_weights(const void* q, int64_t q_row_stride, int64_t q_head_stride, const float* lse,
                                   const int32_t* query_start_loc, const void* kv_cache, int kv_layout,
                                   int64_t num_blocks, int page_size, const int32_t* block_table, int64_t bt_stride,
                                   const int32_t* seq_lens, float* weights, int64_t weight_seq_stride,
                                   int64_t weight_unit_stride, int weight_rows, int weight_units, int R, int Hq,
                                   int Hkv, int head_dim, int max_query_len, int max_rows, int T, int observe,
                                   float scale, int window, int num_sinks, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  if (!q || !lse || !query_start_loc || !kv_cache || !block_table || !seq_lens || !weights) return ABKV_ERR_INVALID_ARG;
  if (R <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || T <= 0 || num_blocks <= 0 || bt_stride <= 0 ||
      !(scale > 0.f) || (kv_layout != 0 && kv_layout != 1) || max_query_len <= 0 || max_query_len > T || max_rows <= 0 ||
      observe < 0 || window < 0 || num_sinks < 0 || weight_rows <= 0 || (weight_units != 1 && weight_units != Hkv) ||
      q_row_stride <= 0 || q_head_stride <= 0)
    return ABKV_ERR_INVALID_ARG;
  if (head_dim != kD || page_size <= 0 || page_size % 16 || 2 * num_blocks > INT32_MAX || R > 65535)
    return ABKV_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv_cache)) & 15) return ABKV_ERR_INVALID_ARG;
  const size_t need = abkv_prompt_weights_workspace_size(R, Hkv, max_rows, weight_units);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return ABKV_ERR_WORKSPACE;
  PromptParams prm;
  std::memset(&prm, 0, sizeof(prm));
  {
    const cuuint64_t dims[4] = {(cuuint64_t)kD, (cuuint64_t)Hq, (cuuint64_t)T, 1};
    const cuuint64_t gstr[3] = {(cuuint64_t)q_head_stride * 2, (cuuint64_t)q_row_stride * 2,
                                (cuuint64_t)q_row_stride * 2 * (cuuint64_t)T};
    const cuuint32_t box[4] = {64, 1, (cuuint32_t)kUnit, 1};
    const int st = tc::encode_tiled_4d(&prm.tm_q, q, dims, gstr, box);
    if (st != ABKV_OK) return st;
  }
  {
    const cuuint64_t row = (cuuint64_t)Hkv * kD * 2;
    const cuuint64_t dims[4] = {(cuuint64_t)kD, (cuuint64_t)Hkv, (cuuint64_t)page_size, (cuuint64_t)(2 * num_blocks)};
    const cuuint64_t gstr[3] = {(cuuint64_t)kD * 2, row, row * (cuuint64_t)page_size};
    const cuuint32_t box[4] = {64, 1, 16, 1};
    const int st = tc::encode_tiled_4d(&prm.tm_k, kv_cache, dims, gstr, box);
    if (st != ABKV_OK) return st;
  }
  const bool shared = weight_units == 1 && Hkv > 1;
  prm.lse = lse;
  prm.bt = block_table;
  prm.seq_lens = seq_lens;
  prm.q_start = query_start_loc;
  prm.w = shared ? reinterpret_cast<float*>(static_cast<char*>(workspace) + 256) : weights;
  prm.w_sb = shared ? (int64_t)Hkv * max_rows : weight_seq_stride;
  prm.w_su = shared ? max_rows : weight_unit_stride;
  prm.w_out = shared ? weights : nullptr;
  prm.out_sb = weight_seq_stride;
  prm.err = static_cast<int32_t*>(workspace);
  prm.bt_stride = bt_stride;
  prm.num_blocks = num_blocks;
  prm.page = page_size;
  prm.fa_layout = kv_layout;
  prm.T = T;
  prm.H = Hq;
  prm.Hkv = Hkv;
  prm.G = Hq / Hkv;
  prm.R = R;
  prm.w_rows = std::min(weight_rows, max_rows);
  prm.max_tiles = (max_rows - 1) / kM + 1;
  const int64_t items = (int64_t)prm.max_tiles * R * Hkv;
  if (items > INT32_MAX / 2) return ABKV_ERR_UNSUPPORTED;
  prm.n_items = (int)items;
  prm.observe = observe;
  prm.window = window;
  prm.n_sink = num_sinks;
  prm.max_query_len = max_query_len;
  prm.scale_log2 = scale * kLog2e;
  int dev = 0, num_sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&num_sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || num_sms <= 0)
    return ABKV_ERR_CUDA;
  if (cudaFuncSetAttribute(prompt_weights_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) !=
      cudaSuccess)
    return ABKV_ERR_CUDA;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  prompt_weights_kernel<<<std::min(prm.n_items, num_sms), kThreads, kSmemBytes, s>>>(prm);
  if (shared) prompt_weights_heads_kernel<<<dim3((max_rows + 255) / 256, R), 256, 0, s>>>(prm);
  if (cudaGetLastError() != cudaSuccess) return ABKV_ERR_CUDA;
  return ABKV_OK;
}
