// Eviction from a paged KV cache by accumulated attention weight, for sm_100a.
//
// For one unit (a KV head, or all heads together) of one (layer, sequence) of n rows with budget m < n:
// kept = the first num_sinks rows, the last num_recent rows, and of the rest the m - num_sinks -
// num_recent rows with the largest accumulated weight w (ties to the lower row), in row order.  Kept
// row i becomes row i of the destination table (the source pages themselves, or other pages of the
// pool), its weight becomes weight i, and weights past the new length become 0.
//
// Two kernels.  select: one CTA per unit.  The weights become order-preserving 32-bit keys (-0 as +0, NaN as -inf),
// are held in shared memory, and the (m - sinks - recent)-th largest key is found by histogram passes over 11, 11
// and 10 key bits, of which the last are left out once they decide nothing (plain shared-memory adds, one per warp
// where its rows share the digit; grouping equal digits first with match.any was 1.3 to 3 us slower on 1311 and
// 8190 rows).  Then every warp walks its contiguous share of the rows twice, counting and emitting by ballot, so
// the kept list comes out in row order with one scan over the warps.
// move: bound by memory, so as many bytes in flight as fit: rows go through a shared-memory ring (see
// evict_move_kernel).
// Measured: 4 layers x 16 sequences of 5003 to 8190 rows to 4096 (2.15 GB with both directions) 392 us, 5.5 TB/s
// of 6.53 measured for a copy; one sequence of 1311 rows to 1024 16 us, which is two launches and the selection's
// three passes, one after another.
#include <algorithm>
#include <cstring>

#include "common.cuh"

namespace abkv {
namespace {

constexpr int kMaxLayers = 48;  // layers per launch
constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCachedKeys = 48 * 1024;  // keys held in shared memory; longer sequences re-read the weights
constexpr int kLoaders = 4, kStorers = 4, kMoveThreads = 32 * (kLoaders + kStorers);
constexpr int kSlot = 16 * 1024, kSlots = 6;  // 96 KiB of rows in flight per CTA, two CTAs per SM
constexpr int kSlotRows = 128;
// A loader waits for a slot's last use by parity, which tells one phase from the next only.  A loader that is
// at slot number c has loaded slot c - kLoaders, so the storers are past slot c - kLoaders - ring depth; with
// no more loaders than ring slots the phase before the one it waits for is then complete.  A shallower
// ring than kSlots is only used where no slot is filled twice.
static_assert(kLoaders <= kSlots, "a loader must not run two phases ahead of a slot");
constexpr int move_smem(int slots) { return slots * (kSlot + 2 * 8 + 16); }
constexpr int kMoveSmem = move_smem(kSlots);
constexpr int kMoveCtas = 2 * 148, kStreamsPerCta = 6;

struct EvictLayer {
  char* kv;
  const int32_t* bt;
  const int32_t* dst;  // destination table (== bt: in place)
  const int32_t* seq_lens;
  int32_t* new_lens;
  const float* w;
  float* w_out;
  int32_t* keep;  // [B][units][keep_stride]
  int64_t bt_stride, dst_stride, num_blocks, w_sb, w_su, o_sb, o_su;
  int budget, keep_stride;
};

struct EvictParams {
  EvictLayer layer[kMaxLayers];
  int32_t* err;
  int B, units, Hkv, P, max_rows, w_rows, out_rows, sinks, recent, cached_keys;
  int row_vecs;   // 16-byte vectors of a whole cache row
  int unit_vecs;  // of a unit's part of it
  int fa_layout;
  int in_place;
  int slices, slice_bytes;  // column slices of a unit's row part
  int ranges, range_rows;   // kept-row ranges of a stream (one in place)
  int n_streams;
  int slots;  // ring depth
};

// Weight -> unsigned key of the same order; NaN counts as -inf, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Rows of sequence b: seq_lens clamped to what the table and the weights can address.
__device__ __forceinline__ int evict_len(const EvictParams& p, const EvictLayer& L, int b, bool report) {
  const int s = __ldg(L.seq_lens + b);
  int64_t cap = L.bt_stride * (int64_t)p.P;
  cap = min(cap, (int64_t)min(p.max_rows, p.w_rows));
  if (s < 0 || (int64_t)s > cap) {
    if (report) set_error(p.err, ABKV_DEVERR_SEQ_OOB);
    return s < 0 ? 0 : (int)cap;
  }
  return s;
}

// Inclusive prefix sum over the lanes of a warp.
__device__ __forceinline__ int warp_incl_scan(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}

__global__ void __launch_bounds__(kSelThreads, 1) evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t s_keys[];
  __shared__ int s_hist[kBins];
  __shared__ int s_scan[kSelWarps];
  __shared__ int s_pick[3];  // digit chosen by a pass, rows still wanted inside it, rows it holds
  __shared__ int s_fix[kSelWarps], s_eq[kSelWarps];
  const EvictLayer& L = p.layer[blockIdx.z];
  const int b = blockIdx.y, u = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = evict_len(p, L, b, u == 0 && tid == 0);
  const int m = min(n, L.budget);
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // the move kernel may get ready
  if (u == 0 && tid == 0) L.new_lens[b] = m;
  const float* w = L.w + b * L.w_sb + u * L.w_su;
  int32_t* keep = L.keep + ((int64_t)b * p.units + u) * L.keep_stride;
  float* wo = L.w_out + b * L.o_sb + u * L.o_su;
  const bool apart = L.w_out != L.w;  // the new weights may be written while the old ones are read
  const int mo = min(m, p.out_rows);
  if (mo < m && tid == 0) set_error(p.err, ABKV_DEVERR_SEQ_OOB);

  if (n <= L.budget) {
    for (int i = tid; i < L.keep_stride; i += kSelThreads) keep[i] = i < n ? i : -1;
  } else {
    const int s = p.sinks, e = n - p.recent;  // rows [s, e) compete
    const bool cached = e - s <= p.cached_keys;
    if (cached) {
      for (int i = s + tid; i < e; i += kSelThreads) s_keys[i - s] = weight_key(__ldg(w + i));
    }
    auto key_at = [&](int i) -> uint32_t { return cached ? s_keys[i - s] : weight_key(__ldg(w + i)); };
    int want = m - s - p.recent;  // >= 0; rows to pick
    uint32_t prefix = 0, mask = 0;
    // ---- the want-th largest key, digit by digit
    if (want > 0) {
#pragma unroll 1
      for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
        const uint32_t dmask = pass == 2 ? 1023u : 2047u;
        for (int i = tid; i < kBins; i += kSelThreads) s_hist[i] = 0;
        __syncthreads();
        for (int i0 = s; i0 < e; i0 += kSelThreads) {
          const int i = i0 + tid;
          const uint32_t k = i < e ? key_at(i) : 0u;
          const bool in = i < e && (k & mask) == prefix;
          const uint32_t digit = in ? (k >> shift) & dmask : 0xFFFFFFFFu;
          // one add where the warp's rows share a digit (rows never attended to, ties)
          const uint32_t act = __ballot_sync(0xffffffffu, in);
          const uint32_t first = __shfl_sync(0xffffffffu, digit, act ? __ffs(act) - 1 : 0);
          if (__all_sync(0xffffffffu, !in || digit == first)) {
            if (act && lane == 0) atomicAdd(&s_hist[first], __popc(act));
          } else if (in) {
            atomicAdd(&s_hist[digit], 1);
          }
        }
        __syncthreads();
        // thread t holds bins kBins - 1 - 2t and kBins - 2 - 2t: a running count from the largest digit
        const int c0 = s_hist[kBins - 1 - 2 * tid], c1 = s_hist[kBins - 2 - 2 * tid];
        const int incl = warp_incl_scan(c0 + c1);
        if (lane == 31) s_scan[warp] = incl;
        __syncthreads();
        if (warp == 0) s_scan[lane] = warp_incl_scan(s_scan[lane]);
        __syncthreads();
        const int before = (warp ? s_scan[warp - 1] : 0) + incl - (c0 + c1);  // keys with a larger digit
        if (before < want && want <= before + c0) {
          s_pick[0] = kBins - 1 - 2 * tid;
          s_pick[1] = want - before;
          s_pick[2] = c0;
        } else if (before + c0 < want && want <= before + c0 + c1) {
          s_pick[0] = kBins - 2 - 2 * tid;
          s_pick[1] = want - before - c0;
          s_pick[2] = c1;
        }
        __syncthreads();
        prefix |= (uint32_t)s_pick[0] << shift;
        mask |= dmask << shift;
        want = s_pick[1];
        if (want == s_pick[2]) break;  // every row of the digit is wanted: the later digits decide nothing
      }
    }
    // now, on the digits looked at: every larger key is kept, and the first `want` rows of the equal ones
    const bool none = m - s - p.recent <= 0;
    auto classify = [&](int i, bool& fix, bool& eq) {
      fix = eq = false;
      if (i >= n) return;
      if (i < s || i >= e) {
        fix = true;
      } else if (!none) {
        const uint32_t k = key_at(i) & mask;
        fix = k > prefix;
        eq = k == prefix;
      }
    };
    const int share = ((n + kSelWarps - 1) / kSelWarps + 31) / 32 * 32;  // rows per warp
    const int r0 = warp * share, r1 = min(n, r0 + share);
    int nfix = 0, neq = 0;
    for (int i0 = r0; i0 < r1; i0 += 32) {
      bool fix, eq;
      classify(i0 + lane, fix, eq);
      nfix += __popc(__ballot_sync(0xffffffffu, fix));
      neq += __popc(__ballot_sync(0xffffffffu, eq));
    }
    if (lane == 0) {
      s_fix[warp] = nfix;
      s_eq[warp] = neq;
    }
    __syncthreads();
    const int fi = warp_incl_scan(s_fix[lane]), ei = warp_incl_scan(s_eq[lane]);
    const int fbase = __shfl_sync(0xffffffffu, fi - s_fix[lane], warp);
    int ebase = __shfl_sync(0xffffffffu, ei - s_eq[lane], warp);  // rows equal to the border before this warp
    int at = fbase + min(ebase, want);                              // kept rows before this warp
    for (int i0 = r0; i0 < r1; i0 += 32) {
      bool fix, eq;
      classify(i0 + lane, fix, eq);
      const uint32_t em = __ballot_sync(0xffffffffu, eq), below = (1u << lane) - 1u;
      const bool take = fix || (eq && ebase + __popc(em & below) < want);
      const uint32_t tm = __ballot_sync(0xffffffffu, take);
      if (take) {
        const int j = at + __popc(tm & below);
        keep[j] = i0 + lane;
        if (apart && j < p.out_rows) wo[j] = __ldg(w + i0 + lane);
      }
      at += __popc(tm);
      ebase += __popc(em);
    }
    for (int i = m + tid; i < L.keep_stride; i += kSelThreads) keep[i] = -1;
  }
  if (n <= L.budget || !apart) {
    __syncthreads();  // the list is complete (and visible to this CTA)
    // weights: chunks read whole, then written (w_out may be w: rows only move down)
    constexpr int kPer = 8;
    for (int j0 = 0; j0 < mo; j0 += kSelThreads * kPer) {
      float v[kPer];
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        const int j = j0 + x * kSelThreads + tid;
        if (j < mo) v[x] = __ldcg(w + (n <= L.budget ? j : keep[j]));
      }
      __syncthreads();
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        const int j = j0 + x * kSelThreads + tid;
        if (j < mo) wo[j] = v[x];
      }
    }
  }
  for (int j = mo + tid; j < p.out_rows; j += kSelThreads) wo[j] = 0.f;
}

// Byte offset of (page, K or V, row in page) in the cache.
__device__ __forceinline__ int64_t row_offset(const EvictParams& p, const EvictLayer& L, int pg, int kind, int off) {
  const int64_t plane = p.fa_layout ? (int64_t)kind * L.num_blocks + pg : 2 * (int64_t)pg + kind;
  return (plane * p.P + off) * (int64_t)p.row_vecs * 16;
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;\n" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// One arrival on `bar` when this thread's cp.async copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}

// Page of row i in a table row, or -1 (recorded) where the table cannot address it.
__device__ __forceinline__ int lookup_page(const EvictParams& p, const EvictLayer& L, const int32_t* bt,
                                           int64_t stride, int i) {
  const int slot = i / p.P;
  if (slot >= stride) {
    set_error(p.err, ABKV_DEVERR_SEQ_OOB);
    return -1;
  }
  const int pg = __ldg(bt + slot);
  if (pg < 0 || pg >= L.num_blocks) {
    set_error(p.err, ABKV_DEVERR_PAGE_OOB);
    return -1;
  }
  return pg;
}

// Moves the kept rows.  A stream is a column slice of K or V of one unit, over all kept rows (in place) or a
// range of them; CTAs take streams round robin.  Four loader warps bring slots of up to 16 KiB into a
// ring, a slot each in turn; four storer warps wait for the slots in order and send the rows to their
// places.  In place that order is all the safety there is to need: a slot is written when it and every slot
// before it has been read, and later slots read rows that lie past everything written so far.
// A lane moves 16 bytes at a time, cp.async in and st.global out.  (One bulk copy per row slice instead: the same
// 394 us for 2 KiB rows, but 740 us against 490 for a head's 256-byte rows, of which the copy engine
// starts one every ~50 clocks.)
__global__ void __launch_bounds__(kMoveThreads, 2) evict_move_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int slots = p.slots;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + slots * kSlot);
  uint64_t* empty = full + slots;
  uint32_t* s_ok = reinterpret_cast<uint32_t*>(empty + slots);  // [slots][4]: rows of the slot that move
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool storer = warp >= kLoaders;
  if (threadIdx.x == 0) {
    for (int i = 0; i < slots; ++i) {
      mbar_init(&full[i], 33);  // every lane's copies, and the loader's row masks
      mbar_init(&empty[i], 32 * kStorers);
    }
  }
  __syncthreads();
  const int slice = p.slice_bytes, per_slot = min(kSlotRows, kSlot / slice);
  const int lg = 31 - __clz(slice >> 4);  // log2 of a row slice's 16-byte vectors
  int sc = 0;                             // slots so far (every warp counts them all)
  bool alive = true;
  asm volatile("griddepcontrol.wait;\n" ::: "memory");  // the kept lists
  for (int st = blockIdx.x; st < p.n_streams && alive; st += gridDim.x) {
    int t = st;
    const int range = t % p.ranges;
    t /= p.ranges;
    const int sl = t % p.slices;
    t /= p.slices;
    const int kind = t & 1;
    t >>= 1;
    const int u = t % p.units;
    t /= p.units;
    const int b = t % p.B;
    const EvictLayer& L = p.layer[t / p.B];
    const int n = evict_len(p, L, b, false), m = min(n, L.budget);
    const bool in_place = p.in_place != 0;
    if (in_place && n <= L.budget) continue;
    const int32_t* keep = L.keep + ((int64_t)b * p.units + u) * L.keep_stride;
    int j0 = range * p.range_rows;
    const int j1 = min(m, j0 + p.range_rows);
    if (in_place) {
      // rows before the first evicted one stay: the first j with keep[j] > j (keep[j] - j never falls)
      int lo = j0, hi = j1;
      while (lo < hi) {
        const int step = max(1, (hi - lo) / 32), j = lo + lane * step;
        const bool moved = j >= hi || __ldcg(keep + j) > j;
        const int f = __ffs(__ballot_sync(0xffffffffu, moved)) - 1;  // the first probe that moves, -1: none
        const int nlo = f < 0 ? lo + 31 * step + 1 : (f == 0 ? lo : lo + (f - 1) * step + 1);
        const int nhi = f < 0 ? hi : min(hi, lo + f * step);
        lo = nlo;
        hi = max(nhi, lo);
      }
      j0 = lo;
    }
    const int64_t col = (int64_t)u * p.unit_vecs * 16 + (int64_t)sl * slice;
    const int32_t* bt = L.bt + b * L.bt_stride;
    const int32_t* dt = L.dst + b * L.dst_stride;
    for (int j = j0; j < j1; j += per_slot, ++sc) {
      const int slot = sc % slots;
      const uint32_t use = (uint32_t)(sc / slots);
      uint8_t* buf = smem + slot * kSlot;
      if (!storer) {
        if (sc % kLoaders != warp) continue;
        int64_t src[4];
        uint32_t ok[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int r = x * 32 + lane;
          src[x] = -1;
          if (r < per_slot && j + r < j1) {
            const int i = __ldcg(keep + j + r);
            if (!in_place || i != j + r) {
              const int pg = lookup_page(p, L, bt, L.bt_stride, i);
              const int dp = lookup_page(p, L, dt, L.dst_stride, j + r);  // a row without a place is not read
              if (pg >= 0 && dp >= 0) src[x] = row_offset(p, L, pg, kind, i % p.P) + col;
            }
          }
          ok[x] = __ballot_sync(0xffffffffu, src[x] >= 0);
        }
        if (lane == 0 && !mbar_wait(&empty[slot], (use & 1u) ^ 1u)) {
          set_error(p.err, ABKV_DEVERR_TIMEOUT);
          alive = false;
        }
        alive = __shfl_sync(0xffffffffu, alive ? 1 : 0, 0) != 0;
        if (!alive) break;
        __syncwarp();  // lane 0's wait orders every lane's copies after the storers' reads
        if (lane == 0) {
#pragma unroll
          for (int x = 0; x < 4; ++x) s_ok[slot * 4 + x] = ok[x];
          mbar_arrive(&full[slot]);  // releases s_ok
        }
        // 16-byte vector v of 32 rows: row v >> lg
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int v1 = max(0, min(32, per_slot - x * 32)) << lg;
          for (int v = lane; v < v1; v += 32) {
            const int64_t from = __shfl_sync(0xffffffffu, src[x], v >> lg);
            if (from >= 0) cp_async16(buf + (((x * 32) << lg) + v) * 16, L.kv + from + (v & ((1 << lg) - 1)) * 16);
          }
        }
        cp_async_arrive(&full[slot]);  // this lane's copies
      } else {
        int64_t dst[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int r = x * 32 + lane;
          dst[x] = -1;
          if (r < per_slot && j + r < j1) {
            const int dp = lookup_page(p, L, dt, L.dst_stride, j + r);
            if (dp >= 0) dst[x] = row_offset(p, L, dp, kind, (j + r) % p.P) + col;
          }
        }
        if (!__all_sync(0xffffffffu, mbar_wait(&full[slot], use & 1u))) {
          if (lane == 0) set_error(p.err, ABKV_DEVERR_TIMEOUT);
          alive = false;
          break;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (!((s_ok[slot * 4 + x] >> lane) & 1u)) dst[x] = -1;
        const int part = warp - kLoaders;  // every storer takes its share of the slot's vectors
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int v1 = max(0, min(32, per_slot - x * 32)) << lg;
#pragma unroll 4
          for (int v = part * 32 + lane; v < v1; v += 32 * kStorers) {
            const int64_t to = __shfl_sync(0xffffffffu, dst[x], v >> lg);
            if (to >= 0)
              __stcs(reinterpret_cast<uint4*>(L.kv + to + (v & ((1 << lg) - 1)) * 16),
                     *reinterpret_cast<const uint4*>(buf + (((x * 32) << lg) + v) * 16));
          }
        }
        mbar_arrive(&empty[slot]);
      }
    }
  }
  asm volatile("cp.async.wait_all;\n" ::: "memory");  // where a wait gave up: no copy outlives its shared memory
}

size_t keep_bytes(int num_layers, int num_seqs, int units, const int32_t* budgets) {
  size_t total = 0;
  for (int l = 0; l < num_layers; ++l) total += (size_t)num_seqs * units * budgets[l] * 4;
  return (total + 255) / 256 * 256;
}

}  // namespace
}  // namespace abkv

using namespace abkv;

extern "C" size_t abkv_evict_by_weight_workspace_size(int num_layers, int num_seqs, int units,
                                                      const int32_t* budgets) {
  if (num_layers <= 0 || num_seqs <= 0 || units <= 0 || !budgets) return 0;
  for (int l = 0; l < num_layers; ++l)
    if (budgets[l] <= 0) return 0;
  return 256 + keep_bytes(num_layers, num_seqs, units, budgets);
}

extern "C" int abkv_evict_by_weight(void* const* kv, const int32_t* const* block_tables, const int64_t* bt_strides,
                                    const int32_t* const* dst_block_tables, const int64_t* dst_strides,
                                    const int32_t* const* seq_lens, int32_t* const* new_lens,
                                    const int64_t* num_blocks, const float* const* weights,
                                    const int64_t* weight_strides, int weight_rows, float* const* weights_out,
                                    const int64_t* weight_out_strides, int weight_out_rows, int32_t* const* keep,
                                    const int32_t* budgets, int num_layers, int num_seqs, int weight_units,
                                    int kv_layout, int num_kv_heads, int head_dim, int page_size,
                                    int max_pages_per_seq, int num_sinks, int num_recent, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (!kv || !block_tables || !bt_strides || !seq_lens || !new_lens || !num_blocks || !weights || !weight_strides ||
      !weights_out || !weight_out_strides || !budgets || (dst_block_tables && !dst_strides))
    return ABKV_ERR_INVALID_ARG;
  if (num_layers <= 0 || num_seqs <= 0 || page_size <= 0 || max_pages_per_seq <= 0 || num_sinks < 0 ||
      num_recent < 0 || weight_rows <= 0 || weight_out_rows <= 0 || (kv_layout != 0 && kv_layout != 1) ||
      (weight_units != 1 && weight_units != num_kv_heads))
    return ABKV_ERR_INVALID_ARG;
  if ((head_dim != 64 && head_dim != 128) ||
      (num_kv_heads != 1 && num_kv_heads != 2 && num_kv_heads != 4 && num_kv_heads != 8) || num_seqs > 65535 / 8)
    return ABKV_ERR_UNSUPPORTED;
  if ((int64_t)max_pages_per_seq * page_size > (1 << 30)) return ABKV_ERR_UNSUPPORTED;
  int max_budget = 0;
  for (int l = 0; l < num_layers; ++l) {
    if (!kv[l] || !block_tables[l] || !seq_lens[l] || !new_lens[l] || !weights[l] || !weights_out[l] ||
        (dst_block_tables && !dst_block_tables[l]) || (keep && !keep[l]) || num_blocks[l] <= 0 || bt_strides[l] <= 0 ||
        (dst_block_tables && dst_strides[l] <= 0))
      return ABKV_ERR_INVALID_ARG;
    if (dst_block_tables && dst_block_tables[l] == block_tables[l]) return ABKV_ERR_INVALID_ARG;
    // rows that a sequence may keep need a place: one without would be lost with its length reported
    const int64_t most = std::min({(int64_t)budgets[l], (int64_t)weight_rows, bt_strides[l] * page_size,
                                   (int64_t)max_pages_per_seq * page_size});
    if (dst_block_tables && dst_strides[l] < (most + page_size - 1) / page_size) return ABKV_ERR_INVALID_ARG;
    if (budgets[l] <= 0 || (int64_t)num_sinks + num_recent > budgets[l]) return ABKV_ERR_INVALID_ARG;
    if (new_lens[l] == seq_lens[l]) return ABKV_ERR_INVALID_ARG;  // other CTAs still read the old lengths
    if (num_blocks[l] > INT32_MAX) return ABKV_ERR_UNSUPPORTED;
    if (reinterpret_cast<uintptr_t>(kv[l]) & 15) return ABKV_ERR_INVALID_ARG;
    max_budget = std::max(max_budget, budgets[l]);
  }
  const size_t need = abkv_evict_by_weight_workspace_size(num_layers, num_seqs, weight_units, budgets);
  if (!workspace || workspace_bytes < (keep ? 256 : need) || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return ABKV_ERR_WORKSPACE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  EvictParams prm;
  std::memset(&prm, 0, sizeof(prm));
  prm.err = static_cast<int32_t*>(workspace);
  prm.B = num_seqs;
  prm.units = weight_units;
  prm.Hkv = num_kv_heads;
  prm.P = page_size;
  prm.max_rows = max_pages_per_seq * page_size;
  prm.w_rows = weight_rows;
  prm.out_rows = weight_out_rows;
  prm.sinks = num_sinks;
  prm.recent = num_recent;
  prm.row_vecs = num_kv_heads * head_dim / 8;
  prm.unit_vecs = prm.row_vecs / weight_units;
  prm.fa_layout = kv_layout;
  prm.in_place = dst_block_tables ? 0 : 1;
  prm.cached_keys = std::min(kMaxCachedKeys, std::min(prm.max_rows, prm.w_rows));
  const int smem = prm.cached_keys * 4;
  if (cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxCachedKeys * 4) !=
          cudaSuccess ||
      cudaFuncSetAttribute(evict_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMoveSmem) != cudaSuccess)
    return ABKV_ERR_CUDA;
  char* list = static_cast<char*>(workspace) + 256;
  for (int l0 = 0; l0 < num_layers; l0 += kMaxLayers) {
    const int nl = std::min(kMaxLayers, num_layers - l0);
    for (int i = 0; i < nl; ++i) {
      const int l = l0 + i;
      EvictLayer& a = prm.layer[i];
      a.kv = static_cast<char*>(kv[l]);
      a.bt = block_tables[l];
      a.bt_stride = bt_strides[l];
      a.dst = dst_block_tables ? dst_block_tables[l] : block_tables[l];
      a.dst_stride = dst_block_tables ? dst_strides[l] : bt_strides[l];
      a.seq_lens = seq_lens[l];
      a.new_lens = new_lens[l];
      a.w = weights[l];
      a.w_sb = weight_strides[2 * l];
      a.w_su = weight_strides[2 * l + 1];
      a.w_out = weights_out[l];
      a.o_sb = weight_out_strides[2 * l];
      a.o_su = weight_out_strides[2 * l + 1];
      a.num_blocks = num_blocks[l];
      a.budget = budgets[l];
      a.keep_stride = budgets[l];
      if (keep) {
        a.keep = keep[l];
      } else {
        a.keep = reinterpret_cast<int32_t*>(list);
        list += (size_t)num_seqs * weight_units * budgets[l] * 4;
      }
    }
    evict_select_kernel<<<dim3(weight_units, num_seqs, nl), kSelThreads, smem, s>>>(prm);
    // Streams: rows are split into ranges where they move elsewhere, and a row part into slices where they move
    // in place -- of 64 bytes at least, and of 1 KiB once every SM has a stream -- until every CTA has a few.
    const int part = prm.unit_vecs * 16;
    const int64_t base = (int64_t)nl * num_seqs * weight_units * 2;
    const int rows = std::min(max_budget, std::min(prm.max_rows, prm.w_rows));
    prm.slices = prm.ranges = 1;
    prm.range_rows = rows;
    if (dst_block_tables) {
      const int slot_rows = std::min(kSlotRows, kSlot / part), most = (rows + slot_rows - 1) / slot_rows;
      const int want = (int)std::min<int64_t>(most, (kStreamsPerCta * kMoveCtas + base - 1) / base);
      prm.range_rows = ((most + want - 1) / want) * slot_rows;
      prm.ranges = (rows + prm.range_rows - 1) / prm.range_rows;
    } else {
      while (base * prm.slices < kStreamsPerCta * kMoveCtas && part / prm.slices > 64 &&
             !(part / prm.slices <= 1024 && base * prm.slices >= 148))
        prm.slices *= 2;
    }
    prm.slice_bytes = part / prm.slices;
    const int64_t streams = base * prm.slices * prm.ranges;
    if (streams > INT32_MAX / 2) return ABKV_ERR_UNSUPPORTED;
    prm.n_streams = (int)streams;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min<int64_t>(streams, kMoveCtas));
    cfg.blockDim = dim3(kMoveThreads);
    // a stream or two of few slots need no deep ring (and its shared memory)
    const int per_slot = std::min(kSlotRows, kSlot / prm.slice_bytes);
    const int64_t used = ((streams + kMoveCtas - 1) / kMoveCtas) * ((prm.range_rows + per_slot - 1) / per_slot);
    prm.slots = (int)std::max<int64_t>(2, std::min<int64_t>(kSlots, used));
    cfg.dynamicSmemBytes = move_smem(prm.slots);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, evict_move_kernel, prm) != cudaSuccess) return ABKV_ERR_CUDA;
  }
  if (cudaGetLastError() != cudaSuccess) return ABKV_ERR_CUDA;
  return ABKV_OK;
}
