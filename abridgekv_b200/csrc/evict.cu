// Eviction from a paged KV cache by accumulated attention weight, for sm_100a.
//
// For one unit (a KV head, or all heads together) of one (layer, sequence) of n rows with budget m < n:
// kept = the first num_sinks rows, the last num_recent rows, and of the rest the m - num_sinks -
// num_recent rows with the largest accumulated weight w (ties to the lower row), in row order.  Kept
// row i becomes row i of the destination table (the source pages themselves, or other pages of the
// pool), its weight becomes weight i, and weights past the new length become 0.
//
// Two kernels.  select: one CTA per unit.  The weights become order-preserving 32-bit keys (-0 as
// +0, NaN as -inf), are held in shared memory, and the (m - sinks - recent)-th largest key is found by
// three histogram passes over 11, 11 and 10 key bits.  A warp first groups equal digits (attention
// weights share few exponents: one shared-memory add per distinct digit instead of up to 32 on one
// address).  Then every warp walks its contiguous share of the rows twice, counting and emitting by
// ballot, so the kept list comes out in row order with one scan over the warps.
// move: bound by memory.  Into other pages every row is independent: a warp has 8 vectors per lane in
// flight.  In place, kept row i moves from keep[i] >= i to i: a chunk of rows is read, the CTA
// synchronises, the chunk is written.  Later chunks read rows >= keep[first of the chunk] > every row
// written so far, so only the order read-before-write inside a chunk matters; 64-byte column slices of
// the row are independent of one another and give the CTAs.
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
constexpr int kMoveThreads = 256;

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

// Exclusive prefix over the block of one value per warp's lane 0 pattern: v summed over warps before this one.
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
  __shared__ int s_pick[2];  // digit chosen by a pass, rows still wanted inside it
  __shared__ int s_fix[kSelWarps], s_eq[kSelWarps];
  const EvictLayer& L = p.layer[blockIdx.z];
  const int b = blockIdx.y, u = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = evict_len(p, L, b, u == 0 && tid == 0);
  const int m = min(n, L.budget);
  if (u == 0 && tid == 0) L.new_lens[b] = m;
  const float* w = L.w + b * L.w_sb + u * L.w_su;
  int32_t* keep = L.keep + ((int64_t)b * p.units + u) * L.keep_stride;

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
          const uint32_t peers = __match_any_sync(0xffffffffu, digit);
          if (in && lane == __ffs(peers) - 1) atomicAdd(&s_hist[digit], __popc(peers));
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
        } else if (before + c0 < want && want <= before + c0 + c1) {
          s_pick[0] = kBins - 2 - 2 * tid;
          s_pick[1] = want - before - c0;
        }
        __syncthreads();
        prefix |= (uint32_t)s_pick[0] << shift;
        mask |= dmask << shift;
        want = s_pick[1];
      }
    }
    // now: every key > prefix is kept, and the first `want` rows with key == prefix
    const bool none = m - s - p.recent <= 0;
    auto classify = [&](int i, bool& fix, bool& eq) {
      fix = eq = false;
      if (i >= n) return;
      if (i < s || i >= e) {
        fix = true;
      } else if (!none) {
        const uint32_t k = key_at(i);
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
      if (take) keep[at + __popc(tm & below)] = i0 + lane;
      at += __popc(tm);
      ebase += __popc(em);
    }
    for (int i = m + tid; i < L.keep_stride; i += kSelThreads) keep[i] = -1;
  }
  __syncthreads();  // the list is complete (and visible to this CTA)
  // weights: chunks read whole, then written (w_out may be w: rows only move down)
  constexpr int kPer = 8;
  float* wo = L.w_out + b * L.o_sb + u * L.o_su;
  const int mo = min(m, p.out_rows);
  if (mo < m && tid == 0) set_error(p.err, ABKV_DEVERR_SEQ_OOB);
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
  for (int j = mo + tid; j < p.out_rows; j += kSelThreads) wo[j] = 0.f;
}

// Byte offset of (page, K or V, row in page) in the cache.
__device__ __forceinline__ int64_t row_offset(const EvictParams& p, const EvictLayer& L, int pg, int kind, int off) {
  const int64_t plane = p.fa_layout ? (int64_t)kind * L.num_blocks + pg : 2 * (int64_t)pg + kind;
  return (plane * p.P + off) * (int64_t)p.row_vecs * 16;
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

// Into other pages: 256 vectors of K and V rows per warp and step, 8 per lane in flight.
__global__ void __launch_bounds__(kMoveThreads) evict_copy_kernel(const __grid_constant__ EvictParams p) {
  const EvictLayer& L = p.layer[blockIdx.z];
  const int b = blockIdx.y / p.units, u = blockIdx.y % p.units;
  const int lane = threadIdx.x & 31;
  const int m = min(evict_len(p, L, b, false), L.budget);
  const int uv = p.unit_vecs, rows_per_step = 128 / uv;  // K and V vectors of the step's rows: 256
  const int j0 = (blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5)) * rows_per_step;
  if (j0 >= m) return;
  const int32_t* keep = L.keep + ((int64_t)b * p.units + u) * L.keep_stride;
  const int32_t* bt = L.bt + b * L.bt_stride;
  const int32_t* dt = L.dst + b * L.dst_stride;
  uint4 buf[8];
  uint4* dst[8];
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    const int v = x * 32 + lane, kind = v >> 7, rv = v & 127;
    const int j = j0 + rv / uv, c = rv % uv;
    dst[x] = nullptr;
    if (j >= m) continue;
    const int i = __ldg(keep + j);
    const int sp = lookup_page(p, L, bt, L.bt_stride, i), dp = lookup_page(p, L, dt, L.dst_stride, j);
    if (sp < 0 || dp < 0) continue;
    const int64_t col = ((int64_t)u * uv + c) * 16;
    buf[x] = ld_stream_v4(L.kv + row_offset(p, L, sp, kind, i % p.P) + col);
    dst[x] = reinterpret_cast<uint4*>(L.kv + row_offset(p, L, dp, kind, j % p.P) + col);
  }
#pragma unroll
  for (int x = 0; x < 8; ++x)
    if (dst[x]) __stcs(dst[x], buf[x]);
}

// In place: one CTA owns a 64-byte column slice of K or V of a unit; chunks of 512 rows are read, then written.
__global__ void __launch_bounds__(kMoveThreads) evict_shift_kernel(const __grid_constant__ EvictParams p) {
  const EvictLayer& L = p.layer[blockIdx.z];
  const int b = blockIdx.y / p.units, u = blockIdx.y % p.units;
  const int slices = p.unit_vecs / 4;
  const int kind = blockIdx.x / slices, slice = blockIdx.x % slices;
  const int n = evict_len(p, L, b, false);
  if (n <= L.budget) return;
  const int m = L.budget;
  const int32_t* keep = L.keep + ((int64_t)b * p.units + u) * L.keep_stride;
  const int32_t* bt = L.bt + b * L.bt_stride;
  const int64_t col = ((int64_t)u * p.unit_vecs + slice * 4 + (threadIdx.x & 3)) * 16;
  const int r = threadIdx.x >> 2;  // 64 rows per step
  constexpr int kStep = kMoveThreads / 4, kPer = 8;
  for (int j0 = 0; j0 < m; j0 += kStep * kPer) {
    uint4 buf[kPer];
    uint4* dst[kPer];
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
      const int j = j0 + x * kStep + r;
      dst[x] = nullptr;
      if (j >= m) continue;
      const int i = __ldg(keep + j);
      if (i == j) continue;  // kept where it is
      const int sp = lookup_page(p, L, bt, L.bt_stride, i), dp = lookup_page(p, L, bt, L.bt_stride, j);
      if (sp < 0 || dp < 0) continue;
      buf[x] = __ldcg(reinterpret_cast<const uint4*>(L.kv + row_offset(p, L, sp, kind, i % p.P) + col));
      dst[x] = reinterpret_cast<uint4*>(L.kv + row_offset(p, L, dp, kind, j % p.P) + col);
    }
    __syncthreads();  // every row of the chunk has been read
#pragma unroll
    for (int x = 0; x < kPer; ++x)
      if (dst[x]) __stcg(dst[x], buf[x]);
  }
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
  prm.cached_keys = std::min(kMaxCachedKeys, std::min(prm.max_rows, prm.w_rows));
  const int smem = prm.cached_keys * 4;
  if (cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxCachedKeys * 4) !=
      cudaSuccess)
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
    if (dst_block_tables) {
      const int rows = std::min(max_budget, std::min(prm.max_rows, prm.w_rows));
      const int per_cta = (kMoveThreads / 32) * (128 / prm.unit_vecs);
      evict_copy_kernel<<<dim3((rows + per_cta - 1) / per_cta, num_seqs * weight_units, nl), kMoveThreads, 0, s>>>(prm);
    } else {
      evict_shift_kernel<<<dim3(2 * prm.unit_vecs / 4, num_seqs * weight_units, nl), kMoveThreads, 0, s>>>(prm);
    }
  }
  if (cudaGetLastError() != cudaSuccess) return ABKV_ERR_CUDA;
  return ABKV_OK;
}
