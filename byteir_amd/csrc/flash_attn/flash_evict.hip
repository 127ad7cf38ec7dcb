// Eviction from a key/value cache by accumulated attention weight (flash_attn_evict): of every
// (sequence, key/value head) at most `budget` rows stay -- the first n_sink, the last n_recent
// and, of those between, the ones of greatest weight (equal weights: the lower row; NaN counts
// below everything) -- and move to the front in their order.
//
// Two kernels.  evict_select_kernel, one workgroup per (sequence, head), finds the weight of the last row
// that stays by radix selection on the order-preserving bits of the weights (three passes of 11,
// 11 and 10 bits over LDS histograms; the weights are a few hundred KiB at most and stay in L2),
// then writes the rows that stay in ascending order: every wave counts its own contiguous part
// with ballots, one scan joins the waves' counts, and each wave writes its part.  It is bound by
// the latency of its passes.  The moving kernel is bound by HBM: each row that stays is read and
// written once.  Into another cache a thread moves one 16-byte chunk, all in parallel.  In place
// a row never moves up (rank <= row), so a workgroup that owns a column slice of one head and
// walks its rows in order, reading a block of rows before a barrier and writing it after, never
// overwrites a row that is still to be read.
// Measured, 16 sequences of 5001..16384 rows to 4096, 8 heads, D = 128: selection 22 us, move 102 us
// (537 MB read and written, 5.3 TB/s); one of 4096 rows to 1024: 9.6 and 3 us.
#include <algorithm>

#include "flash_paged.h"

namespace fa {
namespace {

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;
constexpr int kSelRegs = 16;  // rows a thread can hold: 16384 a head

// bits whose unsigned order is that of the weights: -0 as +0, NaN below -inf
__device__ __forceinline__ uint32_t order_bits(float f) {
  uint32_t u = __builtin_bit_cast(uint32_t, f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0;
  if (u == 0x80000000u) u = 0;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Regs: the rows that compete fit kSelRegs a thread and are read once; else every pass reads them
template <bool Regs>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t wave_sum[kSelWaves], above[kSelWaves], equal[kSelWaves];
  __shared__ uint32_t found[2];  // the bin of the last row that stays, rows above that bin
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int bhk = blockIdx.x, bi = bhk / p.h_k;
  const int len = max(0, min(p.seqlens[bi], p.from.capacity()));
  const float *w = p.w + (int64_t)bhk * p.from.capacity();
  int *kept = p.kept + (int64_t)bhk * p.budget;
  if (len <= p.budget) {
    for (int i = tid; i < p.budget; i += kSelThreads) kept[i] = i < len ? i : -1;
    return;
  }
  const int lo = p.n_sink, hi = len - p.n_recent;  // rows that compete; sinks + recent <= budget < len
  uint32_t take = (uint32_t)(p.budget - p.n_sink - p.n_recent);
  for (int i = tid; i < lo; i += kSelThreads) kept[i] = i;
  for (int i = tid; i < p.n_recent; i += kSelThreads) kept[p.budget - p.n_recent + i] = hi + i;
  if (take == 0) return;

  // a wave owns a contiguous part of the rows, 64 at a time: row w0 + 64 k + lane for k < n_it
  const int part = ((hi - lo + kSelWaves - 1) / kSelWaves + 63) & ~63, n_it = part / 64;
  const int w0 = lo + wave * part, w1 = min(hi, w0 + part);
  uint32_t own[Regs ? kSelRegs : 1];
  if constexpr (Regs) {
#pragma unroll
    for (int k = 0; k < kSelRegs; ++k) {
      const int i = w0 + k * 64 + lane;
      own[k] = k < n_it && i < w1 ? order_bits(w[i]) : 0;
    }
  }
  // body(row, its bits, whether it exists) for every 64 rows of the wave
  auto each = [&](auto body) {
    if constexpr (Regs) {
#pragma unroll
      for (int k = 0; k < kSelRegs; ++k) {
        if (k >= n_it) break;
        body(w0 + k * 64 + lane, own[k], w0 + k * 64 + lane < w1);
      }
    } else {
      for (int k = 0; k < n_it; ++k) {
        const int i = w0 + k * 64 + lane;
        const uint32_t u = i < w1 ? order_bits(w[i]) : 0;
        body(i, u, i < w1);
      }
    }
  };

  // the `take`-th greatest: its leading bits, refined by one digit per pass
  uint32_t prefix = 0, mask = 0;
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digit = pass == 2 ? 1023 : 2047;
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    each([&](int, uint32_t u, bool ok) {
      if (ok && (u & mask) == prefix) FA_LDS_ADD(&hist[(u >> shift) & digit], 1u);
    });
    __syncthreads();
    // bins from the greatest down, two per thread: rows in the bins above this thread's
    const uint32_t b0 = hist[kBins - 1 - 2 * tid], b1 = hist[kBins - 2 - 2 * tid];
    uint32_t incl = b0 + b1;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t t = (uint32_t)__builtin_amdgcn_ds_bpermute((lane - off) * 4, (int)incl);
      if (lane >= off) incl += t;
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    for (int x = 0; x < wave; ++x) incl += wave_sum[x];
    const uint32_t before = incl - b0 - b1;
    if (before < take && take <= incl) {  // one thread
      const bool first = take <= before + b0;
      found[0] = (uint32_t)(kBins - (first ? 1 : 2) - 2 * tid);
      found[1] = first ? before : before + b0;
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= digit << shift;
    take -= found[1];  // of the rows that share the prefix, this many stay
  }
  // rows above `prefix` stay, and the first `take` of those equal to it
  uint32_t n_above = 0, n_equal = 0;
  each([&](int, uint32_t u, bool ok) {
    n_above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(ok && u > prefix));
    n_equal += __builtin_popcountll(__builtin_amdgcn_ballot_w64(ok && u == prefix));
  });
  if (lane == 0) { above[wave] = n_above; equal[wave] = n_equal; }
  __syncthreads();
  uint32_t at_above = 0, at_equal = 0;
  for (int x = 0; x < wave; ++x) { at_above += above[x]; at_equal += equal[x]; }
  const uint64_t below_me = (uint64_t(1) << lane) - 1;
  each([&](int i, uint32_t u, bool ok) {
    const uint64_t ab = __builtin_amdgcn_ballot_w64(ok && u > prefix), eq = __builtin_amdgcn_ballot_w64(ok && u == prefix);
    const uint32_t my_above = at_above + __builtin_popcountll(ab & below_me), my_equal = at_equal + __builtin_popcountll(eq & below_me);
    const bool is_above = (ab >> lane) & 1, is_equal = (eq >> lane) & 1;
    if (is_above || (is_equal && my_equal < take)) kept[lo + my_above + min(my_equal, take)] = i;
    at_above += __builtin_popcountll(ab);
    at_equal += __builtin_popcountll(eq);
  });
}

__device__ __forceinline__ void write_length(const EvictParams &p, int bi) {
  const int n = p.seqlens[bi];
  p.seqlens_out[bi] = n < 0 ? n : min(min(n, p.from.capacity()), p.budget);
}

// into another cache: a thread moves a 16-byte chunk of K and of V of one row (the chunks of a row, then
// the heads, are neighbours, as in the cache that is written; two or four rows a thread: 106 and 115 us
// against 102 on 16 x 4096 rows, 8 heads, D = 128), the threads behind those a weight each
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictParams p) {
  const int cpr = p.d / 8;
  const int64_t rows = (int64_t)p.b * p.budget * p.h_k, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e < p.b) write_length(p, (int)e);
  typedef unsigned short u16;  // either storage type
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  if (e < rows * cpr) {
    const int c = (int)(e % cpr), hk = (int)(e / cpr % p.h_k);
    const int i = (int)(e / cpr / p.h_k % p.budget), bi = (int)(e / cpr / p.h_k / p.budget);
    const int src = p.kept[((int64_t)bi * p.h_k + hk) * p.budget + i];
    if (src < 0) return;
    int sr, dr;
    const int sp = p.from.locate(bi, src, sr), dp = p.to.locate(bi, i, dr);
    if (sp < 0 || dp < 0) return;
    const u32x4 k = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(static_cast<const u16 *>(p.k) + sp * p.from.k_ps + sr * p.from.k_rs + hk * p.from.k_hs + c * 8));
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(static_cast<const u16 *>(p.v) + sp * p.from.v_ps + sr * p.from.v_rs + hk * p.from.v_hs + c * 8));
    *reinterpret_cast<u32x4 *>(static_cast<u16 *>(p.k_out) + dp * p.to.k_ps + dr * p.to.k_rs + hk * p.to.k_hs + c * 8) = k;
    *reinterpret_cast<u32x4 *>(static_cast<u16 *>(p.v_out) + dp * p.to.v_ps + dr * p.to.v_rs + hk * p.to.v_hs + c * 8) = v;
  } else if (e < rows * cpr + rows) {
    const int64_t x = e - rows * cpr;
    const int src = p.kept[x];
    if (src >= 0) p.w_out[x / p.budget * p.to.capacity() + x % p.budget] = p.w[x / p.budget * p.from.capacity() + src];
  }
}

// in place: workgroup (sequence, head, slice): slices [0, 2 * n_slices) are column slices of K and V,
// `cols` chunks each; the last one is the weights.  Block n of 1024 / cols rows is stored behind a
// barrier that every wave reaches only with its loads of block n complete; block n + 1 is in
// flight by then, whose sources lie behind everything that block n's stores touch.
__global__ void __launch_bounds__(1024) evict_in_place_kernel(const EvictParams p, int n_slices, int cols) {
  const int slice = blockIdx.x % (2 * n_slices + 1), bhk = blockIdx.x / (2 * n_slices + 1);
  const int bi = bhk / p.h_k, hk = bhk % p.h_k, tid = threadIdx.x;
  const int *kept = p.kept + (int64_t)bhk * p.budget;
  typedef unsigned short u16;
  if (slice == 2 * n_slices) {
    if (hk == 0 && tid == 0) write_length(p, bi);
    const float *w = p.w + (int64_t)bhk * p.from.capacity();
    float *out = p.w_out + (int64_t)bhk * p.to.capacity();
    int src = tid < p.budget ? kept[tid] : -1;
    float x = src >= 0 ? w[src] : 0.f;
    for (int i0 = 0; i0 < p.budget; i0 += 1024) {
      const int i = i0 + tid, src_next = i + 1024 < p.budget ? kept[i + 1024] : -1;
      const float x_next = src_next >= 0 ? w[src_next] : 0.f;
      FA_PIN(x);  // arrived
      __syncthreads();
      if (src >= 0) out[i] = x;
      src = src_next;
      x = x_next;
    }
    return;
  }
  const bool is_v = slice >= n_slices;
  u16 *base = static_cast<u16 *>(is_v ? p.v_out : p.k_out) + hk * (is_v ? p.from.v_hs : p.from.k_hs);
  const int64_t ps = is_v ? p.from.v_ps : p.from.k_ps, rs = is_v ? p.from.v_rs : p.from.k_rs;
  const int c = slice % n_slices * cols + tid % cols, r = tid / cols, rows = 1024 / cols;
  struct Row { u16 *to; uint4 x; };  // null: nothing to store
  auto load = [&](int i) {
    Row row{nullptr, uint4{0, 0, 0, 0}};
    const int src = i < p.budget && c * 8 < p.d ? kept[i] : -1;
    if (src > i) {  // a row that stays where it is needs nothing
      int sr, dr;
      const int sp = p.from.locate(bi, src, sr), dp = p.from.locate(bi, i, dr);
      if (sp >= 0 && dp >= 0) {
        row.to = base + dp * ps + dr * rs + c * 8;
        row.x = *reinterpret_cast<const uint4 *>(base + sp * ps + sr * rs + c * 8);
      }
    }
    return row;
  };
  Row row = load(r);
  for (int i0 = 0; i0 < p.budget; i0 += rows) {
    const Row next = load(i0 + rows + r);
    FA_PIN2(row.x.x, row.x.y);  // arrived
    FA_PIN2(row.x.z, row.x.w);
    __syncthreads();
    if (row.to) *reinterpret_cast<uint4 *>(row.to) = row.x;
    row = next;
  }
}

}  // namespace

hipError_t launch_evict(const EvictParams &p, hipStream_t stream) {
  const int64_t bhk = (int64_t)p.b * p.h_k;
  if (p.from.capacity() <= kSelRegs * kSelThreads) FA_LAUNCH((evict_select_kernel<true>), dim3((unsigned)bhk), dim3(kSelThreads), stream, p);
  else FA_LAUNCH((evict_select_kernel<false>), dim3((unsigned)bhk), dim3(kSelThreads), stream, p);
  if (hipError_t e = hipGetLastError()) return e;
  if (p.in_place) {
    const int groups = evict_groups(p.d);
    FA_LAUNCH((evict_in_place_kernel), dim3((unsigned)(bhk * groups)), dim3(1024), stream, p, (groups - 1) / 2, kEvictCols);
  } else {
    const int64_t n = bhk * p.budget * (p.d / 8 + 1);
    FA_LAUNCH((evict_move_kernel), dim3((unsigned)((n + 255) / 256)), dim3(256), stream, p);
  }
  return hipGetLastError();
}

}  // namespace fa
