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
#include <algorithm>

#include "flash_paged.h"

namespace fa {
namespace {

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;

// bits whose unsigned order is that of the weights: -0 as +0, NaN below -inf
__device__ __forceinline__ uint32_t order_bits(float f) {
  uint32_t u = __builtin_bit_cast(uint32_t, f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0;
  if (u == 0x80000000u) u = 0;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

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

  // the `take`-th greatest: its leading bits, refined by one digit per pass
  uint32_t prefix = 0, mask = 0;
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digit = pass == 2 ? 1023 : 2047;
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += kSelThreads) {
      const uint32_t u = order_bits(w[i]);
      if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & digit], 1u);
    }
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
  // rows above `prefix` stay, and the first `take` of those equal to it.  A wave owns a contiguous part.
  const int part = ((hi - lo + kSelWaves - 1) / kSelWaves + 63) & ~63;
  const int w0 = lo + wave * part, w1 = min(hi, w0 + part);
  uint32_t n_above = 0, n_equal = 0;
  for (int i0 = w0; i0 < w1; i0 += 64) {
    const int i = i0 + lane;
    const uint32_t u = i < w1 ? order_bits(w[i]) : 0;
    n_above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < w1 && u > prefix));
    n_equal += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < w1 && u == prefix));
  }
  if (lane == 0) { above[wave] = n_above; equal[wave] = n_equal; }
  __syncthreads();
  uint32_t at_above = 0, at_equal = 0;
  for (int x = 0; x < wave; ++x) { at_above += above[x]; at_equal += equal[x]; }
  const uint64_t below_me = (uint64_t(1) << lane) - 1;
  for (int i0 = w0; i0 < w1; i0 += 64) {
    const int i = i0 + lane;
    const uint32_t u = i < w1 ? order_bits(w[i]) : 0;
    const uint64_t ab = __builtin_amdgcn_ballot_w64(i < w1 && u > prefix), eq = __builtin_amdgcn_ballot_w64(i < w1 && u == prefix);
    const uint32_t my_above = at_above + __builtin_popcountll(ab & below_me), my_equal = at_equal + __builtin_popcountll(eq & below_me);
    const bool is_above = (ab >> lane) & 1, is_equal = (eq >> lane) & 1;
    if (is_above || (is_equal && my_equal < take)) kept[lo + my_above + min(my_equal, take)] = i;
    at_above += __builtin_popcountll(ab);
    at_equal += __builtin_popcountll(eq);
  }
}

__device__ __forceinline__ void write_length(const EvictParams &p, int bi) {
  const int n = p.seqlens[bi];
  p.seqlens_out[bi] = n < 0 ? n : min(min(n, p.from.capacity()), p.budget);
}

// into another cache: threads [0, b * budget * h_k * d / 8) move a 16-byte chunk of K and of V each (the
// chunks of a row, then the heads, are neighbours, as in the cache that is written), those behind
// them a weight each
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictParams p) {
  const int cpr = p.d / 8;
  const int64_t rows = (int64_t)p.b * p.budget * p.h_k, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e < p.b) write_length(p, (int)e);
  typedef unsigned short u16;  // either storage type
  if (e < rows * cpr) {
    const int c = (int)(e % cpr), hk = (int)(e / cpr % p.h_k);
    const int i = (int)(e / cpr / p.h_k % p.budget), bi = (int)(e / cpr / p.h_k / p.budget);
    const int src = p.kept[((int64_t)bi * p.h_k + hk) * p.budget + i];
    if (src < 0) return;
    int sr, dr;
    const int sp = p.from.locate(bi, src, sr), dp = p.to.locate(bi, i, dr);
    if (sp < 0 || dp < 0) return;
    const uint4 k = *reinterpret_cast<const uint4 *>(static_cast<const u16 *>(p.k) + sp * p.from.k_ps + sr * p.from.k_rs + hk * p.from.k_hs + c * 8);
    const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const u16 *>(p.v) + sp * p.from.v_ps + sr * p.from.v_rs + hk * p.from.v_hs + c * 8);
    *reinterpret_cast<uint4 *>(static_cast<u16 *>(p.k_out) + dp * p.to.k_ps + dr * p.to.k_rs + hk * p.to.k_hs + c * 8) = k;
    *reinterpret_cast<uint4 *>(static_cast<u16 *>(p.v_out) + dp * p.to.v_ps + dr * p.to.v_rs + hk * p.to.v_hs + c * 8) = v;
  } else if (e < rows * cpr + rows) {
    const int64_t x = e - rows * cpr;
    const int i = (int)(x % p.budget);
    const int64_t bhk = x / p.budget;
    const int src = p.kept[x];
    if (src >= 0) p.w_out[bhk * p.to.capacity() + i] = p.w[bhk * p.from.capacity() + src];
  }
}

// in place: workgroup (sequence, head, slice): slices [0, 2 * n_slices) are column slices of K and V,
// `cols` chunks each; the last one is the weights
__global__ void __launch_bounds__(1024) evict_in_place_kernel(const EvictParams p, int n_slices, int cols) {
  const int slice = blockIdx.x % (2 * n_slices + 1), bhk = blockIdx.x / (2 * n_slices + 1);
  const int bi = bhk / p.h_k, hk = bhk % p.h_k, tid = threadIdx.x;
  const int *kept = p.kept + (int64_t)bhk * p.budget;
  typedef unsigned short u16;
  if (slice == 2 * n_slices) {
    if (hk == 0 && tid == 0) write_length(p, bi);
    const float *w = p.w + (int64_t)bhk * p.from.capacity();
    float *out = p.w_out + (int64_t)bhk * p.to.capacity();
    for (int i0 = 0; i0 < p.budget; i0 += 1024) {
      const int i = i0 + tid, src = i < p.budget ? kept[i] : -1;
      const float x = src >= 0 ? w[src] : 0.f;
      __syncthreads();
      if (src >= 0) out[i] = x;
      __syncthreads();
    }
    return;
  }
  const bool is_v = slice >= n_slices;
  u16 *base = static_cast<u16 *>(is_v ? p.v_out : p.k_out) + hk * (is_v ? p.from.v_hs : p.from.k_hs);
  const int64_t ps = is_v ? p.from.v_ps : p.from.k_ps, rs = is_v ? p.from.v_rs : p.from.k_rs;
  const int c = slice % n_slices * cols + tid % cols, r = tid / cols, rows = 1024 / cols;
  for (int i0 = 0; i0 < p.budget; i0 += rows) {
    const int i = i0 + r, src = r < rows && i < p.budget && c * 8 < p.d ? kept[i] : -1;
    int sr, dr = 0, sp = -1, dp = -1;
    uint4 x = uint4{0, 0, 0, 0};
    if (src > i) {  // a row that stays where it is needs nothing
      sp = p.from.locate(bi, src, sr);
      dp = p.from.locate(bi, i, dr);
      if (sp >= 0 && dp >= 0) x = *reinterpret_cast<const uint4 *>(base + sp * ps + sr * rs + c * 8);
    }
    __syncthreads();
    if (sp >= 0 && dp >= 0) *reinterpret_cast<uint4 *>(base + dp * ps + dr * rs + c * 8) = x;
    __syncthreads();
  }
}

}  // namespace

hipError_t launch_evict(const EvictParams &p, hipStream_t stream) {
  const int64_t bhk = (int64_t)p.b * p.h_k;
  FA_LAUNCH((evict_select_kernel), dim3((unsigned)bhk), dim3(kSelThreads), stream, p);
  if (hipError_t e = hipGetLastError()) return e;
  if (p.in_place) {
    const int cols = 4, n_slices = (p.d / 8 + cols - 1) / cols;
    FA_LAUNCH((evict_in_place_kernel), dim3((unsigned)(bhk * (2 * n_slices + 1))), dim3(1024), stream, p, n_slices, cols);
  } else {
    const int64_t n = bhk * p.budget * (p.d / 8 + 1);
    FA_LAUNCH((evict_move_kernel), dim3((unsigned)((n + 255) / 256)), dim3(256), stream, p);
  }
  return hipGetLastError();
}

}  // namespace fa
