// dK and dV of the sink keys: the first n_sink keys, which every query row sees whatever its window
// (flash_attn_sink_bwd).  The windowed dK/dV kernel walks, for its 128 keys, the query tiles whose
// window reaches them; the sinks are seen by the whole query axis, so they would make one
// workgroup of every head as long as the sequence.  Here they are cut the other way:
//   dV_j = sum_i P_ij dO_i,  dK_j = scale * sum_i P_ij (dO_i . V_j - D_i) Q_i,   j < n_sink,
// over all rows i that see key j (inside the window or out of it: this kernel's rows replace what
// the windowed kernel wrote there, so nothing is counted twice and everything is rounded once).
//
// A workgroup owns 32 keys of one key/value head and a share of the (query head of the group, 32
// query rows) items; its waves take the items in turn, each with K, V and the accumulators of the
// same 32 keys in registers and a private Q / dO tile in LDS (no barrier in the loop; the next
// item's rows are in flight meanwhile).  What bounds it is reading Q and dO once per 32 sinks:
// 4 d bytes a row against 256 d flops a row and key block of MFMA (four products of 32 keys).  The waves' sums meet in LDS,
// the shares' as fp32 partials that sink_join_kernel adds in order: no atomics, same bits every run.
// Without scratch there is one share and the workgroup rounds its sums itself.
// Measured: 4 sinks, 8192 rows, 32 heads on 8, D = 128: 49 us (Q and dO, 134 MB, in 20 at the
// rate of a read stream; four items a wave, each a memory latency); 128 sinks, 2 x 2048 rows, 16
// heads on 2, d = 96: 25 us.  Two waves per SIMD instead of one with the next item in flight: 38 -> 25 us there.
#include <algorithm>

#include "flash_common.h"

namespace fa {
namespace {

constexpr int kSinkWaves = 4;
constexpr int kSinkKeys = 32;   // keys per workgroup
constexpr int kSinkRows = 32;   // query rows per item

struct SinkArgs {
  float *dk_part, *dv_part;  // [shares][b][h_k][n_kb * 32][d]; null: one share, written to p.dk / p.dv
  int n_kb, shares;
};

// D is head_dim rounded up to 32, 64, 96, 128, 192 or 256; columns from head_dim on are zeros
template <typename T, int D>
__global__ void __launch_bounds__(kSinkWaves * 64, D <= 96 ? 2 : 1) sink_dkdv_kernel(const Params p, const SinkArgs a) {
  using vec8 = typename Traits<T>::vec8;
  constexpr int QS = Pad<D>::kPlain;               // row stride of the Q and dO tiles, read plainly and transposed
  constexpr int CPR = D / 8, RPP = 64 / CPR;       // 16-byte chunks per row, rows per pass of a wave
  constexpr int NP = (kSinkRows + RPP - 1) / RPP;
  // Two waves per SIMD up to 96 columns; the next item in flight where the registers hold it (at 96 they do
  // not, and the other wave covers; at 128 they do with one wave, which is as fast as two that spill)
  constexpr bool kPrefetch = D <= 64 || D == 128;
  constexpr int kTile = kSinkRows * QS;
  constexpr int RS = D + 4;                        // row stride of the fp32 sums
  static_assert(kSinkKeys * RS * 4 <= 2 * kTile * (int)sizeof(T), "a wave's sums must fit its tiles");
  __shared__ __attribute__((aligned(16))) T tiles[kSinkWaves][2 * kTile];
  __shared__ __attribute__((aligned(16))) float lse_s[kSinkWaves][kSinkRows], dsm_s[kSinkWaves][kSinkRows];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r32 = lane & 31, g = lane >> 5;
  const int share = blockIdx.x % a.shares, kb = blockIdx.x / a.shares % a.n_kb, bhk = blockIdx.x / a.shares / a.n_kb;
  const int bi = bhk / p.h_k, hk = bhk % p.h_k, group = p.h / p.h_k;
  const int key0 = kb * kSinkKeys, key = key0 + r32, off = p.sk - p.sq;
  const bool key_ok = key < p.n_sink;

  vec8 kf[D / 16], vf[D / 16];
  {
    const T *kg = static_cast<const T *>(p.k) + bi * p.k_bs + (int64_t)key * p.k_rs + hk * p.k_hs;
    const T *vg = static_cast<const T *>(p.v) + bi * p.v_bs + (int64_t)key * p.v_rs + hk * p.v_hs;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const bool ok = key_ok && ks * 16 + g * 8 < p.d;
      kf[ks] = ok ? *reinterpret_cast<const vec8 *>(kg + ks * 16 + g * 8) : vec8{0};
      vf[ks] = ok ? *reinterpret_cast<const vec8 *>(vg + ks * 16 + g * 8) : vec8{0};
    }
  }
  float16v dk_acc[D / 32], dv_acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) { dk_acc[i] = float16v{0}; dv_acc[i] = float16v{0}; }

  // items: query head of the group x 32 rows, from the first row that the right side of the window
  // lets see key0
  const int u0 = p.wr >= 0 ? max(0, key0 - off - p.wr) / kSinkRows : 0;
  const int nu = max(0, (p.sq + kSinkRows - 1) / kSinkRows - u0);
  const int items = group * nu, per = (items + a.shares - 1) / a.shares;
  const int i1 = min(items, (share + 1) * per);

  T *Qt = tiles[wave], *dOt = tiles[wave] + kTile;
  uint4 qr[NP], dor[kPrefetch ? NP : 1];
  float lse_r = INFINITY, dsm_r = 0.f;
  const int ld_c = lane % CPR, ld_r = lane / CPR;
  auto load_rows = [&](const T *rows, int64_t stride, int q0, uint4 *reg) {
#pragma unroll
    for (int s = 0; s < NP; ++s) {
      const int r = s * RPP + ld_r, q = q0 + r;
      const bool in = ld_r < RPP && r < kSinkRows && q < p.sq && ld_c * 8 < p.d;
      reg[s] = in ? *reinterpret_cast<const uint4 *>(rows + (int64_t)q * stride + ld_c * 8) : uint4{0, 0, 0, 0};
    }
  };
  auto store_rows = [&](T *tile, const uint4 *reg) {
#pragma unroll
    for (int s = 0; s < NP; ++s) {
      const int r = s * RPP + ld_r;
      if (ld_r < RPP && r < kSinkRows) *reinterpret_cast<uint4 *>(&tile[r * QS + ld_c * 8]) = reg[s];
    }
  };
  auto load_item = [&](int it) {
    const int hi = hk * group + it / nu, q0 = (u0 + it % nu) * kSinkRows, q = q0 + r32;
    load_rows(static_cast<const T *>(p.q) + bi * p.q_bs + hi * p.q_hs, p.q_rs, q0, qr);
    // +inf: a row that does not exist contributes P = 0
    lse_r = q < p.sq ? p.lse[((int64_t)bi * p.h + hi) * p.sq + q] * kLog2e : INFINITY;
    dsm_r = q < p.sq ? p.dsoftmax[((int64_t)bi * p.h + hi) * p.sq_rounded + q] : 0.f;
    const T *dog = static_cast<const T *>(p.dout) + bi * p.o_bs + hi * p.o_hs;
    if constexpr (kPrefetch) {
      load_rows(dog, p.o_rs, q0, dor);
    } else {  // Q, then dO through the same registers
      store_rows(Qt, qr);
      load_rows(dog, p.o_rs, q0, qr);
    }
  };
  auto store_item = [&]() {
    if constexpr (kPrefetch) {
      store_rows(Qt, qr);
      store_rows(dOt, dor);
    } else {
      store_rows(dOt, qr);
    }
    if (g == 0) { lse_s[wave][r32] = lse_r; dsm_s[wave][r32] = -dsm_r; }
    FA_WAVE_SYNC();  // the wave's own tiles: written by all its lanes, read across lanes
  };

  const float c = p.scale_log2;
  int it = share * per + wave;
  if (kPrefetch && it < i1) {
    load_item(it);
    store_item();
  }
  for (; it < i1; it += kSinkWaves) {
    const bool has_next = it + kSinkWaves < i1;
    if constexpr (kPrefetch) {
      if (has_next) load_item(it + kSinkWaves);
    } else {
      load_item(it);
      store_item();
    }
    const int q0 = (u0 + it % nu) * kSinkRows;
    float16v s = float16v{0}, dp;
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {  // dP starts from -D of its row
      const float4 d4 = *reinterpret_cast<const float4 *>(&dsm_s[wave][i4 * 8 + g * 4]);
      dp[i4 * 4] = d4.x; dp[i4 * 4 + 1] = d4.y; dp[i4 * 4 + 2] = d4.z; dp[i4 * 4 + 3] = d4.w;
    }
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      s = Traits<T>::mfma(lds_read8<T>(&Qt[r32 * QS + ks * 16 + g * 8]), kf[ks], s);
      dp = Traits<T>::mfma(lds_read8<T>(&dOt[r32 * QS + ks * 16 + g * 8]), vf[ks], dp);
    }
    float pv[16], dsv[16];
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const float4 l4 = *reinterpret_cast<const float4 *>(&lse_s[wave][i4 * 8 + g * 4]);
      const float lq[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i4 * 4 + j, q = q0 + i4 * 8 + g * 4 + j;
        const bool kept = key_ok && (p.wr < 0 || key - off - q <= p.wr);
        const float pe = exp2_fast(fmaf(s[i], c, -lq[j]));
        pv[i] = kept ? pe : 0.f;
        dsv[i] = kept ? pe * dp[i] : 0.f;
      }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const vec8 pb = pack8<T>(&pv[w * 8]), dsb = pack8<T>(&dsv[w * 8]);
#pragma unroll
      for (int db = 0; db < D / 32; ++db) {
        dv_acc[db] = Traits<T>::mfma(lds_read_operand_tr<T>(dOt, QS, w * 16, db * 32), pb, dv_acc[db]);
        dk_acc[db] = Traits<T>::mfma(lds_read_operand_tr<T>(Qt, QS, w * 16, db * 32), dsb, dk_acc[db]);
      }
    }
    if (kPrefetch && has_next) store_item();  // after every read of this item in program order
  }

  // the waves' sums through LDS, dK then dV, each wave in its own region
  const int n_rows = min(kSinkKeys, p.n_sink - key0);
  auto join = [&](const float16v (&acc)[D / 32], float mul, float *part, void *out, int64_t bs, int64_t rs, int64_t hs) {
    __syncthreads();  // every wave has left its tiles, or the sums of dK have been read
    float *own = reinterpret_cast<float *>(tiles[wave]);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4)
        *reinterpret_cast<float4 *>(&own[r32 * RS + db * 32 + i4 * 8 + g * 4]) =
            float4{acc[db][i4 * 4] * mul, acc[db][i4 * 4 + 1] * mul, acc[db][i4 * 4 + 2] * mul, acc[db][i4 * 4 + 3] * mul};
    __syncthreads();
    for (int e = tid; e < n_rows * (D / 4); e += kSinkWaves * 64) {
      const int r = e / (D / 4), col = e % (D / 4) * 4;
      if (col >= p.d) continue;
      float4 t = *reinterpret_cast<const float4 *>(&reinterpret_cast<const float *>(tiles[0])[r * RS + col]);
#pragma unroll
      for (int w = 1; w < kSinkWaves; ++w) {
        const float4 x = *reinterpret_cast<const float4 *>(&reinterpret_cast<const float *>(tiles[w])[r * RS + col]);
        t.x += x.x; t.y += x.y; t.z += x.z; t.w += x.w;
      }
      if (part) {
        const int64_t row = ((((int64_t)share * p.b + bi) * p.h_k + hk) * a.n_kb + kb) * kSinkKeys + r;
        *reinterpret_cast<float4 *>(part + row * p.d + col) = t;
      } else {
        typedef T vec4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<vec4 *>(static_cast<T *>(out) + bi * bs + (int64_t)(key0 + r) * rs + hk * hs + col) = vec4{(T)t.x, (T)t.y, (T)t.z, (T)t.w};
      }
    }
  };
  join(dk_acc, p.scale, a.dk_part, p.dk, p.k_bs, p.k_rs, p.k_hs);
  join(dv_acc, 1.f, a.dv_part, p.dv, p.v_bs, p.v_rs, p.v_hs);
}

// the rows of the sinks = sums over the shares' partials, in order, rounded once; a thread per 4 columns
template <typename T>
__global__ void __launch_bounds__(256) sink_join_kernel(const Params p, const SinkArgs a) {
  const int cpr = p.d / 4;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= (int64_t)p.b * p.h_k * p.n_sink * cpr) return;
  const int col = (int)(e % cpr) * 4, key = (int)(e / cpr % p.n_sink);
  const int64_t bhk = e / cpr / p.n_sink;
  const int bi = (int)(bhk / p.h_k), hk = (int)(bhk % p.h_k);
  const int64_t src = (bhk * a.n_kb * kSinkKeys + key) * p.d + col, step = (int64_t)p.b * p.h_k * a.n_kb * kSinkKeys * p.d;
  float4 tk = float4{0, 0, 0, 0}, tv = float4{0, 0, 0, 0};
#pragma unroll 4
  for (int s = 0; s < a.shares; ++s) {
    const float4 x = *reinterpret_cast<const float4 *>(a.dk_part + src + s * step), y = *reinterpret_cast<const float4 *>(a.dv_part + src + s * step);
    tk.x += x.x; tk.y += x.y; tk.z += x.z; tk.w += x.w;
    tv.x += y.x; tv.y += y.y; tv.z += y.z; tv.w += y.w;
  }
  typedef T vec4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<vec4 *>(static_cast<T *>(p.dk) + bi * p.k_bs + (int64_t)key * p.k_rs + hk * p.k_hs + col) = vec4{(T)tk.x, (T)tk.y, (T)tk.z, (T)tk.w};
  *reinterpret_cast<vec4 *>(static_cast<T *>(p.dv) + bi * p.v_bs + (int64_t)key * p.v_rs + hk * p.v_hs + col) = vec4{(T)tv.x, (T)tv.y, (T)tv.z, (T)tv.w};
}

template <typename T, int D>
hipError_t sink_dkdv_td(const Params &p, const SinkArgs &a, hipStream_t stream) {
  FA_LAUNCH((sink_dkdv_kernel<T, D>), dim3((unsigned)((int64_t)p.b * p.h_k * a.n_kb * a.shares)), dim3(kSinkWaves * 64), stream, p, a);
  if (a.dk_part) {
    const int64_t n = (int64_t)p.b * p.h_k * p.n_sink * (p.d / 4);
    if (hipError_t e = hipGetLastError()) return e;
    FA_LAUNCH((sink_join_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), stream, p, a);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t sink_dkdv_t(const Params &p, const SinkArgs &a, hipStream_t stream) {
  if (p.d <= 32) return sink_dkdv_td<T, 32>(p, a, stream);
  if (p.d <= 64) return sink_dkdv_td<T, 64>(p, a, stream);
  if (p.d <= 96) return sink_dkdv_td<T, 96>(p, a, stream);
  if (p.d <= 128) return sink_dkdv_td<T, 128>(p, a, stream);
  if (p.d <= 192) return sink_dkdv_td<T, 192>(p, a, stream);
  return sink_dkdv_td<T, 256>(p, a, stream);
}

// two workgroups for every CU, at least two items a wave, at most 64 shares
int sink_shares(const Params &p) {
  const int64_t base = (int64_t)p.b * p.h_k * ((p.n_sink + kSinkKeys - 1) / kSinkKeys);
  const int64_t items = (int64_t)(p.h / p.h_k) * ((p.sq + kSinkRows - 1) / kSinkRows);
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>((512 + base - 1) / base, items / (2 * kSinkWaves)), 64));
}

}  // namespace

size_t sink_dkdv_bytes(const Params &p) {
  if (p.n_sink <= 0 || p.b * p.h_k == 0) return 0;
  const int shares = sink_shares(p);
  return shares == 1 ? 0 : (size_t)2 * shares * p.b * p.h_k * ((p.n_sink + kSinkKeys - 1) / kSinkKeys) * kSinkKeys * p.d * sizeof(float);
}

hipError_t launch_sink_dkdv(const Params &p, int dtype, void *ws, size_t ws_bytes, hipStream_t stream) {
  if (p.n_sink <= 0 || p.b * p.h_k == 0) return hipSuccess;
  SinkArgs a{};
  a.n_kb = (p.n_sink + kSinkKeys - 1) / kSinkKeys;
  a.shares = 1;
  const size_t need = sink_dkdv_bytes(p);
  void *owned = nullptr;
  if (need) {
    if (!ws || (reinterpret_cast<uintptr_t>(ws) & 15) != 0 || ws_bytes < need) {
      ws = nullptr;
      if (hipMallocAsync(&owned, need, stream) == hipSuccess) ws = owned;
      else { (void)hipGetLastError(); owned = nullptr; }
    }
    if (ws) {
      a.shares = sink_shares(p);
      a.dk_part = static_cast<float *>(ws);
      a.dv_part = a.dk_part + need / 2 / sizeof(float);
    }
  }
  hipError_t e = dtype == 1 ? sink_dkdv_t<_Float16>(p, a, stream) : sink_dkdv_t<__bf16>(p, a, stream);
  if (owned) {
    const hipError_t f = hipFreeAsync(owned, stream);
    if (e == hipSuccess) e = f;
  }
  return e;
}

}  // namespace fa
