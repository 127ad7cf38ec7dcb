// Attention of a few query rows (one new token, a draft, an observation window) over a key/value
// cache in pages, with a window and sink keys, appending the new rows on the way
// (flash_attn_paged):
//   o_i = sum_j P_ij v_j,  P_ij = exp(scale q_i.k_j - lse_i),  j over the keys that row i sees,
// and, when asked for, weights_j += sum of P_ij over the rows and the query heads that share
// key/value head j belongs to.
//
// HBM-bound: every visible K and V row is read once.  The structure is that of flash_decode.hip:
// the query heads of a key/value head times the query rows are the columns of one S^T tile (32
// columns; more make more tiles), a wave streams units of 32 keys through registers into private
// LDS tiles with the next unit in flight and no barrier in the loop, the waves join in LDS, the
// workgroups that share a sequence's keys join through fp32 partials in a second kernel.
// What differs: a unit's 32 row addresses come from the block table, looked up by one lane per row a
// unit ahead of the loads that need them: a scalar for the rows of one pass where the page size is a
// multiple of their number, else handed round by lane permutes; the keys are cut by
// the sequence's own length (units are numbered through sinks and window, and every sequence
// shares its units out evenly over the splits the grid offers it), so a short sequence in a long
// cache does not wait for one workgroup; rows that nobody sees (outside the window, behind the
// last key, on an absent page) are not read and count as zeros.
// Measured, 32 heads on 8, D = 128, fp16: 64 x 8192 keys 340 us = 6.3 TB/s; 64 x 1000..8191 keys
// (bf16, 1.21 GB) 199 us = 6.0 TB/s; one sequence of 31 keys 8.6 us, of 300 12 us (latency: length,
// table, rows, then 2 us a unit); 16 heads, D = 64, 64 x 8192 keys 366 us = 5.9 TB/s.  Above 128 columns
// the registers do not hold a unit in flight: 80 bytes a lane spill, 148 with weights.  Every 32
// columns (rows x query heads of a key/value head) are workgroups of their own that read the keys again.
#include <algorithm>

#include "flash_paged.h"

namespace fa {
namespace {

constexpr int kWaves = 4;
constexpr int kUnit = 32;  // keys per unit

// D: the tile width, the smallest of 32, 64, 128, 256 that holds head_dim.  Scores: keep S for the weights.
template <typename T, int D, bool Scores>
__global__ void __launch_bounds__(kWaves * 64, D <= 128 ? 2 : 1) paged_kernel(const PagedParams p) {
  using vec8 = typename Traits<T>::vec8;
  constexpr int KS = Pad<D>::kPlain, VS = Pad<D>::kTr;
  constexpr int CPR = D / 8;         // 16-byte chunks per row
  constexpr int RPP = 64 / CPR;      // rows per pass of a wave
  constexpr int NPV = kUnit / RPP;   // passes per unit
  constexpr int kWaveLds = kUnit * (KS + VS) * (int)sizeof(T);  // a wave's K and V tile, reused for the join
  constexpr int OS = D + 4;  // row stride of a wave's O when the waves join
  static_assert(kWaveLds >= 32 * OS * 4, "a wave's O must fit its tiles");
  __shared__ __attribute__((aligned(16))) unsigned char lds[kWaves][kWaveLds];
  __shared__ float m_s[kWaves][32], l_s[kWaves][32];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // a scalar: units, masks and branches on them are the wave's
  const int r32 = lane & 31, g = lane >> 5;
  const int split = blockIdx.x % p.n_splits;
  const int tile = p.tile0 + blockIdx.x / p.n_splits;
  const int ct = tile % p.n_ct, bhk = tile / p.n_ct;
  const int bi = bhk / p.h_k, hk = bhk % p.h_k;
  const int group = p.h / p.h_k, n_cols = group * p.sq;
  // column n = ct * 32 + r32 of the S^T tile: query head hk*group + n / sq, query row n % sq.  Its
  // fragments are requested before anything that waits for the sequence's length.
  const int n = ct * 32 + r32;
  const bool col_ok = n < n_cols;
  const int qi = col_ok ? n % p.sq : 0, hq = hk * group + (col_ok ? n / p.sq : 0);
  vec8 qf[D / 16];
  {
    const T *qg = static_cast<const T *>(p.q) + bi * p.q_bs + (int64_t)qi * p.q_rs + hq * p.q_hs;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
      qf[ks] = (col_ok && ks * 16 + g * 8 < p.d) ? *reinterpret_cast<const vec8 *>(qg + ks * 16 + g * 8) : vec8{0};
  }
  const int sk = p.keys_of(bi);

  const idx::SinkTiles st = p.units(sk, ct);
  const int n_units = min(st.n, p.max_units), per = p.per_split(n_units);
  const int u0 = split * per, u1 = min(n_units, u0 + per);
  if (split > 0 && u0 >= n_units) return;  // whole workgroups

  int lo_lim = 0, hi_lim = 0;
  if (col_ok) idx::row_limits(p.sq, sk, p.wl, p.wr, qi, lo_lim, hi_lim);
  // what every column of the tile sees: [all_lo, all_hi) and, below it, the sinks
  int all_lo, all_hi, t0, t1;
  idx::row_limits(p.sq, sk, p.wl, p.wr, p.sq - 1, all_lo, t0);
  idx::row_limits(p.sq, sk, p.wl, p.wr, 0, t1, all_hi);

  const T *kg = static_cast<const T *>(p.k) + hk * p.pages.k_hs;
  const T *vg = static_cast<const T *>(p.v) + hk * p.pages.v_hs;
  T *Kt = reinterpret_cast<T *>(lds[wave]), *Vt = Kt + kUnit * KS;
  const int v_c = lane % CPR, v_r = lane / CPR;
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  // rows from new0 on come from k_new / v_new instead of the cache and are written to it
  // (only where every new row is certain to be visited: p.fuse_append)
  const int new0 = p.fuse_append ? p.seqlens[bi] : 0x7fffffff;
  const T *kng = p.fuse_append ? static_cast<const T *>(p.k_new) + bi * p.kn_bs + hk * p.kn_hs : nullptr;
  const T *vng = p.fuse_append ? static_cast<const T *>(p.v_new) + bi * p.vn_bs + hk * p.vn_hs : nullptr;
  // Where row l % 32 of a unit lies, in lane l: its page number and its row there (-1: nobody sees
  // the row); requested a unit ahead of the loads that need it.  The request is unconditional
  // (some entry of the table, or any word when there is none) and its result is not looked at
  // here: a test, or a choice between it and something else, would wait for it and with it for
  // every load in flight.
  const int *table = p.pages.max_pages ? p.pages.table + (int64_t)bi * p.pages.max_pages : static_cast<const int *>(p.q);
  struct Place { int number, row; };
  auto locate = [&](int j) {
    const int key = idx::sink_tile(st, j) * kUnit + r32;
    const bool seen = key < st.hi && (key >= st.lo || key < st.sink);
    int at = 0, row = key;
    if (p.pages.max_pages) at = p.pages.index(seen ? key : 0, row);
    return Place{table[at], seen ? row : -1};
  };
  auto from_lane = [&](int64_t v, int src) {  // lane src's value
    const int lo = __builtin_amdgcn_ds_bpermute(src * 4, (int)v), hi = __builtin_amdgcn_ds_bpermute(src * 4, (int)(v >> 32));
    return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
  };
  // The rows of one pass lie on one page when the page size is a multiple of their number (or the
  // cache is dense): their
  // address is then a scalar plus an offset that every pass shares, which costs the vector ALU
  // and the registers nothing.
  const bool scalar_rows = (p.pages.max_pages == 0 || p.pages.page % RPP == 0) && (uint64_t)p.pages.k_rs < (1 << 26) && (uint64_t)p.pages.v_rs < (1 << 26);
  const bool col_in = v_c * 8 < p.d;            // columns from head_dim up to D are zeros in the tiles
  const int v_col = col_in ? v_c * 8 : 0;       // their lanes load a column that exists and store nothing
  const uint32_t k_in = (uint32_t)(v_r * (uint32_t)p.pages.k_rs + v_col), v_in = (uint32_t)(v_r * (uint32_t)p.pages.v_rs + v_col);
  // Unit j, located, into the staging registers, when all its 32 rows are to be read from the
  // cache.  A unit with rows that are not (the ends of a sequence or
  // window, absent pages, new rows) is read by store_unit instead: keeping it in flight as well would
  // cost the registers that the LDS reads of the loop need to run ahead of the MFMAs.
  struct Stage {
    uint4 k[NPV], v[NPV];
    int pg = 0, row = -1;
    uint32_t there = 0;   // which of the unit's rows exist
    bool staged = false;
  };
  auto load_unit = [&](int j, const Place &at, Stage &u) {
    const int pg_next = p.pages.max_pages ? at.number : bi, row_next = at.row;
    u.there = (uint32_t)__builtin_amdgcn_ballot_w64(row_next >= 0 && p.pages.present(pg_next));
    u.pg = pg_next;
    u.row = row_next;
    int vr = v_r;
    FA_PIN(vr);  // what the uncommon paths derive from it is computed there, not kept in registers over the loop
    u.staged = u.there == 0xffffffffu && idx::sink_tile(st, j) * kUnit + kUnit <= new0;
    if (u.staged && scalar_rows) {
#pragma unroll
      for (int s = 0; s < NPV; ++s) {
        const int64_t pg = FA_READLANE(pg_next, s * RPP), row = FA_READLANE(row_next, s * RPP);
        const u32x4 a = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kg + pg * p.pages.k_ps + row * p.pages.k_rs + k_in));
        const u32x4 b = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(vg + pg * p.pages.v_ps + row * p.pages.v_rs + v_in));
        u.k[s] = uint4{a.x, a.y, a.z, a.w};
        u.v[s] = uint4{b.x, b.y, b.z, b.w};
      }
    } else if (u.staged) {
      const int64_t k_lane = pg_next * p.pages.k_ps + row_next * p.pages.k_rs, v_lane = pg_next * p.pages.v_ps + row_next * p.pages.v_rs;
#pragma unroll
      for (int s = 0; s < NPV; ++s) {
        const int64_t ko = from_lane(k_lane, s * RPP + vr), vo = from_lane(v_lane, s * RPP + vr);
        const u32x4 a = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kg + ko + v_col));
        const u32x4 b = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(vg + vo + v_col));
        u.k[s] = uint4{a.x, a.y, a.z, a.w};
        u.v[s] = uint4{b.x, b.y, b.z, b.w};
      }
    }
  };
  auto store_unit = [&](int j, Stage &u) {  // unit j into the wave's tiles
    if (!u.staged) {
      const int kv0 = idx::sink_tile(st, j) * kUnit;
      int vr = v_r;
      FA_PIN(vr);
      const int64_t k_lane = u.pg * p.pages.k_ps + u.row * p.pages.k_rs, v_lane = u.pg * p.pages.v_ps + u.row * p.pages.v_rs;
#pragma unroll
      for (int s = 0; s < NPV; ++s) {
        const int r = s * RPP + vr, key = kv0 + r;
        const int64_t ko = from_lane(k_lane, r), vo = from_lane(v_lane, r);
        const bool fresh = key >= new0;
        u.k[s] = uint4{0, 0, 0, 0};  // a row that nobody sees: 0 * finite stays finite in P V
        u.v[s] = uint4{0, 0, 0, 0};
        if (((u.there >> r) & 1u) & col_in) {
          u.k[s] = *reinterpret_cast<const uint4 *>((fresh ? kng + (int64_t)(key - new0) * p.kn_rs : kg + ko) + v_col);
          u.v[s] = *reinterpret_cast<const uint4 *>((fresh ? vng + (int64_t)(key - new0) * p.vn_rs : vg + vo) + v_col);
        }
      }
      if (kv0 + kUnit > new0) {
#pragma unroll
        for (int s = 0; s < NPV; ++s) {
          const int r = s * RPP + vr;
          const int64_t ko = from_lane(k_lane, r), vo = from_lane(v_lane, r);
          if (((u.there >> r) & 1u) && col_in && kv0 + r >= new0) {
            *reinterpret_cast<uint4 *>(const_cast<T *>(kg) + ko + v_col) = u.k[s];
            *reinterpret_cast<uint4 *>(const_cast<T *>(vg) + vo + v_col) = u.v[s];
          }
        }
      }
    }
    if (col_in) {
#pragma unroll
      for (int s = 0; s < NPV; ++s) {
        *reinterpret_cast<uint4 *>(&Kt[(s * RPP + v_r) * KS + v_c * 8]) = u.k[s];
        *reinterpret_cast<uint4 *>(&Vt[(s * RPP + v_r) * VS + v_c * 8]) = u.v[s];
      }
    }
    FA_WAVE_SYNC();  // the wave's own tile: written by all its lanes, read across lanes, no workgroup barrier
  };
  if (p.d != D && !col_in) {
#pragma unroll
    for (int s = 0; s < NPV; ++s) {
      *reinterpret_cast<uint4 *>(&Kt[(s * RPP + v_r) * KS + v_c * 8]) = uint4{0, 0, 0, 0};
      *reinterpret_cast<uint4 *>(&Vt[(s * RPP + v_r) * VS + v_c * 8]) = uint4{0, 0, 0, 0};
    }
  }

  float16v o_acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) o_acc[i] = float16v{0};
  // the reference maximum is raised only when it would grow by more than kSlack (in log2 units), as
  // in flash_fwd.hip: P stays below 2^kSlack and O is rescaled a few times instead of per unit
  constexpr float kSlack = 8.f;
  float m_run = -INFINITY, m_scaled = 0.f, l_run = 0.f;
  const float c = p.scale_log2;

  // One unit in flight beside the one in LDS.  (Two, where the registers allow it: no faster; 16 heads,
  // D = 64, 64 x 8192 keys 376 against 380 us.)
  Stage stage;
  Place next{0, -1};
  const int first = u0 + wave;
  uint32_t there = 0;
  if (first < u1) {
    const Place p0 = locate(first);
    next = locate(min(first + kWaves, u1 - 1));
    load_unit(first, p0, stage);
    store_unit(first, stage);
    there = stage.there;
  }
  // The Q fragments are consumed here: the wait for their loads would otherwise stand before the first
  // MFMA of every unit and drain the loads of the next one too.
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) FA_PIN(qf[ks]);
  for (int j = first; j < u1; j += kWaves) {
    // the table before the rows: loads return in order, and waiting for the number must not mean
    // waiting for the rows requested after it
    const Place after = locate(min(j + 2 * kWaves, u1 - 1));
    if (j + kWaves < u1) load_unit(j + kWaves, next, stage);
    next = after;
    float16v s = float16v{0};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
      s = Traits<T>::mfma(lds_read8<T>(&Kt[r32 * KS + ks * 16 + g * 8]), qf[ks], s);
    const int kv0 = idx::sink_tile(st, j) * kUnit;
    if (there != 0xffffffffu || kv0 + kUnit > all_hi || (kv0 < all_lo && kv0 + kUnit > p.n_sink)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = (i >> 2) * 8 + g * 4 + (i & 3), kv = kv0 + r;
        const bool hidden = (kv >= hi_lim) | ((kv < lo_lim) & (kv >= p.n_sink)) | !((there >> r) & 1u);
        s[i] = hidden ? -INFINITY : s[i];
      }
    }
    if constexpr (Scores) {
      if (col_ok) {
        float *sp = p.s_part + (((int64_t)bhk * n_cols + n - p.row0) * p.max_units + j) * kUnit + g * 4;
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
          *reinterpret_cast<float4 *>(sp + i4 * 8) = float4{s[i4 * 4], s[i4 * 4 + 1], s[i4 * 4 + 2], s[i4 * 4 + 3]};
      }
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    // +inf for the first finite score of a column, NaN (false) for -inf - -inf
    if (__builtin_amdgcn_ballot_w64((mx - m_run) * c > kSlack) != 0) {
      mx = fmaxf(mx, partner32(mx));
      const float m_new = (mx - m_run) * c > kSlack ? mx : m_run;
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2_fast((m_run - m_use) * c);
      l_run *= alpha;
      m_run = m_new;
      m_scaled = m_use * c;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o_acc[db][i] *= alpha;
    }
    float rs = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e = exp2_fast(fmaf(s[i], c, -m_scaled));
      s[i] = e;
      rs += e;
    }
    l_run += rs;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float pf[8];
#pragma unroll
      for (int jj = 0; jj < 8; ++jj) pf[jj] = s[w * 8 + jj];
      const vec8 pb = pack8<T>(pf);  // P in the storage type: half a step of each term, as in the other kernels
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
        o_acc[db] = Traits<T>::mfma(lds_read_operand_tr<T>(Vt, VS, w * 16, db * 32), pb, o_acc[db]);
    }
    if (j + kWaves < u1) {
      store_unit(j + kWaves, stage);  // after every read of unit j in program order
      there = stage.there;
    }
  }

  // ---- the four waves' partials joined through LDS (each wave writes into its own region) ----
  const float l_wave = l_run + partner32(l_run);
  float *Ow = reinterpret_cast<float *>(lds[wave]);  // [32 columns][OS]
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4)
      *reinterpret_cast<float4 *>(&Ow[r32 * OS + db * 32 + i4 * 8 + g * 4]) =
          float4{o_acc[db][i4 * 4], o_acc[db][i4 * 4 + 1], o_acc[db][i4 * 4 + 2], o_acc[db][i4 * 4 + 3]};
  if (g == 0) { m_s[wave][r32] = m_run; l_s[wave][r32] = l_wave; }
  __syncthreads();

  const int on = tid & 31, slice = tid >> 5;  // eight slices of D / 8 output elements per column
  float mw[kWaves], wgt[kWaves], m_all = -INFINITY, l_all = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    mw[w] = m_s[w][on];
    m_all = fmaxf(m_all, mw[w]);
  }
  const float m_ref = m_all == -INFINITY ? 0.f : m_all;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    wgt[w] = exp2_fast((mw[w] - m_ref) * c);  // 0 for a wave that saw no key
    l_all += wgt[w] * l_s[w][on];
  }
  const int cn = ct * 32 + on;
  if (cn >= n_cols) return;
  const int oi = cn % p.sq, oh = hk * group + cn / p.sq;
  const bool final_pass = p.o_part == nullptr;
  const bool empty = l_all == 0.f;
  const float inv = final_pass ? (empty ? 1.f : 1.f / l_all) : 1.f;
  T *og = static_cast<T *>(p.o) + bi * p.o_bs + (int64_t)oi * p.o_rs + oh * p.o_hs;
  const int64_t prow = split * p.n_rows + ((int64_t)bi * p.h + oh) * p.sq + oi - p.row0;
#pragma unroll
  for (int x = 0; x < D / 8; x += 4) {
    const int dcol = slice * (D / 8) + x;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float4 t = *reinterpret_cast<const float4 *>(&reinterpret_cast<const float *>(lds[w])[on * OS + dcol]);
      acc[0] += wgt[w] * t.x; acc[1] += wgt[w] * t.y; acc[2] += wgt[w] * t.z; acc[3] += wgt[w] * t.w;
    }
    typedef T vec4 __attribute__((ext_vector_type(4)));
    if (!final_pass) *reinterpret_cast<float4 *>(p.o_part + prow * D + dcol) = float4{acc[0], acc[1], acc[2], acc[3]};
    else if (dcol < p.d) *reinterpret_cast<vec4 *>(og + dcol) = vec4{(T)(acc[0] * inv), (T)(acc[1] * inv), (T)(acc[2] * inv), (T)(acc[3] * inv)};
  }
  if (slice == 0) {
    if (final_pass) p.lse[((int64_t)bi * p.h + oh) * p.sq + oi] = empty ? INFINITY : m_all * p.scale + log2_fast(l_all) * kLn2;
    else { p.ml_part[prow * 2] = m_all; p.ml_part[prow * 2 + 1] = l_all; }
  }
}

// Joins the splits' partials: D / 4 threads take a row's columns, four each, and `groups` such sets of
// threads share out the row's splits when rows are few and splits many (their sums meet in LDS);
// else every set has a row of its own.  live: the number of splits that have written partials, or 0
// for a paged call, where it follows from the row's sequence.
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(const PagedParams p, int groups, int live) {
  constexpr int TPR = D / 4, SETS = 256 / TPR;
  __shared__ float4 acc_s[256];
  __shared__ float l_s[SETS];
  const int tid = threadIdx.x, set = tid / TPR, col = tid % TPR * 4;
  const int64_t rows = p.n_rows;
  const int64_t row = (int64_t)blockIdx.x * (SETS / groups) + set / groups, at = row < rows ? row : rows - 1;  // of the launch's
  const int64_t r = p.row0 + at;  // (sequence * h + head) * sq + query row
  const int share = set % groups;
  const int qi = (int)(r % p.sq), hq = (int)(r / p.sq % p.h), bi = (int)(r / p.sq / p.h);
  int n_live = live;
  if (live == 0) {
    const int n_units = min(p.units(p.keys_of(bi), (hq % (p.h / p.h_k) * p.sq + qi) / 32).n, p.max_units), per = p.per_split(n_units);
    n_live = max(1, (n_units + per - 1) / per);
  }
  const float2 *ml = reinterpret_cast<const float2 *>(p.ml_part) + at;
  const float *op = p.o_part + at * D + col;
  float m_all = -INFINITY;
#pragma unroll 8
  for (int s = 0; s < n_live; ++s) m_all = fmaxf(m_all, ml[s * rows].x);
  const float m_ref = m_all == -INFINITY ? 0.f : m_all;
  float l = 0.f;
  float4 t = float4{0, 0, 0, 0};
#pragma unroll 4
  for (int s = share; s < n_live; s += groups) {
    const float2 x = ml[s * rows];
    const float w = exp2_fast((x.x - m_ref) * p.scale_log2);  // 0 for a split that saw no key
    const float4 o = *reinterpret_cast<const float4 *>(op + s * rows * D);
    l += w * x.y;
    t.x += w * o.x; t.y += w * o.y; t.z += w * o.z; t.w += w * o.w;
  }
  if (groups > 1) {
    acc_s[tid] = t;
    if (tid % TPR == 0) l_s[set] = l;
    __syncthreads();
    if (share > 0) return;
    for (int x = 1; x < groups; ++x) {
      const float4 o = acc_s[tid + x * TPR];
      l += l_s[set + x];
      t.x += o.x; t.y += o.y; t.z += o.z; t.w += o.w;
    }
  }
  if (row >= rows) return;
  const bool empty = l == 0.f;
  const float inv = empty ? 0.f : 1.f / l;
  typedef T vec4 __attribute__((ext_vector_type(4)));
  if (col < p.d)
    *reinterpret_cast<vec4 *>(static_cast<T *>(p.o) + bi * p.o_bs + (int64_t)qi * p.o_rs + hq * p.o_hs + col) =
        vec4{(T)(t.x * inv), (T)(t.y * inv), (T)(t.z * inv), (T)(t.w * inv)};
  if (col == 0) p.lse[r] = empty ? INFINITY : m_all * p.scale + log2_fast(l) * kLn2;
}

template <typename T, int D>
hipError_t join_td(const PagedParams &p, int live, hipStream_t stream) {
  constexpr int SETS = 256 / (D / 4);
  const int64_t rows = p.n_rows;
  int groups = 1;  // more as long as every CU has a workgroup's rows less than once
  while (groups < SETS && groups < p.n_splits && rows * groups < 256 * SETS) groups *= 2;
  const int per = SETS / groups;
  FA_LAUNCH((join_kernel<T, D>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), stream, p, groups, live);
  return hipGetLastError();
}

// weights_out[key] = weights_in[key] (0 for a row appended by this call) + sum of P over the columns of
// the key/value head, in column order; a thread per 4 keys (of one unit), keys behind the last one
// are left alone.  A launch of some of a key/value head's tiles goes on from the sums of those before it.
__global__ void __launch_bounds__(256) paged_weights_kernel(const PagedParams p, int bhk0) {
  const int cap = p.pages.capacity(), blocks = (cap + 1023) / 1024;
  const int bhk = bhk0 + blockIdx.x / blocks, bi = bhk / p.h_k, hk = bhk % p.h_k;
  const int key = (blockIdx.x % blocks * 256 + threadIdx.x) * 4, sk = p.keys_of(bi);
  if (key >= sk) return;
  const int group = p.h / p.h_k, n_cols = group * p.sq, tile = key / kUnit, old = p.seqlens[bi];
  const int64_t at = (int64_t)bhk * cap + key;
  const int n = min(4, sk - key);
  const int ct0 = max(0, p.tile0 - bhk * p.n_ct), ct1 = min(p.n_ct, p.tile0 + p.n_tiles - bhk * p.n_ct);
  const float *w_in = ct0 > 0 ? p.w_out : p.w_in;
  const int n_in = ct0 > 0 ? sk : w_in ? old : 0;  // rows whose weight does not start from zero
  float w[4];
#pragma unroll
  for (int y = 0; y < 4; ++y) w[y] = y < n && key + y < n_in ? w_in[at + y] : 0.f;
  const float *lse = p.lse + ((int64_t)bi * p.h + hk * group) * p.sq;  // column n's at n
  for (int ct = ct0; ct < ct1; ++ct) {
    const idx::SinkTiles st = p.units(sk, ct);
    const int j = tile < st.ns ? tile : tile - st.n0 + st.ns;  // the unit that holds the keys
    if ((tile >= st.ns && tile < st.n0) || j >= min(st.n, p.max_units)) continue;
    const int c1 = min(n_cols, (ct + 1) * 32);
    const float *sp = p.s_part + (((int64_t)bhk * n_cols - p.row0) * p.max_units + j) * kUnit + key % kUnit;
#pragma unroll 4
    for (int c = ct * 32; c < c1; ++c) {
      const float4 s = *reinterpret_cast<const float4 *>(sp + (int64_t)c * p.max_units * kUnit);
      const float l = -lse[c] * kLog2e;
      // -inf: a key that the column does not see, also where the column sees none (lse = +inf)
      w[0] += s.x == -INFINITY ? 0.f : exp2_fast(fmaf(s.x, p.scale_log2, l));
      w[1] += s.y == -INFINITY ? 0.f : exp2_fast(fmaf(s.y, p.scale_log2, l));
      w[2] += s.z == -INFINITY ? 0.f : exp2_fast(fmaf(s.z, p.scale_log2, l));
      w[3] += s.w == -INFINITY ? 0.f : exp2_fast(fmaf(s.w, p.scale_log2, l));
    }
  }
#pragma unroll
  for (int y = 0; y < 4; ++y)
    if (y < n) p.w_out[at + y] = w[y];
}

// the weights of key/value heads (sequence * h_k + head) bhk0 .. bhk1 - 1
hipError_t launch_weights(const PagedParams &p, int bhk0, int bhk1, hipStream_t stream) {
  FA_LAUNCH((paged_weights_kernel), dim3((unsigned)((int64_t)((p.pages.capacity() + 1023) / 1024) * (bhk1 - bhk0))), dim3(256), stream, p, bhk0);
  return hipGetLastError();
}

// the new rows into the cache, 16 bytes a thread; rows behind the capacity or on an absent page are dropped
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedParams p) {
  const int cpr = p.d / 8;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= (int64_t)p.b * p.n_new * p.h_k * cpr) return;
  const int c = (int)(e % cpr), hk = (int)(e / cpr % p.h_k);
  const int i = (int)(e / cpr / p.h_k % p.n_new), bi = (int)(e / cpr / p.h_k / p.n_new);
  const int old = p.seqlens[bi];
  if (old < 0 || (int64_t)old + i >= p.pages.capacity()) return;
  int row;
  const int pg = p.pages.locate(bi, old + i, row);
  if (pg < 0) return;
  typedef unsigned short u16;  // either storage type
  const u16 *ks = static_cast<const u16 *>(p.k_new) + bi * p.kn_bs + (int64_t)i * p.kn_rs + hk * p.kn_hs + c * 8;
  const u16 *vs = static_cast<const u16 *>(p.v_new) + bi * p.vn_bs + (int64_t)i * p.vn_rs + hk * p.vn_hs + c * 8;
  u16 *kd = static_cast<u16 *>(const_cast<void *>(p.k)) + (int64_t)pg * p.pages.k_ps + (int64_t)row * p.pages.k_rs + hk * p.pages.k_hs + c * 8;
  u16 *vd = static_cast<u16 *>(const_cast<void *>(p.v)) + (int64_t)pg * p.pages.v_ps + (int64_t)row * p.pages.v_rs + hk * p.pages.v_hs + c * 8;
  *reinterpret_cast<uint4 *>(kd) = *reinterpret_cast<const uint4 *>(ks);
  *reinterpret_cast<uint4 *>(vd) = *reinterpret_cast<const uint4 *>(vs);
}

// Scratch for the scores of one launch at most (one column tile's at least): a call that would take more is
// computed in several launches, one after the other in the same scratch.  Its size follows from the
// cache's capacity, which the host knows, and not from the lengths, which it does not.
// Measured where it takes four launches in place of one with 1 GiB, 32 heads on 8, D = 128: 64
// sequences in a cache of 131072 rows, one row each, 300 / 4096 / 32768 keys: 512 / 1626 / 2174 us against
// 480 / 1708 / 2209; 8 sequences of 32768 keys, 32 rows each: 1028 against 1168.
constexpr int64_t kScoreBytes = int64_t(256) << 20;

int tile_rows(const PagedParams &p) { return std::min(32, p.h / p.h_k * p.sq); }  // most rows of a column tile

template <typename T, int D>
hipError_t paged_td(PagedParams &p, hipStream_t stream) {
  const int n_cols = p.h / p.h_k * p.sq;
  const int64_t rows = (int64_t)p.b * p.h * p.sq, tiles = (int64_t)p.b * p.h_k * p.n_ct;
  int64_t part = p.n_tiles;  // tiles of a launch
  size_t s_bytes = 0, need = 0;
  auto plan = [&]() {
    const size_t n = (size_t)std::min(rows, part * tile_rows(p));
    s_bytes = p.w_out ? n * p.max_units * kUnit * sizeof(float) : 0;
    need = s_bytes + (p.n_splits > 1 ? p.n_splits * n * (D + 2) * sizeof(float) : 0);
  };
  plan();
  if (p.ws_query) { *p.ws_query = need; return hipSuccess; }
  const size_t given = p.ws && (reinterpret_cast<uintptr_t>(p.ws) & 15) == 0 ? p.ws_bytes : 0;
  void *ws = nullptr;
  bool owned = false;
  while (need) {
    if (given >= need) { ws = p.ws; break; }
    const hipError_t e = hipMallocAsync(&ws, need, stream);
    if (e == hipSuccess) { owned = true; break; }
    // no memory: one split, then ever fewer tiles a launch, in the caller's scratch if that holds them
    (void)hipGetLastError();
    ws = nullptr;
    if (p.n_splits > 1) p.n_splits = 1;
    else if (part > 1) part = (part + 1) / 2;
    else return e;  // the scores of one tile have nowhere to go
    plan();
  }
  hipError_t e = hipSuccess;
  if (p.n_new > 0 && !p.fuse_append) {
    const int64_t n = (int64_t)p.b * p.n_new * p.h_k * (p.d / 8);
    FA_LAUNCH((paged_append_kernel), dim3((unsigned)((n + 255) / 256)), dim3(256), stream, p);
    e = hipGetLastError();
  }
  auto first_row = [&](int64_t tile) { return tile / p.n_ct * n_cols + tile % p.n_ct * 32; };
  for (int64_t t0 = 0; t0 < tiles && e == hipSuccess; t0 += part) {
    const int64_t t1 = std::min(tiles, t0 + part);
    p.tile0 = (int)t0;
    p.n_tiles = (int)(t1 - t0);
    p.row0 = first_row(t0);
    p.n_rows = first_row(t1) - p.row0;
    p.s_part = s_bytes ? static_cast<float *>(ws) : nullptr;
    if (p.n_splits > 1) {
      p.o_part = static_cast<float *>(ws) + s_bytes / sizeof(float);
      p.ml_part = p.o_part + p.n_splits * p.n_rows * D;
    }
    const dim3 grid((unsigned)(p.n_tiles * p.n_splits));
    if (p.w_out) FA_LAUNCH((paged_kernel<T, D, true>), grid, dim3(kWaves * 64), stream, p);
    else FA_LAUNCH((paged_kernel<T, D, false>), grid, dim3(kWaves * 64), stream, p);
    e = hipGetLastError();
    if (e == hipSuccess && p.n_splits > 1) e = join_td<T, D>(p, 0, stream);
    if (e == hipSuccess && p.w_out) e = launch_weights(p, (int)(t0 / p.n_ct), (int)((t1 + p.n_ct - 1) / p.n_ct), stream);
  }
  if (owned) {
    const hipError_t f = hipFreeAsync(ws, stream);
    if (e == hipSuccess) e = f;
  }
  return e;
}

template <typename T>
hipError_t paged_t(PagedParams &p, hipStream_t stream) {
  if (p.d <= 32) return paged_td<T, 32>(p, stream);
  if (p.d <= 64) return paged_td<T, 64>(p, stream);
  if (p.d <= 128) return paged_td<T, 128>(p, stream);
  return paged_td<T, 256>(p, stream);
}

}  // namespace

hipError_t launch_paged(PagedParams &p, int dtype, hipStream_t stream) {
  const int cap = p.pages.capacity();
  p.n_ct = (p.h / p.h_k * p.sq + 31) / 32;
  if (p.sq == 0) return launch_weights(p, 0, p.b * p.h_k, stream);  // no columns: weights_out = weights, or zero
  // most units a tile visits: the sinks' and those of a window over its rows, or the whole cache
  int64_t units = (cap + kUnit - 1) / kUnit;
  if (p.wl >= 0)
    units = std::min<int64_t>(units, (std::min(p.n_sink, cap) + kUnit - 1) / kUnit + ((int64_t)p.wl + p.sq + kUnit) / kUnit + 2);
  p.max_units = (int)std::max<int64_t>(units, 1);
  const int64_t tiles = (int64_t)p.b * p.h_k * p.n_ct;
  int64_t base = tiles;  // tiles of a launch
  if (p.w_out) {
    const int64_t most = std::max<int64_t>(1, kScoreBytes / ((int64_t)tile_rows(p) * p.max_units * kUnit * (int)sizeof(float)));
    const int64_t launches = (tiles + most - 1) / most;
    base = (tiles + launches - 1) / launches;
  }
  p.n_tiles = (int)base;
  // Splits: one round of workgroups (two for every CU) when the sequences are few, of 128 keys (a unit
  // a wave) at least; 2048 keys each when they are many, so that unequal lengths even out.  Units
  // per split 16 / 32 / 64 / 128, kernel time: 64 x 8192 keys, 8 heads, D = 128: 368 / 351 / 346 /
  // 340 us, 1000..8191 keys: 231 / 212 / 211 / 238 with the join; 8 x 8192: 55 / 52 / 56 / 87.
  p.min_units = (int)std::min<int64_t>(64, std::max<int64_t>(kWaves, (p.max_units * base + 511) / 512));
  // up to three units a wave are read before a second launch would have joined two workgroups
  p.n_splits = p.max_units <= 3 * kWaves ? 1 : (int)std::min<int64_t>(64, (p.max_units + p.min_units - 1) / p.min_units);
  // the threads of a launch are counted in 32 bits
  if (base * p.n_splits > (1 << 23) || (int64_t)p.b * p.h * p.sq > (1 << 24)) p.n_splits = 1;
  // the attention kernel appends when one workgroup's tile covers all columns and its window reaches the first new row
  p.fuse_append = p.n_new > 0 && p.n_ct == 1 && (p.wl < 0 || p.n_new <= (int64_t)p.sq + p.wl);
  return dtype == 1 ? paged_t<_Float16>(p, stream) : paged_t<__bf16>(p, stream);
}

// A few rows per key/value head (two column tiles) against the dense keys of a flash_attn_sink_fwd
// call: streaming the keys beats a block of 128 or 256 rows that is mostly empty.
bool sink_few_rows(const Params &p) { return (int64_t)(p.h / p.h_k) * p.sq <= 64 && p.sk >= 1; }

hipError_t launch_sink_join(const Params &p, int width, int dtype, hipStream_t stream) {
  PagedParams a{};
  a.o = p.o_w; a.lse = p.lse;
  a.o_bs = p.o_bs; a.o_rs = p.o_rs; a.o_hs = p.o_hs;
  a.b = p.b; a.h = p.h; a.h_k = p.h_k; a.d = p.d; a.sq = p.sq;
  a.scale = p.scale; a.scale_log2 = p.scale_log2;
  a.n_splits = p.n_splits;
  a.n_rows = (int64_t)p.b * p.h * p.sq;
  a.o_part = p.o_part; a.ml_part = p.ml_part;
  auto go = [&](auto t) {
    using T = decltype(t);
    return width == 32 ? join_td<T, 32>(a, p.n_splits, stream) : width == 64 ? join_td<T, 64>(a, p.n_splits, stream)
         : width == 128 ? join_td<T, 128>(a, p.n_splits, stream) : join_td<T, 256>(a, p.n_splits, stream);
  };
  return dtype == 1 ? go((_Float16)0) : go((__bf16)0);
}

hipError_t launch_sink_few_rows(const Params &p, int dtype, hipStream_t stream) {
  PagedParams a{};
  a.q = p.q; a.k = p.k; a.v = p.v; a.o = p.o_w; a.lse = p.lse;
  set_page(a.pages, p.sk);
  a.pages.num_pages = p.b;
  a.pages.k_ps = p.k_bs; a.pages.k_rs = p.k_rs; a.pages.k_hs = p.k_hs;
  a.pages.v_ps = p.v_bs; a.pages.v_rs = p.v_rs; a.pages.v_hs = p.v_hs;
  a.q_bs = p.q_bs; a.q_rs = p.q_rs; a.q_hs = p.q_hs;
  a.o_bs = p.o_bs; a.o_rs = p.o_rs; a.o_hs = p.o_hs;
  a.b = p.b; a.h = p.h; a.h_k = p.h_k; a.d = p.d; a.sq = p.sq;
  a.scale = p.scale; a.scale_log2 = p.scale_log2;
  a.wl = p.wl; a.wr = p.wr; a.n_sink = p.n_sink;
  a.ws = p.ws; a.ws_bytes = p.ws_bytes; a.ws_query = p.ws_query;
  return launch_paged(a, dtype, stream);
}

}  // namespace fa
