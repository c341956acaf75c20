// A chunk of new tokens of every sequence of a batch against its pages on CDNA4 (gfx950): what lucid_paged.hip does
// for a few tokens, for as many as a prompt has (modeling_lucid.py:475-496, 576-598 is the cached path of the
// reference; pages, tables and lengths as in lucid_paged.hip).  Sequence b has n rows cached and brings c
// tokens of the batch's L (right-padded).  For its tokens t = n .. n + c - 1:
//   P_tj = exp(s r_t r_j (k_t . k_j) - 1/s),  r = 1 / rms(k)  (j < t, cached or new)
//   v'_t = (v_t - sum_{j<t} P_tj w_j) / P_tt,  P_tt = exp(s d ms_t / (ms_t + eps) - 1/s)
//   o_tg = softmax_j(s q_tg . k_j) w_j over j <= t
// with w_j the V' row as the cache holds it (bf16), new rows too: any cutting of a prompt into chunks, down to
// single tokens, gives the same rows.  The steps, each a launch:
//   lucid_prefill_prep_kernel   the batch read and checked; new keys into their pages; for each panel of 256 new
//                               rows the panel's own P in the form that the solve reads
//   lucid_prefill_sweep_kernel  (couple) y_t = v_t - sum over the cached rows of P_tj w_j
//   lucid_prefill_solve_kernel  one panel's rows solved in order and written into their pages; between two panels
//                               the sweep takes the solved one out of the later rows' y
//   lucid_prefill_sweep_kernel  (attend) the softmax over all rows, cached and new
//   lucid_prefill_join_kernel   parts of a sweep that was cut along the keys
// The sweeps are the work: 4 (Hq + Hkv) d flops for each pair of a token and a row.  2048 tokens of 32/8 heads of 128 columns
// behind 32768 rows (1.42 TFLOP, 185 MB) take 1.71 ms a call.  Its kernels traced one by one sum to 1.85 on the same card: 1.17 of
// attending, 0.42 of coupling, 0.23 in the eight solves and the seven inner sweeps between them, which are one chain, and
// 0.03 of prep and joins.
#include <type_traits>

#include "paged_common.h"

namespace lucid {

constexpr int kPanel = 256;      // new rows that one solve takes
constexpr int kPanelBlocks = 8;  // of 32 rows
constexpr int kSweepKeys = 128;  // keys of a staged tile
// A panel's own -P_tj / P_tt: 28 tiles below the diagonal blocks as operands (hi and lo bf16), 8 diagonal blocks
// transposed in fp32, and 1 / P_tt of its rows
constexpr int kPanelTile = 4 * 512;                                          // bf16 of an operand tile
constexpr size_t kPanelDiag = (size_t)28 * kPanelTile * 2;                   // byte offset of the diagonal blocks
constexpr size_t kPanelInv = kPanelDiag + (size_t)kPanelBlocks * 1024 * 4;   // of the inverses
constexpr size_t kPanelBytes = kPanelInv + kPanel * 4;
constexpr float PREFILL_NEG = -1e30f;  // finite "minus infinity" for empty softmax states

struct PrefillBatch {
  const int32_t* table;  // [B][M] page ids, rows tstride apart
  int64_t tstride;
  const int32_t* lens;    // [B] rows cached
  const int32_t* counts;  // [B] tokens of each sequence, null: L
  int B, M, P, page;
  int shift;  // log2 of page, -1 where it is no power of two
  int L, Hkv;
  int2* info;  // [B] rows cached and tokens (0: nothing to do), left by the prep kernel
};
__device__ __forceinline__ int prefill_page(const PrefillBatch& s, int j) { return s.shift >= 0 ? j >> s.shift : j / s.page; }
// Offset of row j of a sequence with the page ids tbl in a pool, its head's rows
__device__ __forceinline__ unsigned prefill_row(const PrefillBatch& s, const PagedPool& p, int id, int j, int h) {
  return id * p.page + h * p.head + (unsigned)(j - prefill_page(s, j) * s.page) * p.row;
}

// acc + the squares of eight bf16 values
__device__ __forceinline__ float dot8(const bf16x8& x, float acc) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const bf16x2 y = {x[2 * k], x[2 * k + 1]};
    acc = __builtin_amdgcn_fdot2_f32_bf16(y, y, acc, false);
  }
  return acc;
}

// Eight columns c .. c+7 of a row of d, zeros beyond d
__device__ __forceinline__ bf16x8 ld8_cols(const bf16* row, int c, int d, bool vec) {
  const bf16x4 a = ld4_cols(row, c, d, vec), b = ld4_cols(row, c + 4, d, vec);
  return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// A tile of rows in LDS, chunk c (8 columns) of row r at c ^ tile_key(r).  Two kinds of reads have to find distinct banks
// among 64: 16 consecutive rows at one chunk (the rows of a first operand, 16 lanes of 16 bytes at a time) and 4 rows from a
// multiple of 4 at 4 adjacent chunks (a transposing read, 32 lanes of 8 bytes).  Rows of 256 bytes: the row's number in 16
// with its low and high half exchanged; rows of 128 bytes, two to a round of the banks: that of the pair in 8, its bits
// reversed.  Rows of 160 and 192 bytes stay as they are (some pairs of reads meet).
template <int W>
__device__ __forceinline__ int tile_key(int r) {
  if constexpr (W == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
  if constexpr (W == 64) return ((r & 2) << 1) | ((r & 4) >> 1) | ((r & 8) >> 3);
  return 0;
}
template <int W, typename T>
__device__ __forceinline__ T* tile_at(T* tile, int r, int c) {
  return tile + r * W + ((c ^ tile_key<W>(r)) << 3);
}

// --------------------------------------------------------------------------------------------
// Grid (4 panels of L, Hkv, B), 512 threads: four workgroups share a panel's rows to write and its tiles.  Every workgroup of
// a sequence looks its page ids over itself.  13 us for 2048 tokens of 8 heads of 128 columns: latency, a chain of loads (lengths,
// page ids, rows) before 36 tiles of products.  (P as hi + lo bf16, about 17 bits: the solve sums up to 255 of them.)
// --------------------------------------------------------------------------------------------
template <int W>
__global__ __launch_bounds__(512) void lucid_prefill_prep_kernel(const bf16* __restrict__ k, Strides ks, int vec,
                                                                 PagedPool kp, PrefillBatch seq, PagedScale f, float eps, int d,
                                                                 char* __restrict__ pmat, bf16* __restrict__ o, Strides os,
                                                                 int ovec, int G) {
  constexpr int CPR = W / 8, NKS = W / 16;
  __shared__ __attribute__((aligned(16))) bf16 rows[kPanel * W];
  __shared__ float norm[kPanel], inv[kPanel];
  __shared__ int bad_;
  const int panel = blockIdx.x >> 2, share = blockIdx.x & 3, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 5, l32 = lane & 31;
  const int32_t* tbl = seq.table + b * seq.tstride;
  const int n = seq.lens[b];
  int c = seq.counts ? min(max(seq.counts[b], 0), seq.L) : seq.L;
  if (n < 0) c = 0;
  // a page id outside the pool among those that the sequence needs, or a table too short for it
  bool bad = c > 0 && (int64_t)n + c > (int64_t)seq.M * seq.page;
  if (tid == 0) bad_ = 0;
  __syncthreads();
  if (c > 0 && !bad) {
    const int ids = prefill_page(seq, n + c - 1) + 1;
    bool any = false;
    for (int i = tid; i < ids; i += 512) any |= (unsigned)tbl[i] >= (unsigned)seq.P;
    if (any) bad_ = 1;
  }
  __syncthreads();
  bad |= bad_ != 0;
  const int t0 = panel * kPanel;
  // the outputs of padding (zeros) and of a sequence that is left out (NaN)
  const int from = bad ? 0 : c;
  const int each = kPanel / 4, t1 = min(t0 + each * (share + 1), seq.L);
  const bool packed = ovec && os.h == d;  // a row of a group's heads is one run
  for (int t = max(t0 + each * share, from) + w; t < t1; t += 8) {
    const bf16 x = (bf16)(t < c ? __builtin_nanf("") : 0.f);
    bf16* op = o + b * os.b + (int64_t)h * G * os.h + t * os.t;
    if (packed) {
      for (int i = 4 * lane; i < G * d; i += 256) *reinterpret_cast<bf16x4*>(op + i) = bf16x4{x, x, x, x};
    } else {
      for (int q = 0; q < G; ++q)
        for (int i = lane; i < d; i += 64) op[q * os.h + i] = x;
    }
  }
  if (bad) c = 0;
  if (blockIdx.x == 0 && h == 0 && tid == 0) seq.info[b] = make_int2(max(n, 0), c);
  if (t0 >= c) return;
  const int R = min(c - t0, kPanel);
  const bf16* kb = k + b * ks.b + h * ks.h + (int64_t)t0 * ks.t;
  for (int i = tid; i < kPanel * CPR; i += 512) {
    const int r = i / CPR, cc = i % CPR;
    bf16x8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (bf16)0.f;
    if (r < R) {
      x = ld8_cols(kb + r * ks.t, cc * 8, d, vec);
      const int j = n + t0 + r;
      if (r / each == share)
        *reinterpret_cast<bf16x8*>(paged_at(kp, prefill_row(seq, kp, tbl[prefill_page(seq, j)], j, h)) + cc * 8) = x;
    }
    *reinterpret_cast<bf16x8*>(tile_at<W>(rows, r, cc)) = x;
  }
  __syncthreads();
  char* pm = pmat + (((int64_t)b * seq.Hkv + h) * (gridDim.x >> 2) + panel) * kPanelBytes;
  {
    const int r = tid >> 1, half = tid & 1;
    float nn = 0.f;
    for (int cc = half; cc < CPR; cc += 2) {
      const bf16x8 x = ld8(tile_at<W>(rows, r, cc));
#pragma unroll
      for (int e = 0; e < 8; ++e) nn = fmaf((float)x[e], (float)x[e], nn);
    }
    nn += dpp_f32<kDppXor1>(nn);
    if (half == 0) {
      norm[r] = rsqrtf(nn / (float)d + eps);
      // 1 / P_tt; the exponent is the small difference of two terms of size sqrt(d): in fp64
      const double ms = (double)nn / d;
      inv[r] = __builtin_amdgcn_exp2f((float)(1.4426950408889634 * (1.0 / f.s - f.s * d * ms / (ms + eps))));
      if (share == 0) reinterpret_cast<float*>(pm + kPanelInv)[r] = inv[r];
    }
  }
  __syncthreads();
  // tiles (i, j), j <= i, of 32 x 32: S^T = K_j . K_i, lane <-> row of i, element <-> row of j
  for (int idx = 4 * w + share; idx < 36; idx += 32) {
    int i = (int)((sqrtf(8.f * idx + 1.f) - 1.f) * 0.5f);
    if ((i + 1) * (i + 2) / 2 <= idx) ++i;
    if (i * (i + 1) / 2 > idx) --i;
    const int j = idx - i * (i + 1) / 2;
    if (32 * i >= R) break;
    f32x16 sc = zero16();
#pragma unroll
    for (int st = 0; st < NKS; ++st)
      sc = mfma32(ld8(tile_at<W>(rows, 32 * j + l32, 2 * st + g)), ld8(tile_at<W>(rows, 32 * i + l32, 2 * st + g)), sc);
    float nr[16];
    lds_rows16(&norm[32 * j], g, nr);
    const float c1 = f.sl2 * norm[32 * i + l32], over = -inv[32 * i + l32];
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = over * __builtin_amdgcn_exp2f(fmaf(c1 * nr[e], sc[e], -f.c0));
    if (i == j) {
      float* dg = reinterpret_cast<float*>(pm + kPanelDiag) + i * 1024;
#pragma unroll
      for (int e = 0; e < 16; ++e) dg[drow(e, g) * 32 + l32] = l32 > drow(e, g) ? sc[e] : 0.f;
    } else {
      bf16* op = reinterpret_cast<bf16*>(pm) + (i * (i - 1) / 2 + j) * kPanelTile;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const bf16x8 hi = pack_b(sc, q), lo = pack_lo(sc, q, hi);
        *reinterpret_cast<bf16x8*>(op + (2 * q) * 512 + lane * 8) = hi;
        *reinterpret_cast<bf16x8*>(op + (2 * q + 1) * 512 + lane * 8) = lo;
      }
    }
  }
}

// --------------------------------------------------------------------------------------------
// How a sweep is shared out, worked out by every wave from the sequences' lengths and tokens.  All row tiles (RT of a
// sequence's rows, GX for each token) of all kv heads and sequences stand in one line, each as long as its keys' staged tiles, and
// every workgroup takes an equal share of it: whole row tiles, and at either end part of one, along the keys.  A part
// goes to slot 2 s of share s if it holds the share's beginning, else to 2 s + 1.  (Whole row tiles cut into equal parts
// instead left a last round half empty: 4 sequences of 300 to 512 tokens of 32/4 heads of 64 columns behind 8192 rows, 181 us.)
// Row tiles have 64 rows (four waves to 32 of them) or 256.  A place of 64 takes about 1 / 3.2 of one of 256, and a row tile
// costs as much again as 4 of its places: whichever sums to less.  (us of a call with 64 / 256 / as chosen: 16 sequences of 1 to
// 256 tokens of 16/16 heads of 64 columns behind 500 to 4000 rows 131 / 173 / 138; 16 of 256 each behind 4000 434 / 311 / 304,
// of 96 columns 695 / 409 / 412; 14 of 1 to 256 tokens of 32/4 heads of 68 columns behind 50 to 3500 77 / 85 / 74.)
// Places without keys lead every row tile: what beginning and ending one costs.  A share's end at the beginning of a row
// tile, or anywhere in a short one, goes back to where it starts.
// --------------------------------------------------------------------------------------------
struct SweepGrid {
  int GX, attend, target;      // target: shares at most
  int whole;                   // staged tiles of a row tile that is not cut at all
};
struct SweepPiece {
  int b, h, n, c, tile, j0, j1;
  int slot;   // -1: a whole row tile
  int place;  // the row tile's first (its keys follow kSweepLead behind)
  int len;    // its staged tiles
};
constexpr int kSweepLeast = 4;  // places of a share, at least
constexpr int kSweepLead = 4;   // places before a row tile's keys
constexpr int kSweepSnap = 2;   // staged tiles at a row tile's beginning that are not cut off

struct SweepPlan {
  PrefillBatch s;
  SweepGrid a;
  int RT;          // rows of a row tile
  int total, per;  // places of the line and of a share (their number fits: the host's check)
  int2 x0;         // sequence `lane` of the first 64
  __device__ __forceinline__ int tiles(const int2& x) const { return (x.y * a.GX + RT - 1) / RT; }
  __device__ __forceinline__ int keys(const int2& x) const { return x.x + (a.attend ? x.y : 0); }
  __device__ __forceinline__ int len(const int2& x) const { return max(1, (keys(x) + kSweepKeys - 1) / kSweepKeys); }
  __device__ __forceinline__ int2 at(int b) const { return b < 64 ? x0 : b < s.B ? s.info[b] : make_int2(0, 0); }
  __device__ __forceinline__ SweepPlan() {}
  // FORM: rows of a row tile, or 0: chosen here
  template <int FORM>
  __device__ __forceinline__ void init(const PrefillBatch& seq, const SweepGrid& grid) {
    s = seq;
    a = grid;
    const int lane = threadIdx.x & 63;
    x0 = lane < s.B ? s.info[lane] : make_int2(0, 0);
    auto sum = [&](auto of) {
      int all = 0;
      for (int b0 = 0; b0 < s.B; b0 += 64) all += __builtin_amdgcn_readlane(wave_scan(of(at(b0 + lane))), 63);
      return all;
    };
    auto places = [&](int rows) {
      return sum([&](const int2& x) { return s.Hkv * ((x.y * a.GX + rows - 1) / rows) * (len(x) + kSweepLead); });
    };
    RT = FORM;
    if constexpr (FORM == 0) {
      const int many = places(64), few = places(256), tiles64 = sum([&](const int2& x) { return s.Hkv * ((x.y * a.GX + 63) / 64); });
      RT = (float)many + 4.f * (float)tiles64 < 3.2f * (float)few ? 64 : 256;
      total = RT == 64 ? many : few;
    } else {
      total = places(FORM);
    }
    per = max(kSweepLeast, (total + a.target - 1) / a.target);
  }
  // The row tile at a place (below total)
  __device__ __forceinline__ void find(int place, SweepPiece& it) const {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b0 = 0; b0 < s.B; b0 += 64) {
      const int2 x = at(b0 + lane);
      const int tl = tiles(x), ln = len(x), end = base + wave_scan(s.Hkv * tl * (ln + kSweepLead));
      const unsigned long long hit = __ballot(place < end);
      if (hit) {
        const int l = __builtin_amdgcn_readfirstlane(__ffsll(hit) - 1);
        it.b = b0 + l;
        it.n = __builtin_amdgcn_readlane(x.x, l);
        it.c = __builtin_amdgcn_readlane(x.y, l);
        it.len = __builtin_amdgcn_readlane(ln, l);
        const int t = __builtin_amdgcn_readlane(tl, l);
        const int each = it.len + kSweepLead, first = __builtin_amdgcn_readlane(end, l) - s.Hkv * t * each;
        const int k = (place - first) / each;
        it.h = k / t;
        it.tile = k - it.h * t;
        it.place = first + k * each;
        return;
      }
      base = __builtin_amdgcn_readlane(end, 63);
    }
  }
  // Row tile number k of all; false: there are not so many
  __device__ __forceinline__ bool number(int k, SweepPiece& it) const {
    const int lane = threadIdx.x & 63;
    int base = 0, place = 0;
    for (int b0 = 0; b0 < s.B; b0 += 64) {
      const int2 x = at(b0 + lane);
      const int num = s.Hkv * tiles(x), end = base + wave_scan(num), places = num * (len(x) + kSweepLead),
                pend = place + wave_scan(places);
      const unsigned long long hit = __ballot(k < end);
      if (hit) {
        const int l = __builtin_amdgcn_readfirstlane(__ffsll(hit) - 1);
        it.b = b0 + l;
        it.n = __builtin_amdgcn_readlane(x.x, l);
        it.c = __builtin_amdgcn_readlane(x.y, l);
        it.len = __builtin_amdgcn_readlane(len(x), l);
        const int t = __builtin_amdgcn_readlane(tiles(x), l), i = k - (__builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(num, l));
        it.h = i / t;
        it.tile = i - it.h * t;
        it.place = __builtin_amdgcn_readlane(pend, l) - __builtin_amdgcn_readlane(places, l) + i * (it.len + kSweepLead);
        return true;
      }
      base = __builtin_amdgcn_readlane(end, 63);
      place = __builtin_amdgcn_readlane(pend, 63);
    }
    return false;
  }
  // Places from a row tile's first on at which no share ends
  __device__ __forceinline__ int uncut(const SweepPiece& it) const {
    return it.len <= a.whole ? it.len + kSweepLead : kSweepLead + kSweepSnap;
  }
  // Where share number k begins (its row tile goes to it)
  __device__ __forceinline__ int begin(int k, SweepPiece& it) const {
    const int place = k * per;
    if (place >= total) return total;
    find(place, it);
    return place - it.place < uncut(it) ? it.place : place;
  }
};

struct SweepParts {
  float* o;  // [2 shares][RT][W]
  float* m;  // [2 shares][RT]  running max (log2 domain), attend
  float* l;  // [2 shares][RT]  running sum, attend
};

template <int W, int KT>
struct SweepSmem {
  union {
    // staged tiles, filled by direct global -> LDS loads (the transposing reads of W = 80 end 32 bytes behind a tile)
    struct {
      bf16 k[2][KT * W], v[2][KT * W + 64];
    } st;
    struct {
      float o[2][64][W + 4], m[4][64], l[4][64];
    } fin;
  } u;
  float nr[2][KT];  // couple: 1 / rms of a tile's keys
};

// The transposing reads of MFMA A operands (paged_tr_a) from such a tile: the lane's offsets at row 0 for column block
// col0 and its rows of the first and of the second read, 8 on (their keys differ); row0, a multiple of 16, adds row0 W
struct TileTr {
  int o1, o2;
};
template <int W>
__device__ __forceinline__ TileTr tile_tr_off(int col0) {
  const int lane = threadIdx.x & 63, s = lane & 15;
  const int col = col0 + 16 * ((lane >> 4) & 1) + 4 * (s & 3), r1 = 4 * (lane >> 5) + (s >> 2);
  return TileTr{r1 * W + (((col >> 3) ^ tile_key<W>(r1)) << 3) + (col & 7),
                (r1 + 8) * W + (((col >> 3) ^ tile_key<W>(r1 + 8)) << 3) + (col & 7)};
}
template <int W>
__device__ __forceinline__ bf16x8 tile_tr(const bf16* tile, const TileTr& o, int row0) {
  typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
  const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(tile + o.o1 + row0 * W));
  const bf16x4 v2 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(tile + o.o2 + row0 * W));
  return bf16x8{v1[0], v1[1], v1[2], v1[3], v2[0], v2[1], v2[2], v2[3]};
}

// Matrix units and VALU take turns: of a SIMD's cycles, attending at 128 columns has MFMAs in 52 % and the VALU in 41 % (0.97
// PFLOP/s of a large product's 1.36), at 64 columns in 35 and 51 % (0.65), with the LDS read in 26 and 18 % of a CU's.  These are no
// bounds of the chip: the kernels on contiguous rows reach 1.18 and 0.95 PFLOP/s; at 64 columns theirs hold 64 rows a wave, two products
// for each operand read from LDS, where these waves hold 32.  Both products are written so that lanes stay rows: the scores leave the first as the
// second's operand, without LDS.  Only tiles with a key that some row of the wave does not see are masked.
// Eight waves over tiles of 128 keys, staged once for all of them; KSP waves share 32 rows and take every KSP-th 32 keys
// (RT = 256 / KSP rows).  Lane <-> row: S^T[j][i] = K_j . x_i, then acc^T[col][i] +=
// w^T[col][j] p^T[j][i].
//   attend: x = q, rows (token, query head of the group) token by token, online softmax.  Its weights enter the second product
//           as one bf16 and are summed as such, as in the kernels on contiguous rows: O is off by 0.0024 of its norm, 0.0017 of it
//           the rounding of O itself.  As a pair (0.0017 in all) they would cost half the products of this sweep again: 2048 tokens
//           of 32/8 heads of 128 columns behind 32768 rows 1.71 -> 2.20 ms, 4 x 512 of 32/4 of 64 behind 8192 262 -> 335 us.
//           Nothing carries this rounding on, unlike the coupling's, whose errors the solve and the cache keep
//   couple: x = the new keys, p = P as a bf16 pair; y = v - acc
//   inner:  as couple, with the keys of one panel of new rows and out of the y of the rows behind it; grid (row
//           tiles, Hkv, B), where the others go by SweepPlan
enum class Sweep { Couple, Attend, Inner };
template <int W, Sweep MODE, int KSP>
__device__ __forceinline__ void prefill_sweep(
    SweepSmem<W, kSweepKeys>& sm, const SweepPlan& plan, const bf16* x, const Strides& xs, int vec,
    const bf16* v, const Strides& vs, const PagedPool& kp, const PagedPool& vp, const PrefillBatch& seq,
    const SweepGrid& grid, int panel, const PagedScale& f, float eps, int d, float* y, int64_t yrows,
    bf16* o, const Strides& os, int ovec, const SweepParts& part) {
  constexpr bool ATTEND = MODE == Sweep::Attend, LINE = MODE != Sweep::Inner;
  constexpr int NKS = W / 16, NDT = (W + 31) / 32, CPR = W / 8, NST = CPR / 2, KT = kSweepKeys, NMT = KT / 32 / KSP;
  constexpr int NW = 8, RT = 32 * NW / KSP;
  static_assert(KSP == 1 || RT == 64, "the join of key groups holds 64 rows");
  int share = 0, start = 0, place = 0, end = 1, row_base = 0;
  SweepPiece it;
  if constexpr (LINE) {
    // ids go round robin over the 8 XCDs: each takes a run of shares, the row tiles of one kv head next to each other
    const int num = (plan.total + plan.per - 1) / plan.per, each = (num + 7) >> 3;
    share = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= each || share >= num) return;
    SweepPiece behind;
    end = plan.begin(share + 1, behind);
    start = place = plan.begin(share, it);
  }
  while (place < end) {
  if constexpr (LINE) {
    if (place != start) plan.find(place, it);
    const int first = it.place + kSweepLead, next = min(end, first + it.len);
    it.j0 = max(place - first, 0) * kSweepKeys;
    it.j1 = min(plan.keys(make_int2(it.n, it.c)), (next - first) * kSweepKeys);
    it.slot = place == it.place && next == first + it.len ? -1 : 2 * share + (place == start ? 0 : 1);
    place = next;
  } else {
    place = end;
    it.b = blockIdx.z;
    it.h = blockIdx.y;
    it.tile = blockIdx.x;
    const int2 i = seq.info[it.b];
    it.n = __builtin_amdgcn_readfirstlane(i.x);
    it.c = __builtin_amdgcn_readfirstlane(i.y);
    row_base = kPanel * (panel + 1);
    it.j0 = it.n + kPanel * panel;
    it.j1 = it.j0 + kPanel;
    it.slot = -1;
    if (row_base + it.tile * RT >= it.c) return;
  }
  const int b = it.b, h = it.h, n = it.n, GX = grid.GX;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // what follows from it is worked out here, not kept in registers across the pieces
  const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, l32 = lane & 31;
  const int rw = w / KSP, kg = w % KSP;
  const int rows = it.c * GX, row0 = row_base + it.tile * RT + 32 * rw;  // of this wave
  const bool active = row0 < rows;
  const int row = row0 + l32, mine = min(row, rows - 1), t = mine / GX, hq = h * GX + (mine - t * GX);  // of the lane
  // attend: no row of this workgroup sees a key beyond its last token's
  const int last = min(row_base + (it.tile + 1) * RT, rows) - 1;
  const int j0 = it.j0, j1 = ATTEND ? min(it.j1, n + last / GX + 1) : it.j1;
  const int lim = ATTEND ? min(j1 - 1, n + t) : j1 - 1;                           // the lane's last key,
  const int free = ATTEND ? min(j1 - 1, n + min(row0, rows - 1) / GX) : j1 - 1;  // one that all lanes of the wave see,
  const int most = ATTEND ? n + min(row0 + 31, rows - 1) / GX : j1 - 1;  // and one beyond which none does
  const int ntile = (j1 - j0 + KT - 1) / KT;

  // staging: half of the waves the keys, the others V', 32 rows each
  const int32_t* tbl = seq.table + b * seq.tstride;
  const int part_of = w % (NW / 2);
  const bool isv = w >= NW / 2;
  const PagedPool pool = isv ? vp : kp;
  auto key_of = [&](int tile) { return min(j0 + KT * tile + 32 * part_of + l32, j1 - 1); };
  // Pages of whole runs of 32 rows: a wave's rows of a tile lie in one page, whose place is scalar work, and the lanes' offsets
  // in it are those of every tile.  The last tile, whose rows may end before it does, goes row by row in any case.
  const bool runs = seq.page % 32 == 0 && j0 % 32 == 0 && pool.row < (1u << 22);
  unsigned lane_off[NST];
#pragma unroll
  for (int i = 0; i < NST; ++i) {
    const int q = i * 64 + lane, r = q / CPR;
    lane_off[i] = 16 * (r * pool.row + ((q % CPR) ^ tile_key<W>(r)));
  }
  auto whole = [&](int tile) { return runs && j0 + KT * (tile + 1) <= j1; };
  auto page_id = [&](int tile) {
    const int j = whole(tile) ? j0 + KT * tile + 32 * part_of : key_of(tile);
    return tbl[prefill_page(seq, j)];
  };
  auto stage = [&](int tile, int id, int buf) {
    bf16* dst = (isv ? sm.u.st.v[buf] : sm.u.st.k[buf]) + 32 * part_of * W;
    if (whole(tile)) {
      const char* base = reinterpret_cast<const char*>(
          paged_at(pool, prefill_row(seq, pool, __builtin_amdgcn_readfirstlane(id), j0 + KT * tile + 32 * part_of, h)));
#pragma unroll
      for (int i = 0; i < NST; ++i)
        __builtin_amdgcn_global_load_lds(reinterpret_cast<const bf16*>(base + lane_off[i]), dst + i * 512, 16, 0, 0);
      return;
    }
    const unsigned off = prefill_row(seq, pool, id, key_of(tile), h);
#pragma unroll
    for (int i = 0; i < NST; ++i) {
      const int q = i * 64 + lane, r = q / CPR, c = (q % CPR) ^ tile_key<W>(r);
      __builtin_amdgcn_global_load_lds(paged_at(pool, __shfl((int)off, r, 64)) + c * 8, dst + i * 512, 16, 0, 0);
    }
  };
  // couple: once a wave's own keys have landed it works out their norms, two lanes a key
  auto norms = [&](int buf) {
    if (ATTEND || isv) return;
    const int r = 32 * part_of + (lane >> 1);
    float nn = 0.f;
#pragma unroll
    for (int cc = 0; cc < CPR; cc += 2) nn = dot8(ld8(tile_at<W>(sm.u.st.k[buf], r, cc + (lane & 1))), nn);
    nn += dpp_f32<kDppXor1>(nn);
    if ((lane & 1) == 0) sm.nr[buf][r] = rsqrtf(nn / (float)d + eps);
  };
  int idn = 0;
  if (ntile > 0) {
    const int id0 = page_id(0);
    if (ntile > 1) idn = page_id(1);
    stage(0, id0, 0);
  }
  const float c = f.sl2;
  bf16x8 xb[NKS];
  float c1 = 0.f, m = PREFILL_NEG, lsum = 0.f;
  f32x16 acc[NDT];
  const bf16* xr = x + b * xs.b + (ATTEND ? hq : h) * xs.h + t * xs.t;
#pragma unroll
  for (int st = 0; st < NKS; ++st) xb[st] = ld8_cols(xr, 16 * st + 8 * g, d, vec);
#pragma unroll
  for (int q = 0; q < NDT; ++q) acc[q] = zero16();
  if constexpr (!ATTEND) {
    float nt = 0.f;
#pragma unroll
    for (int st = 0; st < NKS; ++st) nt = dot8(xb[st], nt);
    c1 = c * rsqrtf(wave_sum32(nt) / (float)d + eps);
  }
  TileTr tr[NDT];
#pragma unroll
  for (int q = 0; q < NDT; ++q) tr[q] = tile_tr_off<W>(32 * q);
  // the rows have landed before the loop (else every tile's first product waits for the next tile's loads)
#pragma unroll
  for (int st = 0; st < NKS; ++st) asm volatile("" ::"v"(xb[st]));
  dma_wait();
  if (ntile > 0) norms(0);
  __syncthreads();
  for (int jt = 0; jt < ntile; ++jt) {
    const int buf = jt & 1, jb = j0 + KT * jt;
    if (jt + 1 < ntile) {
      stage(jt + 1, idn, buf ^ 1);
      if (jt + 2 < ntile) idn = page_id(jt + 2);
    }
    if (active && jb <= most) {
      const bf16* tk = sm.u.st.k[buf];
      const bf16* tv = sm.u.st.v[buf];
      const bool mask = jb + KT - 1 > free;
      if constexpr (ATTEND) {
        f32x16 s[NMT];
#pragma unroll
        for (int i = 0; i < NMT; ++i) {
          const int mt = kg + KSP * i;
          s[i] = zero16();
#pragma unroll
          for (int st = 0; st < NKS; ++st) {
            const bf16x8 kf = ld8(tile_at<W>(tk, mt * 32 + l32, 2 * st + g));
            s[i] = mfma32(kf, xb[st], s[i]);
          }
        }
        if (mask) {
#pragma unroll
          for (int i = 0; i < NMT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (jb + (kg + KSP * i) * 32 + drow(e, g) > lim) s[i][e] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < NMT; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[i][e]);
        mx = wave_max32(mx) * c;
        if (__builtin_amdgcn_ballot_w64(mx > m + 8.0f)) {  // rescale only where a row grows by 2^8
          const float mnew = fmaxf(m, mx);
          const float alpha = __builtin_amdgcn_exp2f(m - mnew);
          m = mnew;
          lsum *= alpha;
#pragma unroll
          for (int q = 0; q < NDT; ++q)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[q][e] *= alpha;
        }
#pragma unroll
        for (int i = 0; i < NMT; ++i) {
          const int mt = kg + KSP * i;
#pragma unroll
          for (int e = 0; e < 16; ++e) s[i][e] = __builtin_amdgcn_exp2f(fmaf(s[i][e], c, -m));
          const bf16x8 p0 = pack_b(s[i], 0), p1 = pack_b(s[i], 1);
          lsum = add_sum8(p1, add_sum8(p0, lsum));  // sum of the bf16 P of the product
#pragma unroll
          for (int q = 0; q < NDT; ++q) {
            const bf16x8 a0 = tile_tr<W>(tv, tr[q], mt * 32), a1 = tile_tr<W>(tv, tr[q], mt * 32 + 16);
            acc[q] = mfma32(a0, p0, acc[q]);
            acc[q] = mfma32(a1, p1, acc[q]);
          }
        }
      } else {
        // (the masked and the whole tile as two bodies, so that no branch parts the sub-tiles, spill up to 283 registers:
        // 2048 tokens of 32/8 heads of 128 columns behind 32768 rows 394 -> 850 us)
#pragma unroll
        for (int i = 0; i < NMT; ++i) {
          const int mt = kg + KSP * i;
          f32x16 s = zero16();
#pragma unroll
          for (int st = 0; st < NKS; ++st) {
            const bf16x8 kf = ld8(tile_at<W>(tk, mt * 32 + l32, 2 * st + g));
            s = mfma32(kf, xb[st], s);
          }
          float nr[16];
          lds_rows16(&sm.nr[buf][32 * mt], g, nr);
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(c1 * nr[e], s[e], -f.c0));
          if (mask) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (jb + mt * 32 + drow(e, g) > lim) s[e] = 0.f;
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const bf16x8 hi = pack_b(s, k), lo = pack_lo(s, k, hi);
#pragma unroll
            for (int q = 0; q < NDT; ++q) {
              const bf16x8 a = tile_tr<W>(tv, tr[q], mt * 32 + 16 * k);
              acc[q] = mfma32(a, hi, acc[q]);
              acc[q] = mfma32(a, lo, acc[q]);
            }
          }
        }
      }
    }
    dma_wait();
    if (jt + 1 < ntile) norms(buf ^ 1);
    __syncthreads();
  }
  float l = ATTEND ? wave_sum32(lsum) : 0.f;
  if constexpr (KSP > 1) {  // the key groups' sums joined in the waves of group 0
    const int r = 32 * rw + l32;
    if constexpr (ATTEND) {
      if (g == 0) {
        sm.u.fin.m[kg][r] = m;
        sm.u.fin.l[kg][r] = l;
      }
      __syncthreads();
      float M = sm.u.fin.m[0][r];
#pragma unroll
      for (int k = 1; k < KSP; ++k) M = fmaxf(M, sm.u.fin.m[k][r]);
      l = 0.f;
#pragma unroll
      for (int k = 0; k < KSP; ++k) l = fmaf(sm.u.fin.l[k][r], __builtin_amdgcn_exp2f(sm.u.fin.m[k][r] - M), l);
      const float a = __builtin_amdgcn_exp2f(m - M);
      m = M;
#pragma unroll
      for (int q = 0; q < NDT; ++q)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[q][e] *= a;
    }
#pragma unroll
    for (int half = KSP / 2; half >= 1; half /= 2) {
      __syncthreads();
      if (kg >= half && kg < 2 * half) {
#pragma unroll
        for (int q = 0; q < NDT; ++q)
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            if (32 * q + drow(e, 0) < W)
              *reinterpret_cast<f32x4*>(&sm.u.fin.o[kg - half][r][32 * q + drow(e, g)]) =
                  f32x4{acc[q][e], acc[q][e + 1], acc[q][e + 2], acc[q][e + 3]};
      }
      __syncthreads();
      if (kg < half) {
#pragma unroll
        for (int q = 0; q < NDT; ++q)
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            if (32 * q + drow(e, 0) < W) {
              const f32x4 z = *reinterpret_cast<const f32x4*>(&sm.u.fin.o[kg][r][32 * q + drow(e, g)]);
#pragma unroll
              for (int u = 0; u < 4; ++u) acc[q][e + u] += z[u];
            }
      }
    }
  }
  if (kg == 0 && row < rows) {
    if (it.slot >= 0) {
      const int64_t at = (int64_t)it.slot * RT + 32 * rw + l32;
#pragma unroll
      for (int q = 0; q < NDT; ++q)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          if (32 * q + drow(e, 0) < W)
            *reinterpret_cast<f32x4*>(part.o + at * W + 32 * q + drow(e, g)) =
                f32x4{acc[q][e], acc[q][e + 1], acc[q][e + 2], acc[q][e + 3]};
      if (ATTEND && g == 0) {
        part.m[at] = m;
        part.l[at] = l;
      }
    } else if constexpr (ATTEND) {
      const float inv = 1.f / l;
      bf16* op = o + b * os.b + hq * os.h + t * os.t;
#pragma unroll
      for (int q = 0; q < NDT; ++q)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int col = 32 * q + drow(e, g);
          bf16x4 z;
#pragma unroll
          for (int u = 0; u < 4; ++u) z[u] = (bf16)(acc[q][e + u] * inv);
          if (ovec && col + 4 <= d) {
            *reinterpret_cast<bf16x4*>(op + col) = z;
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (col + u < d) op[col + u] = z[u];
          }
        }
    } else {
      float* yp = y + (((int64_t)b * seq.Hkv + h) * yrows + t) * W;
      const bf16* vr = v + b * vs.b + h * vs.h + t * vs.t;
#pragma unroll
      for (int q = 0; q < NDT; ++q)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int col = 32 * q + drow(e, g);
          if (32 * q + drow(e, 0) >= W) continue;
          f32x4 z;
          if (!LINE) {
            z = *reinterpret_cast<const f32x4*>(yp + col);
          } else {
            const bf16x4 v4 = ld4_cols(vr, col, d, ovec);
            z = f32x4{(float)v4[0], (float)v4[1], (float)v4[2], (float)v4[3]};
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) z[u] -= acc[q][e + u];
          *reinterpret_cast<f32x4*>(yp + col) = z;
        }
    }
  }
  if (LINE && KSP > 1 && place < end) __syncthreads();  // the join's rows are read before the next piece's tiles come
  }
}

template <int W, Sweep MODE, int FORM>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) void lucid_prefill_sweep_kernel(
    const bf16* __restrict__ x, Strides xs, int vec, const bf16* __restrict__ v, Strides vs, PagedPool kp, PagedPool vp,
    PrefillBatch seq, SweepGrid grid, int panel, PagedScale f, float eps, int d, float* __restrict__ y, int64_t yrows,
    bf16* __restrict__ o, Strides os, int ovec, SweepParts part) {
  __shared__ __attribute__((aligned(16))) SweepSmem<W, kSweepKeys> sm;
  SweepPlan plan;
  if constexpr (MODE != Sweep::Inner) plan.init<FORM>(seq, grid);
  if constexpr (FORM != 64)
    if (FORM == 256 || plan.RT == 256) {
      prefill_sweep<W, MODE, 1>(sm, plan, x, xs, vec, v, vs, kp, vp, seq, grid, panel, f, eps, d, y, yrows, o, os, ovec, part);
      return;
    }
  if constexpr (FORM != 256)
    prefill_sweep<W, MODE, 4>(sm, plan, x, xs, vec, v, vs, kp, vp, seq, grid, panel, f, eps, d, y, yrows, o, os, ovec, part);
}

// --------------------------------------------------------------------------------------------
// The parts of the row tiles that a share's end cuts, joined in fp32: 10 us for the two of 8 heads, 32 row tiles each, of 128
// columns.  Grid (row tiles at most, pieces of one), 256 threads: a piece of
// join_rows(W) rows, W / 4 lanes a row.
// --------------------------------------------------------------------------------------------
constexpr int join_rows(int W) { return 256 / (W / 4); }
constexpr int join_pieces(int W, int RT) { return (RT + join_rows(W) - 1) / join_rows(W); }
template <int W, bool ATTEND, int FORM>
__global__ __launch_bounds__(256) void lucid_prefill_join_kernel(const bf16* __restrict__ v, Strides vs, int vec,
                                                                 PrefillBatch seq, SweepGrid grid, int d, float* __restrict__ y,
                                                                 int64_t yrows, bf16* __restrict__ o, Strides os, int ovec,
                                                                 SweepParts part) {
  constexpr int CG = W / 4;
  SweepPlan plan;
  plan.init<FORM>(seq, grid);
  SweepPiece it;
  int tile = blockIdx.x, piece = blockIdx.y;
  if constexpr (FORM == 0) {  // a line of them: the first pieces of all row tiles, then the second ones, ..
    const int tiles = seq.B * seq.Hkv * ((seq.L * grid.GX + plan.RT - 1) / plan.RT), index = blockIdx.y * gridDim.x + blockIdx.x;
    piece = index / tiles;
    tile = index - piece * tiles;
  }
  if (!plan.number(tile, it)) return;
  // the last share that begins at its first place, or the one that has it beside others
  const int share = (it.place + plan.uncut(it) - 1) / plan.per;
  const int parts = (it.place + kSweepLead + it.len - 1) / plan.per - share + 1;
  if (parts == 1) return;
  const int slot0 = 2 * share + (share * plan.per >= it.place ? 0 : 1);
  const int GX = grid.GX, rows = it.c * GX;
  {
    const int i = threadIdx.x, r = join_rows(W) * piece + i / CG, col = 4 * (i % CG),
              row = it.tile * plan.RT + r;
    if (i >= join_rows(W) * CG || r >= plan.RT || row >= rows) return;
    const int t = row / GX, hq = it.h * GX + (row - t * GX);
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
    float M = PREFILL_NEG, l = 0.f;
    constexpr int UN = 8;  // parts asked for at a time (those beyond the last: the last, with the weight 0)
    for (int p0 = 0; p0 < parts; p0 += UN) {
      f32x4 x[UN];
      float m[UN], lp[UN];
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        const int p = min(p0 + k, parts - 1);
        const int64_t at = (int64_t)(p == 0 ? slot0 : 2 * (share + p)) * plan.RT + r;
        x[k] = *reinterpret_cast<const f32x4*>(part.o + at * W + col);
        m[k] = ATTEND ? part.m[at] : 0.f;
        lp[k] = ATTEND ? part.l[at] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        const bool on = p0 + k < parts;
        if constexpr (ATTEND) {
          const float mn = on ? fmaxf(M, m[k]) : M;
          const float a = __builtin_amdgcn_exp2f(M - mn), e = on ? __builtin_amdgcn_exp2f(m[k] - mn) : 0.f;
          l = fmaf(l, a, lp[k] * e);
#pragma unroll
          for (int u = 0; u < 4; ++u) z[u] = fmaf(z[u], a, x[k][u] * e);
          M = mn;
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u) z[u] += on ? x[k][u] : 0.f;
        }
      }
    }
    if constexpr (ATTEND) {
      const float inv = 1.f / l;
      bf16* op = o + it.b * os.b + hq * os.h + t * os.t;
      bf16x4 r4;
#pragma unroll
      for (int u = 0; u < 4; ++u) r4[u] = (bf16)(z[u] * inv);
      if (ovec && col + 4 <= d) {
        *reinterpret_cast<bf16x4*>(op + col) = r4;
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (col + u < d) op[col + u] = r4[u];
      }
    } else {
      const bf16x4 r4 = ld4_cols(v + it.b * vs.b + it.h * vs.h + t * vs.t, col, d, vec);
#pragma unroll
      for (int u = 0; u < 4; ++u) z[u] = (float)r4[u] - z[u];
      *reinterpret_cast<f32x4*>(y + (((int64_t)it.b * seq.Hkv + it.h) * yrows + t) * W + col) = z;
    }
  }
}

// --------------------------------------------------------------------------------------------
// One panel's rows in order: with z_t = y_t / P_tt, w_t = bf16(z_t) and z_u -= P_ut / P_uu w_t for u > t.  Grid (32 columns,
// Hkv, B), a wave for each block of 32 rows: columns are independent (lane <-> column, elements <-> rows).  A wave goes
// through its block by itself, row by row, each row's value from one lane half to the other in the VALU; the waves of the
// blocks behind wait for its rows, operands of theirs as they stand in registers, and take them out with MFMAs, their tile of
// P fetched a block ahead.  The chain of 256 dependent rows bounds it.  (One wave for all blocks, with the panel's 145 KB of P
// staged in LDS, took 24.5 us a panel where this takes 16.5.)
// --------------------------------------------------------------------------------------------
template <int W>
__global__ __launch_bounds__(64 * kPanelBlocks) void lucid_prefill_solve_kernel(
    const char* __restrict__ pmat, int panels, int panel, const float* __restrict__ y, int64_t yrows, PagedPool vp,
    PrefillBatch seq, int d) {
  __shared__ __attribute__((aligned(16))) struct {
    float diag[kPanelBlocks][1024];
    bf16 w[kPanelBlocks][1024];  // a block's rows as two operands
    unsigned off[kPanel];
  } sm;
  const int h = blockIdx.y, b = blockIdx.z;
  const int2 info = seq.info[b];
  const int R = min(info.y - panel * kPanel, kPanel);
  if (R <= 0) return;
  const int lane = threadIdx.x & 63, g = lane >> 5, l32 = lane & 31;
  const int own = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // this wave's block
  const int nb = (R + 31) / 32;                                      // blocks with rows
  const int64_t bh = (int64_t)b * seq.Hkv + h;
  const char* pm = pmat + (bh * panels + panel) * kPanelBytes;
  const bf16* tiles = reinterpret_cast<const bf16*>(pm) + (own * (own - 1) / 2) * kPanelTile + lane * 8;
  const int col = 32 * blockIdx.x + l32;
  const bool on = col < d;
  bf16x8 p0, p1, p2, p3;
  auto fetch = [&](int j) {
    p0 = ld8(tiles + j * kPanelTile);
    p1 = ld8(tiles + j * kPanelTile + 512);
    p2 = ld8(tiles + j * kPanelTile + 1024);
    p3 = ld8(tiles + j * kPanelTile + 1536);
  };
  f32x16 z = zero16();
  if (own < nb) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      dma_1k(reinterpret_cast<const bf16*>(pm + kPanelDiag) + own * 2048 + i * 512,
             reinterpret_cast<bf16*>(sm.diag[own]) + i * 512);
    const float* yb = y + (bh * yrows + panel * kPanel) * W + min(col, W - 1);
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = yb[min(32 * own + drow(e, g), R - 1) * W];
    float iv[16];
    lds_rows16(reinterpret_cast<const float*>(pm + kPanelInv) + 32 * own, g, iv);
    if (own > 0) fetch(0);
    const int r = 32 * own + l32;
    if (lane < 32 && r < R) {  // (those behind stay as they are: read, not used)
      const int j = info.x + panel * kPanel + r;
      sm.off[r] = prefill_row(seq, vp, seq.table[b * seq.tstride + prefill_page(seq, j)], j, h);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = 32 * own + drow(e, g) < R ? z[e] * iv[e] : 0.f;
  }
  dma_wait();
  __syncthreads();
#pragma unroll 1
  for (int i = 0; i < nb; ++i) {
    f32x16 fin;
    if (own == i) {
      const float* dg = sm.diag[i] + 4 * g;
      // P of row t arrives kAhead rows before its turn
      constexpr int kAhead = 3;
      f32x4 p[kAhead + 1][4];
      auto ask = [&](int t) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (8 * q + 7 > t) p[t % (kAhead + 1)][q] = *reinterpret_cast<const f32x4*>(dg + 32 * t + 8 * q);
      };
#pragma unroll
      for (int e = 0; e < 16; ++e) fin[e] = 0.f;
#pragma unroll
      for (int t = 0; t < kAhead; ++t) ask(t);
#pragma unroll
      for (int t = 0; t < 32; ++t) {
        const int e_t = 4 * (t >> 3) + (t & 3), g_t = (t >> 2) & 1;
        if (t + kAhead < 32) ask(t + kAhead);
        __builtin_amdgcn_sched_barrier(0);
        const unsigned u = __builtin_bit_cast(unsigned, (float)(bf16)z[e_t]);
        const auto both = __builtin_amdgcn_permlane32_swap(u, u, false, false);  // the first half's, the second's
        const float wt = __builtin_bit_cast(float, g_t ? (unsigned)both[1] : (unsigned)both[0]);
        fin[e_t] = g == g_t ? wt : fin[e_t];
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (8 * q + 4 + k > t) z[4 * q + k] = fmaf(p[t % (kAhead + 1)][q][k], wt, z[4 * q + k]);
      }
      *reinterpret_cast<bf16x8*>(sm.w[i] + lane * 8) = pack_b(fin, 0);
      *reinterpret_cast<bf16x8*>(sm.w[i] + 512 + lane * 8) = pack_b(fin, 1);
    }
    __syncthreads();
    if (own > i && own < nb) {
      const bf16x8 w0 = ld8(sm.w[i] + lane * 8), w1 = ld8(sm.w[i] + 512 + lane * 8);
      z = mfma32(p0, w0, z);
      z = mfma32(p1, w0, z);
      z = mfma32(p2, w1, z);
      z = mfma32(p3, w1, z);
      if (own > i + 1) fetch(i + 1);
    } else if (own == i && col < W) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int r = 32 * i + drow(e, g);
        if (r < R) paged_at(vp, sm.off[r])[col] = (bf16)(on ? fin[e] : 0.f);
      }
    }
  }
}

}  // namespace lucid
