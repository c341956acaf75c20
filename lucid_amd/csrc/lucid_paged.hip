// Paged (K, V') caches on CDNA4 (gfx950): decoding against them, writing a prefill's rows into them
// and copying their pages (modeling_lucid.py:475-496, 576-598 is the cached path of the reference,
// whose cache is one buffer per layer and one length for the whole batch).
//
// Row j of sequence b is row j % page of page table[b][j / page] of a layer's two pools (keys with
// RoPE applied, V' rows; bf16 [P][Hkv][page][W] by their strides, W = 64, 80, 96 or 128 the smallest
// that holds the head dim, columns beyond it zero).  Each sequence has its own length lens[b]; a
// negative one marks a batch slot without a sequence.  For a new token t of a sequence:
//   P_tj = exp(s r_t r_j (k_t . k_j) - 1/s),  r = 1 / rms(k)  (j < t, cached or new)
//   v'_t = (v_t - sum_{j<t} P_tj w_j) / P_tt,  P_tt = exp(s dn ms_t / (ms_t + eps) - 1/s)
//   o_tg = softmax_j(s q_tg . k_j) w_j over j <= t, for the G query heads of the kv head
// with w_j the V' row as the cache holds it (bf16), new rows too, so that L tokens in one call are L
// calls of one token.  The products with the cached rows read each of them once (bytes bound it):
//   lucid_paged_split_kernel    a share of the rows of one kv head, all sequences in a line: of each
//                               sequence that it covers a part of, partial sum_j P_tj w_j and the
//                               online-softmax state of every (token, query head)
//   lucid_paged_combine_kernel  a sequence's parts merged, the new tokens solved in order, the outputs,
//                               and (k_t, v'_t) appended to the pages
#include "lucid_common.h"

namespace lucid {

constexpr float PAGED_NEG = -1e30f;    // finite "minus infinity" for empty softmax states
// Rows that a workgroup takes at a time, a tile for each of its four waves.  (Finer units balance the shares better and
// leave waves without a tile: with 32 rows, and lead to match, 21.7 to 23.3 us for 20.2 at 32 sequences of up
// to 3500 rows, 110 for 104 at one of 131072.)
constexpr int kPagedUnit = 128;
constexpr int kPagedLead = 1;          // places that a sequence takes in the line beside its rows
constexpr int kPagedMaxTokens = 16;    // new tokens of a pass
// Cache policy of the direct loads of V' (the instruction's nt bit): where no page is shared, a pass reads each line
// once, by one instruction, and need not push others out.  131072 rows of 8 kv heads 106 -> 96 us, 32 sequences of
// 8192 rows of 4 102 -> 93 at 128 columns and 61 -> 57 at 64, caches changing from call to call.  The keys keep the
// usual policy: a line of theirs is read by several instructions of a wave (with the bit 125 us).
// Lines that are read again, with the bit and without it: in pages that sequences share it costs up to 5 % (32
// samples of a prompt of 8192 rows 83 and 79 us, 64 of 1024 37.9 and 36.3, 8 of 8192 36.8 and 36.2, 8 of 32768 the
// same); by the second chunk of 32 query heads a kv head it still gains (131072 rows 80.5 and 85.7, 16 sequences of
// 4096 56.6 and 57.8), and by the second pass of eight tokens (94 and 97 at 128 columns, 110 and 111 at 68), while
// 64 tokens in ten passes lose (342 and 337).
constexpr int kPagedOnce = 2;

struct PagedBatch {
  const int32_t* table;  // [B][M] page ids, rows tstride apart
  int64_t tstride;
  const int32_t* lens;  // [B] rows cached before the call
  int B, M, P, page;
  int shift;  // log2 of page, -1 where it is no power of two
  int L;      // new tokens of the call
  int done;   // of earlier passes
};
__device__ __forceinline__ int page_of(const PagedBatch& s, int j) { return s.shift >= 0 ? j >> s.shift : j / s.page; }

// A pool by its strides in units of 16 bytes (8 elements); the host checks that every row's offset
// fits 32 bits, a pool of 64 GB.
struct PagedPool {
  bf16* base;
  unsigned page, head, row;
};
__device__ __forceinline__ bf16* paged_at(const PagedPool& p, unsigned off) { return p.base + (size_t)off * 8; }

// Rows of sequence b before this pass; -1: no sequence, -2: its new rows do not fit its table
__device__ __forceinline__ int paged_rows(const PagedBatch& s, int b) {
  const int n = s.lens[b];
  if (n < 0) return -1;
  return (int64_t)n + s.L > (int64_t)s.M * s.page ? -2 : n + s.done;
}

// The sequences' rows stand in one line, each sequence rounded up to units of kPagedUnit rows and led by
// kPagedLead units without rows, and workgroup s of a kv head takes the places [s per, (s + 1) per): equal
// shares whatever the lengths are, with no tail of workgroups that start late (32 sequences of 8192 rows cut
// into chunks of their own: 580 workgroups for 512 places, 3.6 TB/s against 4.6).  The lead is what another
// sequence costs a share, whose loads start anew (without it 10 us of 40 at 8 sequences of 200 to 16000
// rows, five tokens).  The part of sequence b in share s has the slot s + b among the partials: along the line
// s + b only grows, so the slots are distinct, at most target + B - 1.  Every wave works the line out from the
// lengths, 64 sequences at a time (the first 64 are read once and stay in registers).
struct PagedLine {
  int n0, end0;  // rows of sequence lane (of the first 64; at least 0), and the place behind it
  int total;     // places (their number fits: the host's check)
  int per;       // places of a share
  static __device__ __forceinline__ int places(int rows) {
    return rows > 0 ? (rows + kPagedUnit - 1) / kPagedUnit + kPagedLead : 0;
  }
  __device__ __forceinline__ PagedLine(const PagedBatch& s, int target) {
    const int lane = threadIdx.x & 63;
    n0 = lane < s.B ? max(paged_rows(s, lane), 0) : 0;
    end0 = wave_scan(places(n0));
    total = __builtin_amdgcn_readlane(end0, 63);
    for (int b0 = 64; b0 < s.B; b0 += 64)
      total += __builtin_amdgcn_readlane(wave_scan(places(rows(s, b0 + lane))), 63);
    per = max(1, (total + target - 1) / target);
  }
  __device__ __forceinline__ int rows(const PagedBatch& s, int b) const {  // b = lane + a multiple of 64
    return b < 64 ? n0 : b < s.B ? max(paged_rows(s, b), 0) : 0;
  }
  // the places behind the sequences of a group of 64 (base: those of the groups before)
  __device__ __forceinline__ int ends(const PagedBatch& s, int b0, int base, int n) const {
    return b0 == 0 ? end0 : base + wave_scan(places(n));
  }
  // the shares that hold parts of sequence b: the slot of the first, and how many
  __device__ __forceinline__ void parts(const PagedBatch& s, int b, int& slot, int& n) const {
    const int lane = threadIdx.x & 63;
    int base = 0, end = end0, r = n0;
    for (int b0 = 0; b0 <= b; b0 += 64) {
      if (b0) base = __builtin_amdgcn_readlane(end, 63);
      r = rows(s, b0 + lane);
      end = ends(s, b0, base, r);
    }
    const int u = places(__builtin_amdgcn_readlane(r, b & 63)), after = __builtin_amdgcn_readlane(end, b & 63);
    const int first = (after - u + kPagedLead) / per;  // the share of its first row
    slot = first + b;
    n = u == 0 ? 0 : (after - 1) / per - first + 1;
  }
  // the sequence at a place: its rows n and the place of its first row
  __device__ __forceinline__ void find(const PagedBatch& s, int place, int& b, int& n, int& first) const {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b0 = 0; b0 < s.B; b0 += 64) {
      const int r = rows(s, b0 + lane), end = ends(s, b0, base, r);
      const unsigned long long at = __ballot(place < end);
      if (at) {
        const int l = __builtin_amdgcn_readfirstlane(__ffsll(at) - 1);
        b = b0 + l;
        n = __builtin_amdgcn_readlane(r, l);
        first = __builtin_amdgcn_readlane(end, l) - places(n) + kPagedLead;
        return;
      }
      base = __builtin_amdgcn_readlane(end, 63);
    }
  }
};

// The scale s, and s log2 e and log2 e / s as the exponents take them
struct PagedScale {
  double s;
  float sl2, c0;
};

// Four consecutive columns c .. c+3 of a row of d, zeros beyond d; vec: the row starts at an 8-byte
// boundary
__device__ __forceinline__ bf16x4 ld4_cols(const bf16* row, int c, int d, bool vec) {
  if (vec && c + 4 <= d) return *reinterpret_cast<const bf16x4*>(row + c);
  bf16x4 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = c + e < d ? row[c + e] : (bf16)0.f;
  return x;
}

// Partials of the sequences' parts, slot-major; tokens of the pass Lp, columns t Gs + g
struct PagedPartials {
  float* a;  // [slots][Hkv][Lp][W]      sum_j P_tj w_j
  float* m;  // [slots][Hkv][Lp*Gs]      running max (log2 domain); NaN: a page id outside the pool
  float* l;  // [slots][Hkv][Lp*Gs]      running sum
  float* o;  // [slots][Hkv][Lp*Gs][W]   unnormalised output
};

// V' tile of 32 rows in LDS as the direct loads write it: W / 8 chunks of 16 bytes a row, chunk c of
// row r at c ^ (r & 7) for rows of 128 and 256 bytes; rows of 160 and 192 bytes fall on different
// banks by themselves.
template <int W>
struct PagedSmem {
  static constexpr bool kSwz = W == 64 || W == 128;
  union {
    bf16 v[4][2][32 * W + 64];  // per wave, double buffered (the last tile's transposing reads of W = 80 end 32 bytes behind it)
    struct {
      float so[4][32][W + 4];  // per wave: the columns of O^T (of one column tile at a time)
      float m[4][32], l[4][32];
    } fin;
  } u;
  float nn[4][32];  // per wave: squared norms of the tile's keys
  int bad[4];
};

// MFMA A operand of 16 rows from row0 and columns col0 + lane % 32 of a V' tile (lds_tr_a of
// lucid_common.h for the row widths of a page)
template <int W>
__device__ __forceinline__ bf16x8 paged_tr_a(const bf16* tile, int row0, int col0) {
  typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
  if constexpr (PagedSmem<W>::kSwz) {
    return lds_tr_a<W / 8>(tile, row0, col0);
  } else {
    const int lane = threadIdx.x & 63, s = lane & 15;
    const int col = col0 + 16 * ((lane >> 4) & 1) + 4 * (s & 3);
    const int r1 = row0 + 4 * (lane >> 5) + (s >> 2);
    const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(tile + r1 * W + col));
    const bf16x4 v2 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(tile + (r1 + 8) * W + col));
    return bf16x8{v1[0], v1[1], v1[2], v1[3], v2[0], v2[1], v2[2], v2[3]};
  }
}

// Grid (target, Hkv).  As lucid_decode_split_kernel: each wave sweeps its own 32-row tiles of a
// sequence's part of the share, one MFMA score tile S^T[j][c] = K_j . X_c of the columns c = t (Gs + 1) + i (query head
// g0 + i of token t, its key at i = Gs), then O^T[d][c] += w^T[d][j] p^T[j][c].  p enters the second
// product as a bf16 pair (hi + lo, 2^-17), since V' is returned in fp32 and one bf16 term of P
// would be seen in it.  So would that pair's rounding where the coupling is as large as V' itself: with keys so alike
// that V' is 17 to 33 times V, V' is off by 1.8e-6 to 2.7e-6 of its norm (fp32 throughout: 0.7e-6 to 1.2e-6), with
// independent keys by 6e-8.  A third term would take half as many products again.  Page ids reach registers two tiles ahead, rows one.  Columns of the NCT
// 32-column tiles: Lp (Gs + 1) <= 32 NCT.
// Memory bounds it: 131072 rows of 8 kv heads of 128 columns (537 MB) in 90 us, 6.0 TB/s with nothing read
// twice by the counters.  At 32 sequences of up to 3500 rows it takes 14 us for 27 MB: the lengths, a page
// id, a row, each waiting for the one before, take 7 of them.
template <int W, int NCT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NCT > 1 ? (W <= 64 ? 2 : 1) : (W <= 64 ? 3 : 2)))) void
lucid_paged_split_kernel(const bf16* __restrict__ q, Strides qs, const bf16* __restrict__ kn, Strides kns, int vec,
                         PagedPool kp, PagedPool vp, PagedBatch seq, int target, int Hkv, int Lp, PagedScale factor, float eps,
                         int d, PagedPartials part, int Gs, int Gt, int g0) {
  constexpr int NKS = W / 16, NDT = (W + 31) / 32, CPR = W / 8, NST = 32 * CPR / 64;
  __shared__ __attribute__((aligned(16))) PagedSmem<W> sm;
  const int h = blockIdx.y;
  const PagedLine line(seq, target);
  const int end = min(line.total, ((int)blockIdx.x + 1) * line.per);
  int b = 0, next = 0;
  for (int place = blockIdx.x * line.per; place < end; place = next) {
  int rows = 0, first = 0;
  line.find(seq, place, b, rows, first);
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // what follows from it is worked out here, not kept in registers across the sequences
  const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, l32 = lane & 31;
  next = first + (rows + kPagedUnit - 1) / kPagedUnit;
  // (a share can hold more rows than 32 bits count, a sequence cannot)
  const int j0 = max(place - first, 0) * kPagedUnit, j1 = end >= next ? rows : (end - first) * kPagedUnit;
  if (j1 <= j0) break;  // the share ends in the sequence's lead
  const float sl2 = factor.sl2, c0 = factor.c0, dn = (float)d;

  const int32_t* tbl = seq.table + b * seq.tstride;
  const int ntile = (j1 - j0 + 31) / 32;  // tiles of the part; wave w takes w, w + 4, ...
  bool bad = false;
  // this lane's row of tile t (rows beyond the part: its last row, masked below)
  auto row_of = [&](int t) { return min(j0 + 32 * t + l32, j1 - 1); };
  auto page_id = [&](int t) { return tbl[page_of(seq, row_of(t))]; };
  unsigned koff, voff;  // of this lane's row
  auto locate = [&](int t, int id) {
    const int j = row_of(t);
    if ((unsigned)id >= (unsigned)seq.P) {
      bad = true;
      id = 0;
    }
    const unsigned in = j - page_of(seq, j) * seq.page;
    koff = id * kp.page + h * kp.head + in * kp.row;
    voff = id * vp.page + h * vp.head + in * vp.row;
  };
  bf16x8 kcur[NKS], knx[NKS];  // this tile's and the next tile's key rows
  auto kload = [&](bf16x8* dst) {
    const bf16* r = paged_at(kp, koff);
#pragma unroll
    for (int st = 0; st < NKS; ++st) dst[st] = ld8(r + 16 * st + 8 * g);
  };
  auto vstage = [&](bf16* dst) {  // 32 V' rows into this wave's buffer
#pragma unroll
    for (int i = 0; i < NST; ++i) {
      const int qq = i * 64 + lane, r = qq / CPR;
      int c = qq % CPR;
      if constexpr (PagedSmem<W>::kSwz) c ^= r & 7;
      const bf16* src = paged_at(vp, __shfl((int)voff, r, 64)) + c * 8;
      __builtin_amdgcn_global_load_lds(src, dst + i * 512, 16, 0, kPagedOnce);
    }
  };
  // the first pages' ids, then the new tokens' rows, then the first tile: each wait covers the next loads
  int it = 0, id0 = 0, idn = 0;
  if (w < ntile) id0 = page_id(w);
  if (w + 4 < ntile) idn = page_id(w + 4);
  // B operand: column 32 ct + l32 of X^T (k = d), zero for the padding columns
  bool valid[NCT], isq[NCT];
  bf16x8 xb[NCT][NKS];
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    const int col = 32 * ct + l32, tok = col / (Gs + 1), hi = col - tok * (Gs + 1);
    valid[ct] = tok < Lp;
    isq[ct] = valid[ct] && hi < Gs;
    const int64_t t = seq.done + tok;
    const bf16* x = isq[ct] ? q + b * qs.b + (h * Gt + g0 + hi) * qs.h + t * qs.t : kn + b * kns.b + h * kns.h + t * kns.t;
#pragma unroll
    for (int st = 0; st < NKS; ++st) {
      bf16x8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (bf16)0.f;
      if (valid[ct]) {
        const bf16x4 a = ld4_cols(x, 16 * st + 8 * g, d, vec), c = ld4_cols(x, 16 * st + 8 * g + 4, d, vec);
        v = bf16x8{a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3]};
      }
      xb[ct][st] = v;
    }
  }
  if (w < ntile) {
    locate(w, id0);
    kload(kcur);
    vstage(sm.u.v[w][0]);
  }
  float c1[NCT];  // of the key columns: s log2 e / rms
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    float nt = 0.f;
#pragma unroll
    for (int st = 0; st < NKS; ++st)
#pragma unroll
      for (int e = 0; e < 8; ++e) nt = fmaf((float)xb[ct][st][e], (float)xb[ct][st][e], nt);
    nt = wave_sum32(nt);  // both lane halves
    c1[ct] = sl2 * rsqrtf(nt / dn + eps);
  }
  f32x16 oacc[NCT][NDT];
  float m[NCT], l[NCT];
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    m[ct] = PAGED_NEG;
    l[ct] = 0.f;
#pragma unroll
    for (int t = 0; t < NDT; ++t) oacc[ct][t] = zero16();
  }

  for (int t = w; t < ntile; t += 4, ++it) {
    const int cur = it & 1;
    const bool more = t + 4 < ntile;
    if (more) {
      locate(t + 4, idn);
      if (t + 8 < ntile) idn = page_id(t + 8);
      kload(knx);
      vstage(sm.u.v[w][cur ^ 1]);
      asm volatile("" ::: "memory");  // the loads stay before the wait that counts them
    }
    const int jb = j0 + 32 * t;
    f32x16 scs[NCT];
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) scs[ct] = zero16();
    float nn = 0.f;
#pragma unroll
    for (int st = 0; st < NKS; ++st) {
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) scs[ct] = mfma32(kcur[st], xb[ct][st], scs[ct]);
#pragma unroll
      for (int e = 0; e < 8; ++e) nn = fmaf((float)kcur[st][e], (float)kcur[st][e], nn);
    }
    nn = wave_sum32(nn);
    if (g == 0) sm.nn[w][l32] = rsqrtf(nn / dn + eps);
    float nr[16];
    lds_rows16(&sm.nn[w][0], g, nr);
    bf16x8 ph[NCT][2], pl[NCT][2];
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) {
      f32x16& sc = scs[ct];
      // online max of the query columns (lazy: rescale only when a row grows by 2^8)
      float mx = PAGED_NEG;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (jb + drow(e, g) < j1) mx = fmaxf(mx, sc[e] * sl2);
      mx = isq[ct] ? wave_max32(mx) : PAGED_NEG;
      if (__builtin_amdgcn_ballot_w64(mx > m[ct] + 8.0f)) {
        const float mnew = fmaxf(m[ct], mx);
        const float al = __builtin_amdgcn_exp2f(m[ct] - mnew);
        m[ct] = mnew;
        l[ct] *= al;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int e = 0; e < 16; ++e) oacc[ct][dt][e] *= isq[ct] ? al : 1.f;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool ok = jb + drow(e, g) < j1 && valid[ct];
        const float arg = isq[ct] ? fmaf(sc[e], sl2, -m[ct]) : fmaf(c1[ct] * nr[e], sc[e], -c0);
        const float p = ok ? __builtin_amdgcn_exp2f(arg) : 0.f;
        if (isq[ct]) l[ct] += p;
        sc[e] = p;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        ph[ct][k] = pack_b(sc, k);
        pl[ct][k] = pack_lo(sc, k, ph[ct][k]);
      }
    }
    // this tile's V' rows have landed once at most the next tile's loads are in flight (its page
    // ids came before them)
    if (more)
      dma_wait_but<NKS + NST>();
    else
      dma_wait();
    asm volatile("" ::: "memory");
    const bf16* vt = sm.u.v[w][cur];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const bf16x8 va = paged_tr_a<W>(vt, 16 * k, dt * 32);
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) {
          oacc[ct][dt] = mfma32(va, ph[ct][k], oacc[ct][dt]);
          oacc[ct][dt] = mfma32(va, pl[ct][k], oacc[ct][dt]);
        }
      }
    }
    if (more) {
#pragma unroll
      for (int st = 0; st < NKS; ++st) kcur[st] = knx[st];
    }
  }
  // the four waves' columns merged, one column tile at a time
  const unsigned long long anybad = __ballot(bad);
  if (lane == 0) sm.bad[w] = anybad != 0;
  const int64_t at = (int64_t)(blockIdx.x + b) * Hkv + h;
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    const float lw = wave_sum32(l[ct]);
    __syncthreads();  // every wave is done with the staging buffers (the first tile's columns)
    if (valid[ct]) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; e += 4)  // four rows of the tile side by side
          if (32 * dt + drow(e, 0) < W)
            *reinterpret_cast<f32x4*>(&sm.u.fin.so[w][l32][32 * dt + drow(e, g)]) =
                f32x4{oacc[ct][dt][e], oacc[ct][dt][e + 1], oacc[ct][dt][e + 2], oacc[ct][dt][e + 3]};
      if (isq[ct] && g == 0) {
        sm.u.fin.m[w][l32] = m[ct];
        sm.u.fin.l[w][l32] = lw;
      }
    }
    __syncthreads();
    const bool poison = sm.bad[0] | sm.bad[1] | sm.bad[2] | sm.bad[3];
    // W / 4 lanes a column, two or four columns a wave
    constexpr int CGP = W == 64 ? 16 : 32, CPW = 64 / CGP;
    const int cg = lane % CGP;
#pragma unroll 1
    for (int cl = w * CPW + lane / CGP; cl < 32; cl += 4 * CPW) {
      const int t = (32 * ct + cl) / (Gs + 1), gg = 32 * ct + cl - t * (Gs + 1);
      if (t >= Lp) break;
      if (cg >= W / 4) continue;
      const bool key = gg == Gs;
      float mw[4], lt = 0.f, mn = PAGED_NEG;
#pragma unroll
      for (int ww = 0; ww < 4; ++ww) {
        mw[ww] = sm.u.fin.m[ww][cl];
        mn = fmaxf(mn, mw[ww]);
      }
      f32x4 ot = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ww = 0; ww < 4; ++ww) {
        const float al = key ? 1.f : __builtin_amdgcn_exp2f(mw[ww] - mn);
        lt = fmaf(sm.u.fin.l[ww][cl], al, lt);
        const f32x4 x = *reinterpret_cast<const f32x4*>(&sm.u.fin.so[ww][cl][4 * cg]);
#pragma unroll
        for (int j = 0; j < 4; ++j) ot[j] = fmaf(x[j], al, ot[j]);
      }
      const int64_t pi = at * (Lp * Gs) + t * Gs + gg;
      *reinterpret_cast<f32x4*>((key ? part.a + (at * Lp + t) * W : part.o + pi * W) + 4 * cg) = ot;
      if (cg == 0 && !key) {
        part.m[pi] = poison ? __builtin_nanf("") : mn;
        part.l[pi] = lt;
      }
    }
  }
  if (next < end) __syncthreads();  // the columns are read before the next sequence's rows come
  }
}

// The combine kernel's workgroup: CGP lanes (W / 4 of them, 4 columns each) for every token and slice of
// the parts.  One token of 32 sequences takes 20 us in workgroups of 256 and 25 in those of 512 (five tokens 44 in
// 512, 57 in 1024): more slices wait for one another.
template <int LM>
constexpr int paged_threads() {
  return LM == 1 ? 256 : 512;
}

// Grid (B Hkv, Gs): workgroup (sequence, kv head, query head g0 + g), for the Lp <= LM tokens of the
// pass.  Merges the parts of each token (a slice of them per lane group, the slices through LDS), solves the new
// tokens in order (a column group needs only its own columns), writes the outputs; the g = 0 workgroups of
// the first group of query heads append (k_t, v'_t).  A slot without a sequence gets zeros; one whose table
// names a page outside the pool, or that has no room for the new rows, gets NaN, and nothing is appended to
// it.  What bounds it is the chain of dependent loads (lengths, partials) and three barriers: 6.5 us for one
// sequence of 300 rows, 7.4 for 32, 10.2 at five tokens of 8 sequences (19.7 when every lane held all tokens
// of its columns, most of it in reductions over lanes).
template <int W, int LM>
__global__ __launch_bounds__(paged_threads<LM>()) void lucid_paged_combine_kernel(
    const bf16* __restrict__ q, Strides qs, const bf16* __restrict__ kn, Strides kns, const bf16* __restrict__ vn,
    Strides vns, int vec, int ovec, PagedPool kp, PagedPool vp, PagedBatch seq, int target, bf16* __restrict__ o, Strides os,
    float* __restrict__ vp_new, int Hkv, int Lp, PagedScale factor, float eps, int d, PagedPartials part, int Gs, int Gt,
    int g0, int append) {
  constexpr int CG = W / 4, CGP = W == 64 ? 16 : 32, NT = paged_threads<LM>(), NG = NT / CGP, SL = NG / LM;
  static_assert(SL >= 1, "a lane group for every token");
  constexpr int UN = 4;  // parts whose loads a lane has in flight (8: 57 us for 44 at five tokens of 32 sequences)
  __shared__ float kk[LM][LM], qk[LM][LM];  // k_t . k_u and q_tg . k_u (u <= t)
  __shared__ float pp[LM][LM], ww[LM][LM];  // P_tu (1 / P_tt), and u's weight in token t's softmax
  __shared__ f32x4 os_[NG][CGP], as_[NG][CGP], vps[LM][CGP];
  __shared__ float ms_[NG], ls_[NG], top_[LM];
  __shared__ unsigned krow[LM], vrow[LM];
  __shared__ int bads;
  const int bh = blockIdx.x, g = blockIdx.y;
  const int b = bh / Hkv, h = bh - b * Hkv;
  const int tid = threadIdx.x, grp = tid / CGP, cg = tid % CGP, d0 = 4 * cg;
  const int t = grp % LM, slice = grp / LM;
  const int hq = h * Gt + g0 + g;
  const PagedLine line(seq, target);
  const int rows = paged_rows(seq, b);
  const bf16* kb = kn + b * kns.b + h * kns.h + (int64_t)seq.done * kns.t;
  const bf16* vb = vn + b * vns.b + h * vns.h + (int64_t)seq.done * vns.t;
  const bf16* qb = q + b * qs.b + hq * qs.h + (int64_t)seq.done * qs.t;
  bf16* ob = o + b * os.b + hq * os.h + (int64_t)seq.done * os.t;
  float* vo = vp_new + ((int64_t)bh * seq.L + seq.done) * d;
  const bool write_v = g == 0 && append;
  if (rows < 0) {  // no sequence (zeros), or no room (NaN)
    const float x = rows == -1 ? 0.f : __builtin_nanf("");
    for (int i = tid; i < Lp * d; i += NT) {
      ob[(i / d) * os.t + i % d] = (bf16)x;
      if (write_v) vo[i] = x;
    }
    return;
  }
  int base, nparts;
  line.parts(seq, b, base, nparts);
  if (tid == 0) bads = 0;
  __syncthreads();
  // the pages that the call's new rows go to
  for (int i = tid; i < seq.L; i += NT) {
    const int j = rows - seq.done + i, pg = page_of(seq, j);
    const int id = seq.table[b * seq.tstride + pg];
    if ((unsigned)id >= (unsigned)seq.P) atomicOr(&bads, 1);
    const int u = i - seq.done;
    if (u >= 0 && u < Lp) {
      const unsigned in = j - pg * seq.page;
      krow[u] = id * kp.page + h * kp.head + in * kp.row;
      vrow[u] = id * vp.page + h * vp.head + in * vp.row;
    }
  }
  bf16x4 vrows[LM];  // the new tokens' value rows, for the lanes that solve
  if (grp == 0) {
#pragma unroll
    for (int i = 0; i < LM; ++i)
      if (i < Lp) vrows[i] = ld4_cols(vb + i * vns.t, d0, d, vec);
  }
  // dot products among the new tokens (t, u <= t), 32 lanes a pair, four columns a lane
  const int npair = Lp * (Lp + 1) / 2;
  auto pair = [&](int i, int& x, int& y) {  // i = x (x + 1) / 2 + y
    x = (int)((sqrtf(8.f * i + 1.f) - 1.f) * 0.5f);
    if ((x + 1) * (x + 2) / 2 <= i) ++x;
    if (x * (x + 1) / 2 > i) --x;
    y = i - x * (x + 1) / 2;
  };
  constexpr int PU = LM <= 4 ? 1 : LM == 8 ? 2 : 4;
  for (int i0 = tid / 32; i0 < npair; i0 += PU * (NT / 32)) {
    int ts[PU], us[PU];
    bf16x4 kt[PU], ku[PU], qt[PU];
#pragma unroll
    for (int p = 0; p < PU; ++p) {
      pair(min(i0 + p * (NT / 32), npair - 1), ts[p], us[p]);
      kt[p] = ld4_cols(kb + ts[p] * kns.t, 4 * (tid & 31), d, vec);
      ku[p] = ld4_cols(kb + us[p] * kns.t, 4 * (tid & 31), d, vec);
      qt[p] = ld4_cols(qb + ts[p] * qs.t, 4 * (tid & 31), d, vec);
    }
#pragma unroll
    for (int p = 0; p < PU; ++p) {
      float dkk = 0.f, dqk = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        dkk = fmaf((float)kt[p][e], (float)ku[p][e], dkk);
        dqk = fmaf((float)qt[p][e], (float)ku[p][e], dqk);
      }
      dkk = lanes_sum<32>(dkk);
      dqk = lanes_sum<32>(dqk);
      if ((tid & 31) == 0) {
        kk[ts[p]][us[p]] = dkk;
        qk[ts[p]][us[p]] = dqk;
      }
    }
  }
  // this group's slice of the parts of its token: the key column and the query column (parts beyond the
  // last: the last again, with the weight 0)
  float M = PAGED_NEG, lv = 0.f;
  f32x4 ov = {0.f, 0.f, 0.f, 0.f}, av = {0.f, 0.f, 0.f, 0.f};
  if (t < Lp) {
    const int dc = CG == CGP ? d0 : min(d0, W - 4);
    bool bad = false;
    for (int p0 = slice; p0 < nparts; p0 += UN * SL) {
      float mi[UN], li[UN];
      f32x4 oi[UN], ai[UN];
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        const int64_t at = (int64_t)(base + min(p0 + k * SL, nparts - 1)) * Hkv + h;
        const int64_t i = at * (Lp * Gs) + t * Gs + g;
        mi[k] = part.m[i];
        li[k] = part.l[i];
        oi[k] = *reinterpret_cast<const f32x4*>(part.o + i * W + dc);
        ai[k] = *reinterpret_cast<const f32x4*>(part.a + (at * Lp + t) * W + dc);
      }
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        const bool on = p0 + k * SL < nparts;
        bad |= mi[k] != mi[k];
        const float mn = on ? fmaxf(M, mi[k]) : M;
        const float c = __builtin_amdgcn_exp2f(M - mn), e = on ? __builtin_amdgcn_exp2f(mi[k] - mn) : 0.f;
        const float one = on ? 1.f : 0.f;
        lv = fmaf(lv, c, li[k] * e);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          ov[x] = fmaf(ov[x], c, oi[k][x] * e);
          av[x] = fmaf(ai[k][x], one, av[x]);
        }
        M = mn;
      }
    }
    if (bad) atomicOr(&bads, 1);
  }
  os_[grp][cg] = ov;
  as_[grp][cg] = av;
  if (cg == 0) {
    ms_[grp] = M;
    ls_[grp] = lv;
  }
  __syncthreads();
  const bool poison = bads != 0;
  const float sl2 = factor.sl2, c0 = factor.c0, dn = (float)d;
  // the largest score of a token: over the slices and the new keys
  auto top_of = [&](int x) {
    float m = ms_[x];
#pragma unroll
    for (int s = 1; s < SL; ++s) m = fmaxf(m, ms_[x + s * LM]);
    for (int u = 0; u <= x; ++u) m = fmaxf(m, qk[x][u] * sl2);
    return m;
  };
  // the new tokens among themselves, a pair a lane
  if (tid < npair) {
    int x, u;
    pair(tid, x, u);
    const float m = top_of(x);
    ww[x][u] = __builtin_amdgcn_exp2f(fmaf(qk[x][u], sl2, -m));
    if (u < x) {
      const float rx = rsqrtf(kk[x][x] / dn + eps), ru = rsqrtf(kk[u][u] / dn + eps);
      pp[x][u] = __builtin_amdgcn_exp2f(fmaf(sl2 * rx * ru, kk[x][u], -c0));
    } else {
      // 1 / P_tt; the exponent is the small difference of two terms of size sqrt(d): in fp64, and from the scale in
      // fp64 (from its fp32 value every V' was off by up to 2 sqrt(d) 2^-24: 3.4e-7 at d = 68, now 6e-8)
      const double ms = (double)kk[x][x] / d;
      pp[x][x] = __builtin_amdgcn_exp2f((float)(1.4426950408889634 * (1.0 / factor.s - factor.s * d * ms / (ms + eps))));
      top_[x] = m;
    }
  }
  __syncthreads();
  // the slices of a token merged at its largest score; the sum with the new keys' weights
  float den = 1.f;
  if (slice == 0 && t < Lp) {
    const float m = top_[t];
    den = 0.f;
    ov = av = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < SL; ++s) {
      const float e = __builtin_amdgcn_exp2f(ms_[t + s * LM] - m);
      den = fmaf(ls_[t + s * LM], e, den);
      const f32x4 os4 = os_[t + s * LM][cg], as4 = as_[t + s * LM][cg];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        ov[x] = fmaf(os4[x], e, ov[x]);
        av[x] += as4[x];
      }
    }
    for (int u = 0; u <= t; ++u) den += ww[t][u];
    as_[t][cg] = av;  // (read by this lane alone so far)
  }
  __syncthreads();
  // the new rows in order (this lane's columns): v'_t = (v_t - a_t - sum_{u<t} P_tu w_u) / P_tt
  if (grp == 0) {
    f32x4 held[LM];
#pragma unroll
    for (int x = 0; x < LM; ++x) {
      if (x < Lp) {
        f32x4 v = as_[x][cg];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)vrows[x][j] - v[j];
#pragma unroll
        for (int u = 0; u < x; ++u) {
          const float p = pp[x][u];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = fmaf(-p, held[u][j], v[j]);
        }
        const float inv = pp[x][x];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] *= inv;
          held[x][j] = (float)(bf16)v[j];
        }
        vps[x][cg] = v;
      }
    }
  }
  __syncthreads();
  if (slice == 0 && t < Lp && cg < CG) {
    for (int u = 0; u <= t; ++u) {
      const float es = ww[t][u];
      const f32x4 vu = vps[u][cg];
#pragma unroll
      for (int j = 0; j < 4; ++j) ov[j] = fmaf(es, (float)(bf16)vu[j], ov[j]);
    }
    const float rden = poison ? __builtin_nanf("") : 1.f / den;
    const f32x4 vt = vps[t][cg];
    if (d0 < d) {
      if (ovec) {
        bf16x4 o4;
#pragma unroll
        for (int j = 0; j < 4; ++j) o4[j] = (bf16)(ov[j] * rden);
        *reinterpret_cast<bf16x4*>(ob + t * os.t + d0) = o4;
        if (write_v) *reinterpret_cast<f32x4*>(vo + t * d + d0) = poison ? f32x4{rden, rden, rden, rden} : vt;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (d0 + j >= d) break;
          ob[t * os.t + d0 + j] = (bf16)(ov[j] * rden);
          if (write_v) vo[t * d + d0 + j] = poison ? rden : vt[j];
        }
      }
    }
    if (write_v && !poison) {
      bf16x4 v4;
#pragma unroll
      for (int j = 0; j < 4; ++j) v4[j] = (bf16)(d0 + j < d ? vt[j] : 0.f);
      *reinterpret_cast<bf16x4*>(paged_at(kp, krow[t]) + d0) = ld4_cols(kb + t * kns.t, d0, d, vec);
      *reinterpret_cast<bf16x4*>(paged_at(vp, vrow[t]) + d0) = v4;
    }
  }
}

// Rows t < count_b of k and v' [B][Hkv][T][d] into the pages from row lens[b] on, columns d .. W-1 zero;
// rows whose page id lies outside the pool, or beyond the table, are left out.  A lane per 8 columns of a
// row of both.  Grid (rows Hkv CPR / 256, B).  30011 rows of 8 heads of 128 columns, V' in fp32 (307 MB
// read and written): 55.5 us, 5.5 TB/s, with stores that pass the caches by (58.5 without: a long prompt's pages do
// not stay there until they are read); four prompts of 300 to 2048 rows (4 heads of 68) 5.7 us both ways, which is
// little more than a launch.
template <int W, typename TV>
__global__ __launch_bounds__(256) void lucid_write_pages_kernel(const bf16* __restrict__ k, Strides kst, int kvec,
                                                                const TV* __restrict__ v, Strides vst, int vvec,
                                                                PagedPool kp, PagedPool vp, PagedBatch seq,
                                                                const int32_t* __restrict__ counts, int Hkv, int T,
                                                                int d) {
  constexpr int CPR = W / 8;
  const int b = blockIdx.y;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int c = (int)(idx % CPR) * 8;
  const int64_t th = idx / CPR;
  const int h = (int)(th % Hkv);
  const int64_t t = th / Hkv;
  if (t >= T || (counts && t >= counts[b])) return;
  const int64_t j = seq.lens[b] + t;
  if (seq.lens[b] < 0 || j >= (int64_t)seq.M * seq.page) return;
  const int pg = page_of(seq, (int)j);
  const int id = seq.table[b * seq.tstride + pg];
  if ((unsigned)id >= (unsigned)seq.P) return;
  const unsigned in = (unsigned)j - pg * seq.page;
  const bf16* kr = k + b * kst.b + h * kst.h + t * kst.t;
  const TV* vr = v + b * vst.b + h * vst.h + t * vst.t;
  bf16x8 x, y;
  const bf16x4 a = ld4_cols(kr, c, d, kvec), e = ld4_cols(kr, c + 4, d, kvec);
  x = bf16x8{a[0], a[1], a[2], a[3], e[0], e[1], e[2], e[3]};
  if constexpr (sizeof(TV) == 2) {
    const bf16x4 f = ld4_cols(vr, c, d, vvec), i = ld4_cols(vr, c + 4, d, vvec);
    y = bf16x8{f[0], f[1], f[2], f[3], i[0], i[1], i[2], i[3]};
  } else {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      f32x4 f;
      if (vvec && c + 4 * q + 4 <= d) {
        f = *reinterpret_cast<const f32x4*>(vr + c + 4 * q);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = c + 4 * q + i < d ? vr[c + 4 * q + i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) y[4 * q + i] = (bf16)f[i];
    }
  }
  bf16* kd = paged_at(kp, id * kp.page + h * kp.head + in * kp.row) + c;
  bf16* vd = paged_at(vp, id * vp.page + h * vp.head + in * vp.row) + c;
  __builtin_nontemporal_store(x, reinterpret_cast<bf16x8*>(kd));
  __builtin_nontemporal_store(y, reinterpret_cast<bf16x8*>(vd));
}

// Pages copied within each of several pools of one layout.  Pool pointers and page pairs travel in the
// kernel argument: no upload, and a captured launch keeps them.  Grid (pieces, pairs, pools); a
// workgroup copies one piece of kCopyUnits units U a lane (8 units: 216 us where 4 take 211).  400 pages of 16
// layers' pools (524 MB read, 524 written) take 203 us, 5.2 TB/s, past the caches (through them 214; 100 pages
// 53 and 56; 30 pages 17 both ways, and 15.5 where 12.7 if they are in the cache); 8 pages 3 us, a launch.
constexpr int kCopyPools = 64, kCopyPairs = 256;
constexpr int kCopyUnits = 4;
struct CopyPages {
  char* pool[kCopyPools];
  int src[kCopyPairs], dst[kCopyPairs];
};
template <typename U>
__global__ __launch_bounds__(256) void lucid_copy_pages_kernel(const CopyPages a, int64_t stride, int64_t units) {
  const U* s = reinterpret_cast<const U*>(a.pool[blockIdx.z] + a.src[blockIdx.y] * stride);
  U* t = reinterpret_cast<U*>(a.pool[blockIdx.z] + a.dst[blockIdx.y] * stride);
  const int64_t i0 = (int64_t)blockIdx.x * 256 * kCopyUnits + threadIdx.x;
  U x[kCopyUnits];
#pragma unroll
  for (int i = 0; i < kCopyUnits; ++i)
    if (i0 + 256 * i < units) x[i] = __builtin_nontemporal_load(s + i0 + 256 * i);
#pragma unroll
  for (int i = 0; i < kCopyUnits; ++i)
    if (i0 + 256 * i < units) __builtin_nontemporal_store(x[i], t + i0 + 256 * i);
}

}  // namespace lucid
