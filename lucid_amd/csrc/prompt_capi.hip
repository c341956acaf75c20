// C ABI (declared in include/lucid_amd.h) of the operators around prompts: chunks of new tokens against a paged cache,
// rotary positions and constraints on logits.  The library's second translation unit.
#include <algorithm>
#include <cmath>
#include <string>

#include "constrain.hip"
#include "lucid_prefill.hip"
#include "paged_capi.h"
#include "rotary.hip"

namespace {

// Results of so many bytes pass the 256 MB cache by (past it / through it, us: 131072 tokens of 40 heads of 128 bf16 columns
// turned, 1.3 GB, 489 / 612; constraints on 1700 rows of 32000 bf16 values, 109 MB, 47 / 49, on 8192 with gradient 472 / 479)
constexpr int64_t kPastBytes = 100000000;

constexpr int kSweepShares = 256;  // of the line of a sweep: a workgroup to a CU

struct PrefillWs {
  int2* info;       // [B]
  char* pmat;       // [B][Hkv][panels][kPanelBytes]
  float* y;         // [B][Hkv][256 panels][W]
  lucid::SweepParts part;  // slots of either sweep
  size_t bytes;
};

// Places of a row tile in the line of a sweep, at most
int64_t prefill_len(int page, int max_pages) {
  return ((int64_t)page * max_pages + lucid::kSweepKeys - 1) / lucid::kSweepKeys + lucid::kSweepLead;
}

// Staged tiles of a row tile that is not cut. Where a sequence can have no more (`tiles` of them at most), nothing is cut and
// nothing joined (37 tokens of 16/16 heads of 64 columns behind 300 rows: 35 us, cut and joined 42)
int sweep_whole(int64_t tiles) { return tiles <= 8 ? 8 : 4; }

PrefillWs carve_prefill(void* base, int B, int Hq, int Hkv, int L, int page, int max_pages, int W) {
  const size_t panels = ((size_t)L + lucid::kPanel - 1) / lucid::kPanel;
  size_t off = 0;
  char* p = static_cast<char*>(base);
  auto take = [&](size_t n) {
    char* r = p ? p + off : nullptr;
    off += align256(n);
    return r;
  };
  PrefillWs w{};
  w.info = reinterpret_cast<int2*>(take((size_t)B * 8));
  w.pmat = take((size_t)B * Hkv * panels * lucid::kPanelBytes);
  w.y = reinterpret_cast<float*>(take((size_t)B * Hkv * panels * lucid::kPanel * W * 4));
  // rows of the parts of either sweep: of two row tiles a share, of 64 rows at up to 128 to a kv head
  const int64_t tiles = prefill_len(page, max_pages) - lucid::kSweepLead;
  const size_t rows = tiles <= sweep_whole(tiles) ? 0 : (size_t)2 * kSweepShares * ((int64_t)L * (Hq / Hkv) <= 128 ? 64 : 256);
  w.part.o = reinterpret_cast<float*>(take(rows * W * 4));
  w.part.m = reinterpret_cast<float*>(take(rows * 4));
  w.part.l = reinterpret_cast<float*>(take(rows * 4));
  w.bytes = off;
  return w;
}

bool prefill_sizes_ok(int B, int Hq, int Hkv, int L, int page, int max_pages, int D) {
  return B > 0 && B <= 65535 && Hkv > 0 && Hkv <= 65535 && Hq > 0 && Hq % Hkv == 0 && L > 0 && page > 0 && max_pages > 0 &&
         page_width(D) && (int64_t)page * max_pages <= (1 << 30) && (int64_t)L * (Hq / Hkv) <= (1 << 24) &&
         (int64_t)B * Hkv * (((int64_t)L * (Hq / Hkv) + 63) / 64) <= (1 << 23) &&
         (int64_t)B * Hkv * (((int64_t)L * (Hq / Hkv) + 63) / 64) * prefill_len(page, max_pages) < (1 << 30);
}

struct PrefillCall {
  const bf16 *q, *k, *v;
  const int64_t *qs, *ks, *vs, *os;
  lucid::PagedPool kp, vp;
  lucid::PrefillBatch seq;
  bf16* o;
  PrefillWs ws;
  int Hq, D;
  lucid::PagedScale scale;
  float eps;
  hipStream_t st;
};

template <int W, lucid::Sweep MODE>
int prefill_sweep(const PrefillCall& c, int panel = 0) {
  using lucid::Sweep;
  constexpr bool ATTEND = MODE == Sweep::Attend, LINE = MODE != Sweep::Inner;
  const int GX = ATTEND ? c.Hq / c.seq.Hkv : 1;
  const int panels = (c.seq.L + lucid::kPanel - 1) / lucid::kPanel;
  const int64_t rows = (int64_t)c.seq.L * GX, yrows = (int64_t)panels * lucid::kPanel;
  const int64_t most = prefill_len(c.seq.page, c.seq.M) - lucid::kSweepLead;  // staged tiles of a sequence's keys
  const lucid::SweepGrid grid{GX, ATTEND, kSweepShares, sweep_whole(most)};
  const bf16* x = ATTEND ? c.q : c.k;
  const int64_t* xs = ATTEND ? c.qs : c.ks;
  const int vec = rows_of_4(x, xs, 2), vvec = rows_of_4(c.v, c.vs, 2);
  const int ovec = ATTEND ? c.D % 4 == 0 && rows_of_4(c.o, c.os, 2) : vvec;
  const dim3 blocks = LINE ? dim3(kSweepShares) : dim3((c.seq.L - lucid::kPanel * (panel + 1) + 63) / 64, c.seq.Hkv, c.seq.B);
  auto go = [&](auto form) -> int {
    constexpr int FORM = decltype(form)::value;
    LUCID_LAUNCH_B(ATTEND ? "lucid_prefill_attend_kernel" : LINE ? "lucid_prefill_couple_kernel" : "lucid_prefill_inner_kernel",
                   (lucid::lucid_prefill_sweep_kernel<W, MODE, FORM>), blocks, dim3(512), c.st, x, S(xs), vec, c.v, S(c.vs), c.kp,
                   c.vp, c.seq, grid, panel, c.scale, c.eps, c.D, c.ws.y, yrows, c.o, S(c.os), ovec, c.ws.part);
    if constexpr (LINE) {
      if (most <= grid.whole) return LUCID_OK;
      const int64_t heads = (int64_t)c.seq.B * c.seq.Hkv;
      const int64_t fine = heads * ((rows + 63) / 64), wide = heads * ((rows + 255) / 256);  // row tiles at most
      const int64_t all = std::max(fine * lucid::join_pieces(W, 64), wide * lucid::join_pieces(W, 256));
      const dim3 pieces = FORM == 64    ? dim3((unsigned)fine, lucid::join_pieces(W, 64))
                          : FORM == 256 ? dim3((unsigned)wide, lucid::join_pieces(W, 256))
                                        : dim3((unsigned)std::min<int64_t>(all, 1 << 20), (unsigned)((all + (1 << 20) - 1) >> 20));
      LUCID_LAUNCH("lucid_prefill_join_kernel", (lucid::lucid_prefill_join_kernel<W, ATTEND, FORM>), pieces, c.st, c.v, S(c.vs),
                   vvec, c.seq, grid, c.D, c.ws.y, yrows, c.o, S(c.os), ovec, c.ws.part);
    }
    return LUCID_OK;
  };
  // Up to 128 rows 64 to a row tile (100 tokens of 8/8 heads of 128 columns behind 8000 rows: 68 us, with 256 to a tile 76;
  // 8 x 20 tokens of 32/8 heads behind 4000: 81 and 100), from 513 on 256 (with 64: 2048 tokens of 32/8 heads of 128 columns behind
  // 32768 1.67 -> 2.25 ms; left to the plan, both kinds in one kernel, 1 % slower); between, the plan looks at the tokens.
  if (!LINE || rows <= 128) return go(std::integral_constant<int, 64>{});
  if constexpr (LINE)
    if (rows <= 512) return go(std::integral_constant<int, 0>{});
  return go(std::integral_constant<int, LINE ? 256 : 64>{});
}

template <int W>
int prefill(const PrefillCall& c) {
  const int panels = (c.seq.L + lucid::kPanel - 1) / lucid::kPanel;
  const int64_t yrows = (int64_t)panels * lucid::kPanel;
  LUCID_LAUNCH_B("lucid_prefill_prep_kernel", lucid::lucid_prefill_prep_kernel<W>, dim3(4 * panels, c.seq.Hkv, c.seq.B), dim3(512),
                 c.st, c.k, S(c.ks), (int)rows_of_4(c.k, c.ks, 2), c.kp, c.seq, c.scale, c.eps, c.D, c.ws.pmat, c.o, S(c.os),
                 (int)(c.D % 4 == 0 && rows_of_4(c.o, c.os, 2)), c.Hq / c.seq.Hkv);
  if (int rc = prefill_sweep<W, lucid::Sweep::Couple>(c)) return rc;
  for (int p = 0; p < panels; ++p) {
    LUCID_LAUNCH_B("lucid_prefill_solve_kernel", lucid::lucid_prefill_solve_kernel<W>, dim3((W + 31) / 32, c.seq.Hkv, c.seq.B),
                   dim3(64 * lucid::kPanelBlocks), c.st, c.ws.pmat, panels, p, c.ws.y, yrows, c.vp, c.seq, c.D);
    if (p + 1 < panels)
      if (int rc = prefill_sweep<W, lucid::Sweep::Inner>(c, p)) return rc;
  }
  return prefill_sweep<W, lucid::Sweep::Attend>(c);
}

template <typename T, bool INTER>
int rotary_launch(lucid::RotaryCall c, unsigned blocks, hipStream_t st) {
  // pairs of a unit: as many as 16 bytes hold (of either half, or of adjacent columns), where a head has so many
  constexpr int per = INTER ? 2 : 1, most = 16 / (int)sizeof(T) / per;
  const int half = c.part / 2, stay = c.d - c.part;
  int V = most;
  while (V > 1 && ((half && half < V) || (stay && stay < V))) V /= 2;
  c.stay = stay >= V * per ? V * per : V;
  c.turning = (half + V - 1) / V;
  c.units = c.turning + (stay + c.stay - 1) / c.stay;
  c.per_unit = 1.f / c.units;
  c.per_head = 1.f / (c.units * (c.q.heads + c.k.heads));
  // (stores past the caches want whole lines: with units that overlap, 83 us for 321 MB of rows of 68 fp32 columns)
  const bool past = (int64_t)c.B * c.T * (c.q.heads + c.k.heads) * c.d * (int64_t)sizeof(T) >= kPastBytes &&
                    half * per % (16 / (int)sizeof(T)) == 0 && stay % (16 / (int)sizeof(T)) == 0;
  auto go = [&](auto v) -> int {
    constexpr int N = decltype(v)::value;
    LUCID_LAUNCH("lucid_rotary_kernel",
                 (past ? lucid::lucid_rotary_kernel<T, N, INTER, true> : lucid::lucid_rotary_kernel<T, N, INTER, false>),
                 dim3(blocks), st, c);
    return LUCID_OK;
  };
  if constexpr (most >= 8)
    if (V == 8) return go(std::integral_constant<int, 8>{});
  if constexpr (most >= 4)
    if (V == 4) return go(std::integral_constant<int, 4>{});
  if (V == 2) return go(std::integral_constant<int, 2>{});
  return go(std::integral_constant<int, 1>{});
}

// Workgroups of a row (a misaligned one's first chunk is not whole)
int constrain_segs(int V) { return (V + 7 + lucid::kConstrainSeg - 1) / lucid::kConstrainSeg; }

int check_constrain(const std::string& w, const void* logits, int64_t sb, int64_t st, int R, int Tn, int V, int dtype,
                    const lucid::ConstrainRows& a, bool raw = true) {  // raw: logits are read
  if (dtype != LUCID_DTYPE_BF16 && dtype != LUCID_DTYPE_F32) return fail(w + ": dtype LUCID_DTYPE_BF16 or LUCID_DTYPE_F32");
  if (R < 0 || Tn < 1 || R % Tn) return fail(w + ": R a multiple of the rows of a batch, got R=" + std::to_string(R));
  if (V < 1 || V > 2000000) return fail(w + ": V from 1 to 2000000, got " + std::to_string(V));
  if (sb < 0 || st < 0 || a.hstride < 0 || a.bstride < 0 || a.astride < 0) return fail(w + ": negative strides");
  if (a.N < 0 || (a.N > 0 && R > 0 && !a.history)) return fail(w + ": a history of N tokens a row, N >= 0");
  if (!a.rep && !(a.rep0 > 0.f && std::isfinite(a.rep0))) return fail(w + ": the repetition penalty must be positive and finite");
  if ((!a.pres && !std::isfinite(a.pres0)) || (!a.freq && !std::isfinite(a.freq0))) return fail(w + ": penalties must be finite");
  if (R > 0 && raw && !logits) return fail(w + ": logits are null");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == LUCID_DTYPE_F32 ? 4 : 2)) return fail(w + ": logits are misaligned");
  if ((int64_t)R * constrain_segs(V) * 512 >= ((int64_t)1 << 32)) return fail(w + ": too many rows");
  return LUCID_OK;
}

template <typename T, bool BWD>
int constrain_launch(const T* x, int64_t sb, int64_t st, const T* raw, int64_t rb, int64_t rt, int R, int Tn, int V,
                     lucid::ConstrainRows a, T* out, hipStream_t stream) {
  const int segs = constrain_segs(V);
  const dim3 grid((unsigned)R * segs);
  auto go = [&](auto kernel) -> int {
    LUCID_LAUNCH_B("lucid_constrain_kernel", kernel, grid, dim3(lucid::kConstrainThreads), stream, x, sb, st, raw, rb, rt, Tn,
                   V, segs, a, out);
    return LUCID_OK;
  };
  using lucid::History;
  const bool past = (int64_t)R * V * (int64_t)sizeof(T) >= kPastBytes;
  auto pick = [&](auto h) -> int {
    constexpr History H = decltype(h)::value;
    return past ? go(lucid::lucid_constrain_kernel<T, H, BWD, true>) : go(lucid::lucid_constrain_kernel<T, H, BWD, false>);
  };
  if (a.N == 0) return pick(std::integral_constant<History, History::None>{});
  if constexpr (BWD)
    if (a.N <= lucid::kConstrainThreads * lucid::kConstrainHeld) return pick(std::integral_constant<History, History::Held>{});
  return pick(std::integral_constant<History, History::Counted>{});
}

}  // namespace

extern "C" {

size_t lucid_prefill_paged_workspace_bytes(int B, int Hq, int Hkv, int L, int page_size, int max_pages, int D) {
  if (!prefill_sizes_ok(B, Hq, Hkv, L, page_size, max_pages, D)) return 0;
  return carve_prefill(nullptr, B, Hq, Hkv, L, page_size, max_pages, page_width(D)).bytes;
}

int lucid_prefill_paged(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                        const int64_t* v_strides, void* k_pages, const int64_t* k_page_strides, void* vp_pages,
                        const int64_t* vp_page_strides, const int32_t* page_table, int64_t table_stride,
                        const int32_t* cache_lens, const int32_t* new_lens, void* o, const int64_t* o_strides, void* ws, int B,
                        int Hq, int Hkv, int L, int num_pages, int page_size, int max_pages, int D, double scale, float eps,
                        void* stream) {
  g_last_error.clear();
  if (!page_width(D)) return fail("head_dim must be in [1, 128], got " + std::to_string(D));
  if (!prefill_sizes_ok(B, Hq, Hkv, L, page_size, max_pages, D))
    return fail("lucid_prefill_paged: B, Hq, Hkv, L, page_size and max_pages positive, Hq a multiple of Hkv, B and Hkv at most "
                "65535, at most 2^30 rows a sequence, 2^24 rows of query heads to a kv head, 2^23 tiles of 64 of them in all, and "
                "2^30 pairs of these and of tiles of 128 rows");
  if (num_pages < 1) return fail("lucid_prefill_paged: the pools have no pages");
  if (!q || !q_strides || !k || !k_strides || !v || !v_strides || !o || !o_strides || !page_table || !cache_lens || !ws)
    return fail("lucid_prefill_paged: null argument");
  if (table_stride < 0) return fail("lucid_prefill_paged: negative table stride");
  // (a negative one makes the coupling of unlike keys exp(2/|s|) of a key's own: the solve overflows within a few rows)
  if (!(scale > 0.) || !std::isfinite(scale)) return fail("lucid_prefill_paged: scale must be positive and finite");
  if (int rc = check_ws("ws", ws)) return rc;
  constexpr double kLog2e = 1.4426950408889634;
  const int W = page_width(D);
  PrefillCall c{(const bf16*)q, (const bf16*)k, (const bf16*)v, q_strides, k_strides, v_strides, o_strides, {}, {}, {},
                (bf16*)o, carve_prefill(ws, B, Hq, Hkv, L, page_size, max_pages, W), Hq, D,
                {scale, (float)(scale * kLog2e), (float)(kLog2e / scale)}, eps, static_cast<hipStream_t>(stream)};
  if (int rc = check_pool("k_pages", k_pages, k_page_strides, num_pages, Hkv, page_size, W, &c.kp)) return rc;
  if (int rc = check_pool("vp_pages", vp_pages, vp_page_strides, num_pages, Hkv, page_size, W, &c.vp)) return rc;
  c.seq = lucid::PrefillBatch{page_table, table_stride, cache_lens, new_lens, B, max_pages, num_pages, page_size,
                              page_shift(page_size), L, Hkv, c.ws.info};
  switch (W) {
    case 64: return prefill<64>(c);
    case 80: return prefill<80>(c);
    case 96: return prefill<96>(c);
    default: return prefill<128>(c);
  }
}

int lucid_rotary(const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, int Hq, const void* k,
                 const int64_t* k_strides, void* k_out, const int64_t* k_out_strides, int Hkv, const void* positions,
                 int positions_64, int64_t position_batch_stride, int64_t position_stride, const void* inv_freq,
                 int inv_freq_64, int B, int T, int D, int part, double scale, int interleaved, int inverse, int dtype,
                 void* stream) {
  g_last_error.clear();
  if (dtype != LUCID_DTYPE_BF16 && dtype != LUCID_DTYPE_F32) return fail("lucid_rotary: dtype LUCID_DTYPE_BF16 or LUCID_DTYPE_F32");
  if (B < 0 || T < 0 || Hq < 0 || Hkv < 0) return fail("lucid_rotary: negative size");
  if (D < 1 || D > 2 * lucid::kRotaryPairs || part < 0 || part > D || part % 2)
    return fail("lucid_rotary: head_dim from 1 to 256 and an even part of it, got " + std::to_string(D) + " and " + std::to_string(part));
  if (Hq + (int64_t)Hkv > 2048) return fail("lucid_rotary: at most 2048 heads");
  if (!std::isfinite(scale)) return fail("lucid_rotary: the scale must be finite");
  if (B == 0 || T == 0 || Hq + Hkv == 0) return LUCID_OK;
  if ((Hq && (!q || !q_strides || !q_out || !q_out_strides)) || (Hkv && (!k || !k_strides || !k_out || !k_out_strides)) ||
      !positions || (part && !inv_freq))
    return fail("lucid_rotary: null argument");
  const int64_t size = dtype == LUCID_DTYPE_F32 ? 4 : 2;
  lucid::RotaryCall c{};
  if (reinterpret_cast<uintptr_t>(q) % size || reinterpret_cast<uintptr_t>(k) % size) return fail("lucid_rotary: misaligned operands");
  if (Hq) c.q = {q, S(q_strides), q_out, S(q_out_strides), Hq};
  if (Hkv) c.k = {k, S(k_strides), k_out, S(k_out_strides), Hkv};
  c.pos = positions;
  c.pos64 = positions_64;
  c.pb = position_batch_stride;
  c.pt = position_stride;
  c.freq = inv_freq;
  c.freq64 = inv_freq_64;
  c.B = B;
  c.T = T;
  c.d = D;
  c.part = part;
  c.scale = (float)scale;
  c.dir = inverse ? -1.f : 1.f;
  const int64_t tokens = (int64_t)B * T;
  // Two tokens share a workgroup where there are many.  us with one / two / four: 8 x 2048 tokens of 36 heads of 68 fp32 columns
  // and their gradient 137 / 139 / 152, 131072 of 40 of 128 bf16, half of it turned, 598 / 503 / 491, 65536 interleaved whole
  // 239 / 226 / 242; of kernel with one / two: 32 tokens 3.9 / 4.5, 512 to 2048 the same
  c.tokens = tokens >= 4096 ? lucid::kRotaryTokens : 1;
  const int64_t blocks = (tokens + c.tokens - 1) / c.tokens;
  if (blocks > 0x7fffffff / 256) return fail("lucid_rotary: too many tokens");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == LUCID_DTYPE_F32)
    return interleaved ? rotary_launch<float, true>(c, (unsigned)blocks, st) : rotary_launch<float, false>(c, (unsigned)blocks, st);
  return interleaved ? rotary_launch<bf16, true>(c, (unsigned)blocks, st) : rotary_launch<bf16, false>(c, (unsigned)blocks, st);
}

int lucid_constrain_logits(const void* logits, int64_t batch_stride, int64_t row_stride, int R, int T, int V, int dtype,
                           const int64_t* history, int64_t history_stride, int N, const int32_t* prompt_lens,
                           const float* repetitions, float repetition, const float* presences, float presence,
                           const float* frequencies, float frequency, const float* bias, int64_t bias_stride,
                           const uint32_t* allowed, int64_t allowed_stride, void* out, void* stream) {
  g_last_error.clear();
  const lucid::ConstrainRows a{history, history_stride, N, prompt_lens, repetitions, presences, frequencies, repetition, presence,
                               frequency, bias, bias_stride, allowed, allowed_stride};
  if (int rc = check_constrain("lucid_constrain_logits", logits, batch_stride, row_stride, R, T, V, dtype, a)) return rc;
  if (R == 0) return LUCID_OK;
  if (!out) return fail("lucid_constrain_logits: null output");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == LUCID_DTYPE_F32)
    return constrain_launch<float, false>((const float*)logits, batch_stride, row_stride, nullptr, 0, 0, R, T, V, a, (float*)out, st);
  return constrain_launch<bf16, false>((const bf16*)logits, batch_stride, row_stride, nullptr, 0, 0, R, T, V, a, (bf16*)out, st);
}

int lucid_constrain_logits_bwd(const void* logits, int64_t batch_stride, int64_t row_stride, int R, int T, int V, int dtype,
                               const int64_t* history, int64_t history_stride, int N, const float* repetitions,
                               float repetition, const uint32_t* allowed, int64_t allowed_stride, const void* dout,
                               void* dlogits, void* stream) {
  g_last_error.clear();
  const lucid::ConstrainRows a{history, history_stride, N, nullptr, repetitions, nullptr, nullptr, repetition, 0.f, 0.f, nullptr,
                               0, allowed, allowed_stride};
  if (int rc = check_constrain("lucid_constrain_logits_bwd", logits, batch_stride, row_stride, R, T, V, dtype, a, N > 0))
    return rc;
  if (R == 0) return LUCID_OK;
  if (!dout || !dlogits) return fail("lucid_constrain_logits_bwd: null argument");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t sb = (int64_t)T * V;
  if (dtype == LUCID_DTYPE_F32)
    return constrain_launch<float, true>((const float*)dout, sb, V, (const float*)logits, batch_stride, row_stride, R, T, V, a,
                                         (float*)dlogits, st);
  return constrain_launch<bf16, true>((const bf16*)dout, sb, V, (const bf16*)logits, batch_stride, row_stride, R, T, V, a,
                                      (bf16*)dlogits, st);
}

}  // extern "C"
