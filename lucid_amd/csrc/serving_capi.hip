// C ABI of the serving operators (declared in include/lucid_amd.h): paged (K, V') caches and token log
// probabilities.  Part of lucid_capi.hip's translation unit, whose helpers it uses.

namespace {

// Most workgroups of one resident round of the split pass for a kv head
constexpr int kPagedRound = 512;

// Workgroups of one resident round of the split pass: as many as the registers leave place for, one to a CU
// with two column tiles of more than 64 columns, else two.  Both sides at 32 sequences of 8000 rows of 4 kv
// heads, the column tiles of one token and of five of 8 query heads:
//   rows of 128, five tokens: 160 us with 256 workgroups, 177 with 512
//   rows of 64, five tokens:  100 us with 256, 81 with 512
//   rows of 128, one token:   100 us with 512, 112 with 768
// (a third of rows of 64 with one column tile has its place, and takes as long: 51 us with 512 and with 768)
int paged_round(int W, int tiles) { return W > 64 && tiles == 2 ? 256 : kPagedRound; }

// Workgroups of each kv head: one resident round, and no more than there can be units of rows
int paged_target(int B, int Hkv, int64_t cap, int round) {
  const int64_t most = (int64_t)B * ((cap + lucid::kPagedUnit - 1) / lucid::kPagedUnit);
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, round / Hkv));
}

// Query heads of a chunk of a group (at most 31 and their key fill the columns of a score tile), and new
// tokens of a pass: one 32-column tile, or two where the tokens do not fit one.  At 8 query heads and 32
// sequences of up to 3500 rows of 68 columns five tokens take 44 us in one pass of two tiles and 58 in two of
// one; one token takes 20 us with one tile and 30 with two.  The last pass takes what its own tokens need
// (8 tokens as 7 and 1: 75 us, 84 with two tiles for the one).
int paged_heads(int G) {
  const int chunks = (G + 30) / 31;
  return (G + chunks - 1) / chunks;
}
int paged_tiles(int Gs, int L) { return L > std::min(32 / (Gs + 1), lucid::kPagedMaxTokens) ? 2 : 1; }
int paged_pass(int Gs, int L) {
  return std::min(L, std::min(32 * paged_tiles(Gs, L) / (Gs + 1), lucid::kPagedMaxTokens));
}

lucid::PagedPartials carve_paged(void* base, int64_t slots, int Hkv, int Gs, int Lp, int W, size_t* bytes) {
  const size_t n = (size_t)slots * Hkv * Lp;
  size_t off = 0;
  char* p = static_cast<char*>(base);
  auto take = [&](size_t floats) {
    float* r = reinterpret_cast<float*>(p ? p + off : nullptr);
    off += align256(floats * 4);
    return r;
  };
  lucid::PagedPartials part;
  part.a = take(n * W);
  part.m = take(n * Gs);
  part.l = take(n * Gs);
  part.o = take(n * Gs * W);
  if (bytes) *bytes = off;
  return part;
}

// The places of the line of sequences, and those of a share behind its end for every workgroup (the shares are rounded
// up, and a share's end is worked out before it is cut to the line's), are counted in 32 bits.
bool paged_sizes_ok(int B, int Hq, int Hkv, int L, int page, int max_pages, int D) {
  return B > 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && L > 0 && page > 0 && max_pages > 0 && page_width(D) &&
         (int64_t)page * max_pages <= (1 << 30) && (int64_t)B * Hkv <= (1 << 22) && B <= (1 << 20) && Hkv <= 65535 &&
         B * (((int64_t)page * max_pages + lucid::kPagedUnit - 1) / lucid::kPagedUnit + lucid::kPagedLead) <
             ((int64_t)1 << 31) - 2 * kPagedRound;
}

struct PagedCall {
  const void *q, *k, *v;
  const int64_t *qs, *ks, *vs, *os;
  lucid::PagedPool kp, vp;
  lucid::PagedBatch seq;
  void *o, *ws;
  float* vp_new;
  int Hq, Hkv, D;
  lucid::PagedScale scale;
  float eps;
  hipStream_t st;
};

template <int W, int LM>
int paged_combine(const PagedCall& c, int vec, const lucid::PagedBatch& seq, int target, int Lp,
                  const lucid::PagedPartials& part, int Gs, int g0, int gc) {
  // whole groups of 4 columns at 8-byte boundaries of o and 16-byte boundaries of vp_new
  const int ovec = c.D % 4 == 0 && rows_of_4(c.o, c.os, 2) && !misaligned16(c.vp_new);
  LUCID_LAUNCH_B("lucid_paged_combine_kernel", (lucid::lucid_paged_combine_kernel<W, LM>), dim3(seq.B * c.Hkv, gc),
                 dim3(lucid::paged_threads<LM>()), c.st, (const bf16*)c.q, S(c.qs), (const bf16*)c.k, S(c.ks),
                 (const bf16*)c.v, S(c.vs), vec, ovec, c.kp, c.vp, seq, target, (bf16*)c.o, S(c.os), c.vp_new, c.Hkv, Lp, c.scale,
                 c.eps, c.D, part, gc, c.Hq / c.Hkv, g0, g0 == 0 ? 1 : 0);
  return LUCID_OK;
}

template <int W>
int paged_decode(const PagedCall& c) {
  const int G = c.Hq / c.Hkv, Gs = paged_heads(G), L = c.seq.L;
  const int most = paged_pass(Gs, L);
  // (rows at boundaries of 4 elements: 20.5 us where value by value takes 22.4, at five tokens 43 and 61)
  const int vec = rows_of_4(c.q, c.qs, 2) && rows_of_4(c.k, c.ks, 2) && rows_of_4(c.v, c.vs, 2);
  lucid::PagedBatch seq = c.seq;
  for (int t0 = 0; t0 < L; t0 += most) {
    const int Lp = std::min(most, L - t0), tiles = paged_tiles(Gs, Lp);
    const int target = paged_target(c.seq.B, c.Hkv, (int64_t)c.seq.M * c.seq.page, paged_round(W, tiles));
    seq.done = t0;
    for (int g0 = 0; g0 < G; g0 += Gs) {
      const int gc = std::min(Gs, G - g0);  // query heads of this chunk
      const lucid::PagedPartials part = carve_paged(c.ws, target + c.seq.B, c.Hkv, gc, Lp, W, nullptr);
      const dim3 grid(target, c.Hkv);
      if (tiles == 2)
        LUCID_LAUNCH("lucid_paged_split_kernel", (lucid::lucid_paged_split_kernel<W, 2>), grid, c.st, (const bf16*)c.q,
                     S(c.qs), (const bf16*)c.k, S(c.ks), vec, c.kp, c.vp, seq, target, c.Hkv, Lp, c.scale, c.eps, c.D, part, gc,
                     G, g0);
      else
        LUCID_LAUNCH("lucid_paged_split_kernel", (lucid::lucid_paged_split_kernel<W, 1>), grid, c.st, (const bf16*)c.q,
                     S(c.qs), (const bf16*)c.k, S(c.ks), vec, c.kp, c.vp, seq, target, c.Hkv, Lp, c.scale, c.eps, c.D, part, gc,
                     G, g0);
      // lane groups for the next 1, 4, 8 or 16 tokens: the instance of 4 takes 25 us of a call of one token where
      // that of 1 takes 20, that of 16 takes 52 where that of 4 takes 45 at four tokens, 46 where that of 8
      // takes 43 at five
      const int rc = Lp == 1   ? paged_combine<W, 1>(c, vec, seq, target, Lp, part, gc, g0, gc)
                     : Lp <= 4 ? paged_combine<W, 4>(c, vec, seq, target, Lp, part, gc, g0, gc)
                     : Lp <= 8 ? paged_combine<W, 8>(c, vec, seq, target, Lp, part, gc, g0, gc)
                               : paged_combine<W, lucid::kPagedMaxTokens>(c, vec, seq, target, Lp, part, gc, g0, gc);
      if (rc) return rc;
    }
  }
  return LUCID_OK;
}

template <int W>
int write_pages(const void* k, const int64_t* ks, const void* v, const int64_t* vs, int v_f32, const lucid::PagedPool& kp,
                const lucid::PagedPool& vp, const lucid::PagedBatch& seq, const int32_t* counts, int Hkv, int T, int D,
                hipStream_t st) {
  const int64_t blocks = ((int64_t)T * Hkv * (W / 8) + 255) / 256;
  if (blocks > (1 << 23)) return fail("lucid_write_pages: too many rows");
  const dim3 grid((unsigned)blocks, seq.B);
  // (rows at boundaries of 4 elements: 51 us for 30011 rows of 8 heads of 128 columns, value by value 90)
  const int kvec = rows_of_4(k, ks, 2), vvec = rows_of_4(v, vs, v_f32 ? 4 : 2);
  if (v_f32)
    LUCID_LAUNCH("lucid_write_pages_kernel", (lucid::lucid_write_pages_kernel<W, float>), grid, st, (const bf16*)k, S(ks),
                 kvec, (const float*)v, S(vs), vvec, kp, vp, seq, counts, Hkv, T, D);
  else
    LUCID_LAUNCH("lucid_write_pages_kernel", (lucid::lucid_write_pages_kernel<W, bf16>), grid, st, (const bf16*)k, S(ks),
                 kvec, (const bf16*)v, S(vs), vvec, kp, vp, seq, counts, Hkv, T, D);
  return LUCID_OK;
}

// Token log probabilities: workgroups of 256 lanes for rows of up to 8192 values (and what a
// misaligned row's first chunk leaves out), else of 1024 on segments of 32768.  8000 rows of 8184 values take
// 26 us in workgroups of 256 and 86 in those of 1024, 4 rows 3.5 and 5.3; 4000 of 32000 take 49 in those of
// 1024, with no second launch to join four segments.  A workgroup costs nearly the same however few of its lanes hold
// values: 8000 bf16 rows of 2000 take 26 us (7 at the rate of a copy), of 8192 (which an aligned row would fit
// into 256 lanes) 92 (27), of 16000 86 (53), of 32000 97, of 33000 in two segments 182 (109)
int lp_threads(int V) { return V + 7 <= 256 * lucid::kLpLane ? 256 : 1024; }
int lp_segs(int V, bool aligned = false) {
  const int seg = lp_threads(V) * lucid::kLpLane;
  return (int)(((int64_t)V + (aligned ? 0 : 7) + seg - 1) / seg);
}
// whether every row starts at a 16-byte boundary (its first chunk is whole)
bool lp_aligned(const void* logits, int64_t sb, int64_t st, int dtype) {
  const int64_t es = dtype == LUCID_DTYPE_F32 ? 4 : 2;
  return reinterpret_cast<uintptr_t>(logits) % 16 == 0 && sb * es % 16 == 0 && st * es % 16 == 0;
}

lucid::LpOut carve_lp(void* base, int64_t R, int segs, int top, size_t* bytes) {
  lucid::LpOut o{};
  size_t off = 0;
  char* p = static_cast<char*>(base);
  auto take = [&](size_t n) {
    char* r = p ? p + off : nullptr;
    off += align256(n);
    return r;
  };
  if (segs > 1) {
    o.pm = reinterpret_cast<float*>(take((size_t)R * segs * 4));
    o.ps = reinterpret_cast<float*>(take((size_t)R * segs * 4));
    o.pt = reinterpret_cast<float*>(take((size_t)R * segs * 4));
    o.pkey = reinterpret_cast<unsigned long long*>(take((size_t)R * segs * top * 8));
  }
  if (bytes) *bytes = off;
  return o;
}

int check_lp(const char* what, const void* logits, int64_t sb, int64_t st, const int64_t* tokens, int R, int Tn, int V,
             int dtype, float temperature, int top) {
  const std::string w = what;
  if (dtype != LUCID_DTYPE_BF16 && dtype != LUCID_DTYPE_F32) return fail(w + ": dtype LUCID_DTYPE_BF16 or LUCID_DTYPE_F32");
  if (R < 0 || Tn < 1 || R % Tn) return fail(w + ": R a multiple of the rows of a batch, got R=" + std::to_string(R));
  if (V < 1 || V > 2000000) return fail(w + ": V from 1 to 2000000, got " + std::to_string(V));
  if (top < 0 || top > lucid::kLpMaxTop || top > V) return fail(w + ": top from 0 to 64 and at most V, got " + std::to_string(top));
  // (log2 e / temperature too, the factor of the exponents: from 4.24e-39 down it is infinite)
  if (!(temperature > 0.f) || std::isinf(temperature) || std::isinf(LOG2E_F * (1.f / temperature)))
    return fail(w + ": the temperature and its inverse must be positive and finite");
  if (sb < 0 || st < 0) return fail(w + ": negative strides");
  if (R == 0) return LUCID_OK;
  if (!logits || !tokens) return fail(w + ": logits or tokens are null");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == LUCID_DTYPE_F32 ? 4 : 2)) return fail(w + ": logits are misaligned");
  if ((int64_t)R * lp_segs(V) * lp_threads(V) >= ((int64_t)1 << 32)) return fail(w + ": too many rows");
  return LUCID_OK;
}

template <typename T>
int lp_fwd(const void* logits, int64_t sb, int64_t st, const int64_t* tokens, int R, int Tn, int V, int segs, float inv_temp,
           int top, const lucid::LpOut& out, hipStream_t stream) {
  const int nt = lp_threads(V);
  const dim3 grid((unsigned)R * segs);
  if (nt == 256)
    LUCID_LAUNCH("lucid_token_logprobs_kernel",
                 (top ? lucid::lucid_token_logprobs_kernel<T, 256, true> : lucid::lucid_token_logprobs_kernel<T, 256, false>),
                 grid, stream, (const T*)logits, sb, st, Tn, tokens, V, inv_temp, top, segs, out);
  else
    LUCID_LAUNCH_B("lucid_token_logprobs_kernel",
                   (top ? lucid::lucid_token_logprobs_kernel<T, 1024, true> : lucid::lucid_token_logprobs_kernel<T, 1024, false>),
                   grid, dim3(1024), stream, (const T*)logits, sb, st, Tn, tokens, V, inv_temp, top, segs, out);
  if (segs > 1)
    LUCID_LAUNCH("lucid_token_logprobs_merge_kernel", lucid::lucid_token_logprobs_merge_kernel<T>, dim3(R), stream,
                 (const T*)logits, sb, st, Tn, tokens, V, inv_temp, top, segs, out);
  return LUCID_OK;
}

}  // namespace

extern "C" {

int lucid_page_width(int D) { return page_width(D); }

size_t lucid_decode_paged_workspace_bytes(int B, int Hq, int Hkv, int L, int page_size, int max_pages, int D) {
  if (!paged_sizes_ok(B, Hq, Hkv, L, page_size, max_pages, D)) return 0;
  const int W = page_width(D), Gs = paged_heads(Hq / Hkv);
  const int slots = paged_target(B, Hkv, (int64_t)page_size * max_pages, paged_round(64, 1)) + B;
  size_t bytes = 0;
  carve_paged(nullptr, slots, Hkv, Gs, paged_pass(Gs, L), W, &bytes);
  return bytes;
}

int lucid_decode_paged(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                       const int64_t* v_strides, void* k_pages, const int64_t* k_page_strides, void* vp_pages,
                       const int64_t* vp_page_strides, const int32_t* page_table, int64_t table_stride,
                       const int32_t* cache_lens, void* o, const int64_t* o_strides, float* vp_new, void* ws, int B, int Hq,
                       int Hkv, int L, int num_pages, int page_size, int max_pages, int D, double scale, float eps,
                       void* stream) {
  g_last_error.clear();
  if (!page_width(D)) return fail("head_dim must be in [1, 128], got " + std::to_string(D));
  if (!paged_sizes_ok(B, Hq, Hkv, L, page_size, max_pages, D))
    return fail("lucid_decode_paged: B, Hq, Hkv, L, page_size and max_pages positive, Hq a multiple of Hkv, at most 2^30 "
                "rows a sequence, 2^38 in the tables together and 2^22 kv heads in the batch");
  if (num_pages < 1) return fail("lucid_decode_paged: the pools have no pages");
  if (!q || !q_strides || !k || !k_strides || !v || !v_strides || !o || !o_strides || !vp_new || !page_table ||
      !cache_lens || !ws)
    return fail("lucid_decode_paged: null argument");
  if (table_stride < 0) return fail("lucid_decode_paged: negative table stride");
  if (scale == 0.) return fail("lucid_decode_paged: scale must not be 0");
  if (int rc = check_ws("ws", ws)) return rc;
  constexpr double kLog2e = 1.4426950408889634;
  PagedCall c{q, k, v, q_strides, k_strides, v_strides, o_strides, {}, {}, {}, o, ws, vp_new, Hq, Hkv, D,
              {scale, (float)(scale * kLog2e), (float)(kLog2e / scale)}, eps,
              static_cast<hipStream_t>(stream)};
  const int W = page_width(D);
  if (int rc = check_pool("k_pages", k_pages, k_page_strides, num_pages, Hkv, page_size, W, &c.kp)) return rc;
  if (int rc = check_pool("vp_pages", vp_pages, vp_page_strides, num_pages, Hkv, page_size, W, &c.vp)) return rc;
  c.seq = lucid::PagedBatch{page_table, table_stride, cache_lens, B, max_pages, num_pages, page_size, page_shift(page_size), L, 0};
  switch (W) {
    case 64: return paged_decode<64>(c);
    case 80: return paged_decode<80>(c);
    case 96: return paged_decode<96>(c);
    default: return paged_decode<128>(c);
  }
}

int lucid_write_pages(const void* k, const int64_t* k_strides, const void* vprime, const int64_t* vprime_strides,
                      int vprime_f32, void* k_pages, const int64_t* k_page_strides, void* vp_pages,
                      const int64_t* vp_page_strides, const int32_t* page_table, int64_t table_stride,
                      const int32_t* cache_lens, const int32_t* new_lens, int B, int Hkv, int T, int num_pages,
                      int page_size, int max_pages, int D, void* stream) {
  g_last_error.clear();
  if (!page_width(D)) return fail("head_dim must be in [1, 128], got " + std::to_string(D));
  if (B < 0 || T < 0 || B > 65535 || !paged_sizes_ok(1, Hkv, Hkv, 1, page_size, max_pages, D))
    return fail("lucid_write_pages: B in [0, 65535], T >= 0, Hkv, page_size and max_pages positive, at most 2^30 rows a "
                "sequence");
  if (B == 0 || T == 0) return LUCID_OK;
  if (num_pages < 1) return fail("lucid_write_pages: the pools have no pages");
  if (!k || !k_strides || !vprime || !vprime_strides || !page_table || !cache_lens)
    return fail("lucid_write_pages: null argument");
  if (table_stride < 0) return fail("lucid_write_pages: negative table stride");
  const int W = page_width(D);
  lucid::PagedPool kp, vp;
  if (int rc = check_pool("k_pages", k_pages, k_page_strides, num_pages, Hkv, page_size, W, &kp)) return rc;
  if (int rc = check_pool("vp_pages", vp_pages, vp_page_strides, num_pages, Hkv, page_size, W, &vp)) return rc;
  const lucid::PagedBatch seq{page_table, table_stride, cache_lens, B, max_pages, num_pages, page_size, page_shift(page_size), 0, 0};
  auto* run = W == 64 ? write_pages<64> : W == 80 ? write_pages<80> : W == 96 ? write_pages<96> : write_pages<128>;
  return run(k, k_strides, vprime, vprime_strides, vprime_f32 != 0, kp, vp, seq, new_lens, Hkv, T, D,
             static_cast<hipStream_t>(stream));
}

int lucid_copy_pages(int num_pools, void* const* pools, int64_t page_stride_bytes, int64_t page_bytes, int num_pages,
                     int num_copies, const int* src, const int* dst, void* stream) {
  g_last_error.clear();
  if (num_pools < 0 || num_copies < 0 || num_pages < 0 || page_bytes < 0 || page_stride_bytes < page_bytes)
    return fail("lucid_copy_pages: negative size, or pages that overlap");
  if (num_pools == 0 || num_copies == 0) return LUCID_OK;
  if (!pools || !src || !dst) return fail("lucid_copy_pages: null argument");
  try {
    std::vector<unsigned char> used(num_pages);  // 1: read, 2: written
    for (int i = 0; i < num_copies; ++i) {
      if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages)
        return fail("lucid_copy_pages: page " + std::to_string(src[i]) + " -> " + std::to_string(dst[i]) +
                    " outside the pool's " + std::to_string(num_pages));
      if (used[dst[i]] & 2) return fail("lucid_copy_pages: page " + std::to_string(dst[i]) + " is written twice");
      used[src[i]] |= 1;
      used[dst[i]] |= 2;
    }
    for (int i = 0; i < num_copies; ++i)
      if (used[dst[i]] & 1) return fail("lucid_copy_pages: page " + std::to_string(dst[i]) + " is both read and written");
  } catch (const std::exception&) {
    return fail("lucid_copy_pages: out of host memory");
  }
  if (page_bytes == 0) return LUCID_OK;
  uintptr_t bits = (uintptr_t)page_bytes | (uintptr_t)page_stride_bytes;
  for (int i = 0; i < num_pools; ++i) {
    if (!pools[i]) return fail("lucid_copy_pages: pool " + std::to_string(i) + " is null");
    bits |= reinterpret_cast<uintptr_t>(pools[i]);
  }
  // (in 16 bytes a lane 12.7 us for 30 pages of 16 layers, in 4 bytes 13.8; 400 pages 213 and 211, and 764 in bytes)
  const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
  const int64_t units = page_bytes / unit, pieces = (units + 256 * lucid::kCopyUnits - 1) / (256 * lucid::kCopyUnits);
  if (pieces > (1 << 23)) return fail("lucid_copy_pages: pages of more than 2^33 units");
  hipStream_t st = static_cast<hipStream_t>(stream);
  for (int p0 = 0; p0 < num_pools; p0 += lucid::kCopyPools)
    for (int c0 = 0; c0 < num_copies; c0 += lucid::kCopyPairs) {
      lucid::CopyPages a;
      const int np = std::min(lucid::kCopyPools, num_pools - p0), nc = std::min(lucid::kCopyPairs, num_copies - c0);
      std::copy(pools + p0, pools + p0 + np, reinterpret_cast<void**>(a.pool));
      std::copy(src + c0, src + c0 + nc, a.src);
      std::copy(dst + c0, dst + c0 + nc, a.dst);
      const dim3 grid((unsigned)pieces, nc, np);
      if (unit == 16)
        LUCID_LAUNCH("lucid_copy_pages_kernel", lucid::lucid_copy_pages_kernel<u32x4>, grid, st, a, page_stride_bytes, units);
      else if (unit == 4)
        LUCID_LAUNCH("lucid_copy_pages_kernel", lucid::lucid_copy_pages_kernel<uint32_t>, grid, st, a, page_stride_bytes,
                     units);
      else
        LUCID_LAUNCH("lucid_copy_pages_kernel", lucid::lucid_copy_pages_kernel<uint8_t>, grid, st, a, page_stride_bytes,
                     units);
    }
  return LUCID_OK;
}

size_t lucid_token_logprobs_workspace_bytes(int R, int V, int top) {
  if (R < 0 || V < 1 || top < 0) return 0;
  size_t bytes = 0;
  carve_lp(nullptr, R, lp_segs(V), top, &bytes);
  return bytes;
}

int lucid_token_logprobs_fwd(const void* logits, int64_t batch_stride, int64_t row_stride, const int64_t* tokens, int R,
                             int T, int V, int dtype, float temperature, int top, float* logprobs, float* entropy,
                             float* stats, float* top_logprobs, int64_t* top_indices, void* ws, void* stream) {
  g_last_error.clear();
  if (int rc = check_lp("lucid_token_logprobs_fwd", logits, batch_stride, row_stride, tokens, R, T, V, dtype, temperature,
                        top))
    return rc;
  if (R == 0) return LUCID_OK;
  const int segs = lp_segs(V, lp_aligned(logits, batch_stride, row_stride, dtype));
  if (!logprobs || !entropy || (top && (!top_logprobs || !top_indices)) || (segs > 1 && !ws))
    return fail("lucid_token_logprobs_fwd: null output or workspace");
  if (segs > 1)
    if (int rc = check_ws("ws", ws)) return rc;
  lucid::LpOut out = carve_lp(ws, R, segs, top, nullptr);
  out.logprob = logprobs;
  out.entropy = entropy;
  out.stats = reinterpret_cast<lucid::LpStats*>(stats);
  out.top_lp = top_logprobs;
  out.top_idx = top_indices;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return (dtype == LUCID_DTYPE_F32 ? lp_fwd<float> : lp_fwd<bf16>)(logits, batch_stride, row_stride, tokens, R, T, V, segs,
                                                                   1.f / temperature, top, out, st);
}

int lucid_token_logprobs_bwd(const void* logits, int64_t batch_stride, int64_t row_stride, const int64_t* tokens, int R,
                             int T, int V, int dtype, float temperature, int top, const float* stats,
                             const int64_t* top_indices, const float* dlogprobs, const float* dentropy,
                             const float* dtop_logprobs, void* dlogits, void* stream) {
  g_last_error.clear();
  if (int rc = check_lp("lucid_token_logprobs_bwd", logits, batch_stride, row_stride, tokens, R, T, V, dtype, temperature,
                        top))
    return rc;
  if (R == 0) return LUCID_OK;
  if (!stats || !dlogits || (top && !top_indices)) return fail("lucid_token_logprobs_bwd: null argument");
  if (reinterpret_cast<uintptr_t>(dlogits) % (dtype == LUCID_DTYPE_F32 ? 4 : 2))
    return fail("lucid_token_logprobs_bwd: dlogits are misaligned");
  const int per = 256 * lucid::kLpLane;
  const int blocks = (int)(((int64_t)V + 7 + per - 1) / per);
  if ((int64_t)R * blocks * 256 >= ((int64_t)1 << 32)) return fail("lucid_token_logprobs_bwd: too many rows");
  const dim3 grid((unsigned)R * blocks);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const lucid::LpGrads g{dlogprobs, dentropy, dtop_logprobs};
  const auto* z = reinterpret_cast<const lucid::LpStats*>(stats);
  // A gradient of 100 MB or more is not kept in the 256 MB cache for what reads it next.  Forward and backward of 8192
  // rows of 32000 bf16 values 290 -> 274 us, of 4000 147 -> 123, of 1021 of 32003 fp32 ones 84 -> 72.  That is the
  // pair by itself.  With the product that reads the gradient (2048 columns) a step gains nothing: 8192 rows 1042 -> 1047,
  // 4000 557 -> 555, 3000 441 -> 439, 2000 461 -> 461, 1600 (102 MB) 366 -> 367, 1500 350 -> 350; below the rule it would
  // lose 1 %: 1250 332 -> 336, 1000 321 -> 324, 500 200 -> 204.
  const bool past = (int64_t)R * V * (dtype == LUCID_DTYPE_F32 ? 4 : 2) >= 100000000;
  auto go = [&](auto zero, auto kernel) -> int {
    using E = decltype(zero);
    LUCID_LAUNCH("lucid_token_logprobs_bwd_kernel", kernel, grid, st, (const E*)logits, batch_stride, row_stride, T,
                 tokens, V, 1.f / temperature, top, z, top_indices, g, (E*)dlogits, blocks);
    return LUCID_OK;
  };
  using lucid::lucid_token_logprobs_bwd_kernel;
  if (dtype == LUCID_DTYPE_F32)
    return go(0.f, past ? lucid_token_logprobs_bwd_kernel<float, true> : lucid_token_logprobs_bwd_kernel<float, false>);
  return go((bf16)0.f, past ? lucid_token_logprobs_bwd_kernel<bf16, true> : lucid_token_logprobs_bwd_kernel<bf16, false>);
}

int lucid_abi_minor(void) { return 2; }

}  // extern "C"
