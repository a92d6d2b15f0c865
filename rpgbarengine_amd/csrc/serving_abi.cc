// extern "C" entry points of the serving operators (include/rpg_hip.h): checks
// of the callers' arguments, then one enqueue. Nothing here touches the GPU
// before every check has passed.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.h"
#include "edit_rows.h"
#include "paged.h"
#include "rpg_hip.h"
#include "sample_rows.h"

namespace rpg {
namespace {

template <typename F>
auto Guard(F&& f, decltype(f()) fail) -> decltype(f()) {
  try {
    SetLastError("");
    return f();
  } catch (const std::exception& e) {
    SetLastError(e.what());
  } catch (...) {
    SetLastError("unknown exception");
  }
  return fail;
}

int ElementBytes(int32_t type) {
  RPG_CHECK(type == kF32 || type == kF16 || type == kBF16, "element type %d is none of f32 (0), f16 (1), bf16 (30)",
            type);
  return type == kF32 ? 4 : 2;
}

// Byte strides of this size keep every product with a 32-bit count in 64 bits.
constexpr int64_t kMaxStride = int64_t{1} << 31;

// Of a sequence: a kernel's steps may count some thousand past them.
constexpr int32_t kMaxPositions = 1 << 30;

int64_t StrideBytes(const char* what, int64_t elements, int bytes) {
  RPG_CHECK(elements >= -kMaxStride && elements <= kMaxStride, "%s of %lld elements", what, (long long)elements);
  RPG_CHECK(elements * bytes % 16 == 0, "%s of %lld elements is not a multiple of 16 bytes", what,
            (long long)elements);
  return elements * bytes;
}

void CheckPointer(const char* what, const void* p, int align) {
  RPG_CHECK(p != nullptr, "%s is null", what);
  RPG_CHECK(reinterpret_cast<uintptr_t>(p) % align == 0, "%s does not lie at a multiple of %d bytes", what, align);
}

void CheckSizes(int32_t head_dim, int32_t page_size, int32_t n_pages, int32_t n_kv) {
  RPG_CHECK(head_dim == 64 || head_dim == 128, "head_dim %d is neither 64 nor 128", head_dim);
  RPG_CHECK(page_size >= 16 && page_size <= 65536 && (page_size & (page_size - 1)) == 0,
            "page_size %d is not a power of two from 16 to 65536", page_size);
  RPG_CHECK(n_pages >= 1, "a cache of %d pages", n_pages);
  RPG_CHECK(n_kv >= 1, "%d key heads", n_kv);
}

// The strides and sizes of rows of `bytes` bytes an element.
void PageStrides(int64_t page_stride, int64_t head_stride, int64_t row_stride, int32_t head_dim, int32_t page_size,
                 int32_t n_pages, int32_t n_kv, int bytes, paged::Cache* out) {
  out->page_bytes = StrideBytes("page_stride", page_stride, bytes);
  out->head_bytes = StrideBytes("head_stride", head_stride, bytes);
  const int64_t row = StrideBytes("row_stride", row_stride, bytes);
  // positions of a page are addressed by 32-bit offsets; no two of them overlap
  RPG_CHECK(row >= head_dim * bytes && row * page_size < kMaxStride, "row_stride %lld", (long long)row_stride);
  RPG_CHECK((n_kv == 1 || std::abs(out->head_bytes) >= head_dim * bytes) &&
                (n_pages == 1 || std::abs(out->page_bytes) >= head_dim * bytes),
            "head_stride %lld or page_stride %lld is less than a row", (long long)head_stride,
            (long long)page_stride);
  out->row_bytes = static_cast<int32_t>(row);
  out->n_pages = n_pages;
  out->n_kv = n_kv;
  out->page_log2 = __builtin_ctz(static_cast<unsigned>(page_size));
  out->head_dim = head_dim;
}

paged::Cache CacheSizes(const rpg_hip_paged_cache* c) {
  RPG_CHECK(c != nullptr, "the cache is null");
  paged::Cache out;
  const int bytes = ElementBytes(c->type);
  CheckSizes(c->head_dim, c->page_size, c->n_pages, c->n_kv);
  PageStrides(c->page_stride, c->head_stride, c->row_stride, c->head_dim, c->page_size, c->n_pages, c->n_kv, bytes, &out);
  out.type = static_cast<uint32_t>(c->type);
  return out;
}

paged::Cache CacheOf(const rpg_hip_paged_cache* c) {
  paged::Cache out = CacheSizes(c);
  CheckPointer("the cache's k", c->k, 16);
  CheckPointer("the cache's v", c->v, 16);
  out.k = static_cast<char*>(c->k);
  out.v = static_cast<char*>(c->v);
  return out;
}

// A cache of codes; `type`: of the rows.
paged::Cache QuantSizes(const rpg_hip_quant_cache* c, int32_t type, paged::Scales* scales) {
  RPG_CHECK(c != nullptr, "the cache is null");
  paged::Cache out;
  ElementBytes(type);
  RPG_CHECK(c->code == RPG_HIP_I8 || c->code == RPG_HIP_E4M3, "code %d is neither i8 (0) nor e4m3 (1)", c->code);
  CheckSizes(c->head_dim, c->page_size, c->n_pages, c->n_kv);
  PageStrides(c->page_stride, c->head_stride, c->row_stride, c->head_dim, c->page_size, c->n_pages, c->n_kv, 1, &out);
  scales->page_bytes = StrideBytes("scale_page_stride", c->scale_page_stride, 4);
  scales->head_bytes = StrideBytes("scale_head_stride", c->scale_head_stride, 4);
  RPG_CHECK((c->n_kv == 1 || std::abs(c->scale_head_stride) >= c->page_size) &&
                (c->n_pages == 1 || std::abs(c->scale_page_stride) >= c->page_size),
            "scale_head_stride %lld or scale_page_stride %lld is less than a page's positions",
            (long long)c->scale_head_stride, (long long)c->scale_page_stride);
  out.type = static_cast<uint32_t>(type);
  return out;
}

paged::Cache QuantOf(const rpg_hip_quant_cache* c, int32_t type, paged::Scales* scales) {
  paged::Cache out = QuantSizes(c, type, scales);
  CheckPointer("the cache's k", c->k, 16);
  CheckPointer("the cache's v", c->v, 16);
  CheckPointer("the cache's k_scale", c->k_scale, 16);
  CheckPointer("the cache's v_scale", c->v_scale, 16);
  out.k = static_cast<char*>(c->k);
  out.v = static_cast<char*>(c->v);
  scales->k = reinterpret_cast<char*>(c->k_scale);
  scales->v = reinterpret_cast<char*>(c->v_scale);
  return out;
}

paged::Seqs SeqSizes(const rpg_hip_sequences* s, int page_size) {
  RPG_CHECK(s != nullptr, "the sequences are null");
  paged::Seqs out;
  RPG_CHECK(s->n_seqs >= 0 && s->n_tokens >= 0, "%d sequences of %d new tokens", s->n_seqs, s->n_tokens);
  RPG_CHECK(s->pages >= 0 && s->pages <= kMaxPositions / page_size,
            "%d pages of %d positions for a sequence", s->pages, page_size);
  out.n_seqs = s->n_seqs;
  out.n_tokens = s->n_tokens;
  out.capacity = s->pages * page_size;
  return out;
}

paged::Seqs SeqsOf(const rpg_hip_sequences* s, int page_size, bool packed) {
  paged::Seqs out = SeqSizes(s, page_size);
  if (s->n_seqs == 0) return out;
  if (s->pages > 0) CheckPointer("the page table", s->table, 4);
  RPG_CHECK(s->n_seqs == 1 || s->table_stride >= s->pages, "table_stride %lld is less than %d pages",
            (long long)s->table_stride, s->pages);
  RPG_CHECK(s->table_stride <= kMaxStride, "table_stride %lld", (long long)s->table_stride);
  CheckPointer("lens", s->lens, 4);
  if (packed) CheckPointer("starts", s->starts, 4);
  out.table = s->table;
  out.table_stride = s->n_seqs == 1 ? 0 : s->table_stride;
  out.lens = s->lens;
  out.starts = s->starts;
  return out;
}

paged::Rows RowsOf(const char* what, const rpg_hip_rows* r, const paged::Cache& c, int n_tokens, int n_heads,
                   bool written) {
  RPG_CHECK(r != nullptr, "%s is null", what);
  const int bytes = ElementBytes(static_cast<int32_t>(c.type));
  CheckPointer(what, r->data, 16);
  paged::Rows out;
  out.p = static_cast<char*>(r->data);
  out.token_bytes = StrideBytes(what, r->token_stride, bytes);
  out.head_bytes = StrideBytes(what, r->head_stride, bytes);
  if (written) {
    const int64_t row = c.head_dim * bytes;
    RPG_CHECK((n_tokens == 1 || std::abs(out.token_bytes) >= row) && (n_heads == 1 || std::abs(out.head_bytes) >= row),
              "%s: rows that overlap are not written", what);
  }
  return out;
}

// Rows that are written where others are read: those of one token and head lie in
// one place, or else some are overwritten before they are read.
void CheckInPlace(const char* out_is_in, const paged::Rows& out, const paged::Rows& in, int n_tokens, int n_heads) {
  RPG_CHECK(out.p != in.p || ((n_tokens == 1 || out.token_bytes == in.token_bytes) &&
                              (n_heads == 1 || out.head_bytes == in.head_bytes)),
            "%s with other strides", out_is_in);
}

void CheckHeads(const paged::Cache& c, const paged::Seqs& s, int32_t n_heads) {
  RPG_CHECK(n_heads >= c.n_kv && n_heads % c.n_kv == 0, "%d query heads on %d key heads", n_heads, c.n_kv);
  RPG_CHECK(static_cast<int64_t>(n_heads) * std::max(s.n_tokens, s.n_seqs) < (int64_t{1} << 31) - 4096,
            "%d x %d query rows", std::max(s.n_tokens, s.n_seqs), n_heads);
}

int Splits(const paged::Cache& c, const paged::Seqs& s, int32_t n_heads, bool prompt, bool codes, int* least) {
  *least = 0;
  const int bytes = ElementBytes(static_cast<int32_t>(c.type));
  if (codes && prompt) return paged::CodesPromptSplits(s.n_tokens, s.n_seqs, n_heads, c.n_kv, s.capacity);
  if (codes) return paged::CodesDecodeSplits(s.n_seqs, n_heads, c.n_kv, s.capacity, least);
  if (prompt) return paged::PromptSplits(s.n_tokens, s.n_seqs, n_heads, c.n_kv, bytes, s.capacity);
  return paged::DecodeSplits(s.n_seqs, n_heads, c.n_kv, bytes, s.capacity);
}

// Calls without sequences or new tokens have nothing to do.
bool Empty(const paged::Seqs& s, bool packed) { return s.n_seqs == 0 || (packed && s.n_tokens == 0); }

int64_t AttentionWork(const paged::Cache& c, const paged::Seqs& s, int32_t n_heads, bool prompt, bool codes) {
  if (Empty(s, prompt)) return 0;
  const int64_t rows = static_cast<int64_t>(prompt ? s.n_tokens : s.n_seqs) * n_heads;
  int least;
  return paged::WorkBytes(rows, c.head_dim, Splits(c, s, n_heads, prompt, codes, &least));
}

void CheckWork(void* work, int64_t work_bytes, int64_t need) {
  if (need == 0) return;
  CheckPointer("work", work, 16);
  RPG_CHECK(work_bytes >= need, "%lld bytes of work memory, %lld are needed", (long long)work_bytes, (long long)need);
}

// Queries and outputs of a call on a.c and a.s, one for each of n_tokens.
void AttentionRows(paged::AttentionArgs* to, const rpg_hip_rows* q, const rpg_hip_rows* out, int32_t n_tokens,
                   int32_t n_heads, float scale) {
  paged::AttentionArgs& a = *to;
  CheckHeads(a.c, a.s, n_heads);
  a.q = RowsOf("q", q, a.c, n_tokens, n_heads, false);
  a.out = RowsOf("out", out, a.c, n_tokens, n_heads, true);
  CheckInPlace("out is q", a.out, a.q, n_tokens, n_heads);
  RPG_CHECK(scale > 0.0f && std::isfinite(scale), "scale %g is not positive and finite", scale);
  a.n_heads = n_heads;
  a.scale = scale;
}

void AttentionParts(paged::AttentionArgs* a, bool prompt, bool codes, void* work, int64_t work_bytes) {
  a->splits = Splits(a->c, a->s, a->n_heads, prompt, codes, &a->least);
  CheckWork(work, work_bytes, AttentionWork(a->c, a->s, a->n_heads, prompt, codes));
  a->work = static_cast<float*>(work);
}

int32_t Attention(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs, const rpg_hip_rows* q,
                  const rpg_hip_rows* out, int32_t n_heads, float scale, void* work, int64_t work_bytes, void* stream,
                  bool prompt) {
  paged::AttentionArgs a;
  a.c = CacheOf(cache);
  a.s = SeqsOf(seqs, cache->page_size, prompt);
  if (Empty(a.s, prompt)) return 0;
  AttentionRows(&a, q, out, prompt ? a.s.n_tokens : a.s.n_seqs, n_heads, scale);
  AttentionParts(&a, prompt, false, work, work_bytes);
  if (prompt)
    paged::Prompt(a, static_cast<hipStream_t>(stream));
  else
    paged::Decode(a, static_cast<hipStream_t>(stream));
  return 0;
}

int32_t QuantAttention(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs, int32_t type,
                       const rpg_hip_rows* q, const rpg_hip_rows* out, int32_t n_heads, float scale, void* work,
                       int64_t work_bytes, void* stream, bool prompt) {
  paged::CodesAttentionArgs a;
  a.a.c = QuantOf(cache, type, &a.scales);
  a.code = cache->code;
  a.a.s = SeqsOf(seqs, cache->page_size, prompt);
  if (Empty(a.a.s, prompt)) return 0;
  AttentionRows(&a.a, q, out, prompt ? a.a.s.n_tokens : a.a.s.n_seqs, n_heads, scale);
  AttentionParts(&a.a, prompt, true, work, work_bytes);
  if (prompt)
    paged::PromptCodes(a, static_cast<hipStream_t>(stream));
  else
    paged::DecodeCodes(a, static_cast<hipStream_t>(stream));
  return 0;
}

paged::SharedSplits SharedSizes(const paged::Cache& c, const paged::Seqs& s, int32_t n_groups, int32_t n_heads,
                                bool codes, int64_t* bytes) {
  RPG_CHECK(n_groups >= 0, "%d groups", n_groups);
  CheckHeads(c, s, n_heads);
  const paged::SharedSplits n = paged::SplitsOfShared(
      s.n_seqs, n_groups, n_heads, c.n_kv, codes ? 2 : ElementBytes(static_cast<int32_t>(c.type)), s.capacity);
  *bytes = paged::WorkBytes(static_cast<int64_t>(s.n_seqs) * n_heads, c.head_dim, n.prefix + n.own);
  return n;
}

// The groups, splits and work memory of a call whose rows `a` has.
paged::Seqs GroupsOf(const rpg_hip_groups* g, paged::AttentionArgs* a, bool codes, int64_t* prefix_splits, void* work,
                     int64_t work_bytes) {
  RPG_CHECK(g != nullptr, "the groups are null");
  int64_t need;
  const paged::SharedSplits n = SharedSizes(a->c, a->s, g->n_groups, a->n_heads, codes, &need);
  if (g->n_groups > 0) {
    CheckPointer("the groups' starts", g->starts, 4);
    CheckPointer("shared", g->shared, 4);
  }
  CheckWork(work, work_bytes, need);
  a->work = static_cast<float*>(work);
  a->splits = n.prefix + n.own;
  a->least = n.least;
  *prefix_splits = n.prefix;
  paged::Seqs out;
  out.starts = g->starts;
  out.lens = g->shared;
  out.n_seqs = g->n_groups;
  out.n_tokens = a->s.n_seqs;
  out.capacity = a->s.capacity;
  return out;
}

void AppendRows(paged::AppendArgs* to, const rpg_hip_rows* k, const rpg_hip_rows* v, const rpg_hip_rows* q,
                const rpg_hip_rows* q_out, int32_t n_heads, const float* q_norm, const float* k_norm, float eps,
                const float* rope, int64_t rope_rows) {
  paged::AppendArgs& a = *to;
  a.k = RowsOf("k", k, a.c, a.s.n_tokens, a.c.n_kv, false);
  a.v = RowsOf("v", v, a.c, a.s.n_tokens, a.c.n_kv, false);
  if (q != nullptr && q->data != nullptr) {
    CheckHeads(a.c, a.s, n_heads);
    RPG_CHECK(n_heads <= 65536 && a.c.n_kv <= 65536, "%d query heads on %d key heads", n_heads, a.c.n_kv);
    a.q = RowsOf("q", q, a.c, a.s.n_tokens, n_heads, false);
    a.q_out = RowsOf("q_out", q_out, a.c, a.s.n_tokens, n_heads, true);
    CheckInPlace("q_out is q", a.q_out, a.q, a.s.n_tokens, n_heads);
    a.n_heads = n_heads;
  } else {
    RPG_CHECK(a.c.n_kv <= 65536, "%d key heads", a.c.n_kv);
  }
  if (q_norm != nullptr) CheckPointer("q_norm", q_norm, 16);
  if (k_norm != nullptr) CheckPointer("k_norm", k_norm, 16);
  if (rope != nullptr) CheckPointer("rope", rope, 16);
  RPG_CHECK(rope == nullptr || rope_rows >= 0, "%lld rotation rows", (long long)rope_rows);
  RPG_CHECK(eps >= 0.0f, "eps %g", eps);
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.eps = eps;
  a.rope = rope;
  a.rope_rows = rope_rows;
}

// Rows that are written while others are read, `bytes` each: those of one number lie in
// one place, or none of them touches another (two parts of the rows of one matrix may).
void CheckApart(const char* out_overlaps_in, const void* out, int64_t out_stride, const void* in, int64_t in_stride,
                int64_t n_rows, int64_t bytes) {
  const int64_t d = static_cast<int64_t>(reinterpret_cast<uintptr_t>(out) - reinterpret_cast<uintptr_t>(in));
  if (d == 0 || d >= (n_rows - 1) * in_stride + bytes || -d >= (n_rows - 1) * out_stride + bytes) return;
  const bool matrix = n_rows > 1 && out_stride == in_stride;
  const int64_t off = matrix ? (d % out_stride + out_stride) % out_stride : 0;
  RPG_CHECK(matrix && off >= bytes && out_stride - off >= bytes, "%s", out_overlaps_in);
}

// Rows of 4-byte elements that may be given more than once (stride 0).
void CheckList(const char* what, const void* p, int64_t stride) {
  CheckPointer(what, p, 4);
  RPG_CHECK(stride >= 0 && stride <= kMaxStride, "%s: rows %lld elements apart", what, (long long)stride);
}

}  // namespace
}  // namespace rpg

using namespace rpg;

extern "C" {

int32_t rpg_hip_paged_append(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs, const rpg_hip_rows* k,
                             const rpg_hip_rows* v, const rpg_hip_rows* q, const rpg_hip_rows* q_out, int32_t n_heads,
                             const float* q_norm, const float* k_norm, float eps, const float* rope,
                             int64_t rope_rows, void* stream) {
  return Guard(
      [&] {
        paged::AppendArgs a;
        a.c = CacheOf(cache);
        a.s = SeqsOf(seqs, cache->page_size, true);
        if (Empty(a.s, true)) return 0;
        AppendRows(&a, k, v, q, q_out, n_heads, q_norm, k_norm, eps, rope, rope_rows);
        paged::Append(a, static_cast<hipStream_t>(stream));
        return 0;
      },
      -1);
}

int32_t rpg_hip_paged_decode(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs, const rpg_hip_rows* q,
                             const rpg_hip_rows* out, int32_t n_heads, float scale, void* work, int64_t work_bytes,
                             void* stream) {
  return Guard([&] { return Attention(cache, seqs, q, out, n_heads, scale, work, work_bytes, stream, false); }, -1);
}

int32_t rpg_hip_paged_prompt(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs, const rpg_hip_rows* q,
                             const rpg_hip_rows* out, int32_t n_heads, float scale, void* work, int64_t work_bytes,
                             void* stream) {
  return Guard([&] { return Attention(cache, seqs, q, out, n_heads, scale, work, work_bytes, stream, true); }, -1);
}

int64_t rpg_hip_paged_work(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs, int32_t n_heads,
                           int32_t prompt) {
  return Guard(
      [&]() -> int64_t {
        const paged::Cache c = CacheSizes(cache);
        const paged::Seqs s = SeqSizes(seqs, cache->page_size);
        CheckHeads(c, s, n_heads);
        return AttentionWork(c, s, n_heads, prompt != 0, false);
      },
      -1);
}

int32_t rpg_hip_sample_rows(int32_t type, const void* logits, int64_t n_rows, int64_t vocab, int64_t row_stride,
                            const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                            const float* u, int32_t* tokens, float* logprobs, void* work, int64_t work_bytes,
                            void* stream) {
  return Guard(
      [&] {
        const int bytes = ElementBytes(type);
        RPG_CHECK(n_rows >= 0 && n_rows <= 65535, "%lld rows outside [0, 65535]", (long long)n_rows);
        RPG_CHECK(vocab >= 1 && vocab <= 262144, "%lld logits outside [1, 262144]", (long long)vocab);
        if (n_rows == 0) return 0;
        CheckPointer("logits", logits, bytes);
        RPG_CHECK(n_rows == 1 || (row_stride >= 0 && row_stride <= kMaxStride), "row_stride %lld",
                  (long long)row_stride);
        for (const void* p : {static_cast<const void*>(temperature), static_cast<const void*>(top_k),
                              static_cast<const void*>(top_p), static_cast<const void*>(min_p),
                              static_cast<const void*>(logprobs)})
          if (p != nullptr) CheckPointer("a row parameter", p, 4);
        CheckPointer("u", u, 4);
        CheckPointer("tokens", tokens, 4);
        CheckPointer("work", work, 16);
        const int64_t need = rows::WorkBytes(n_rows, vocab);
        RPG_CHECK(work_bytes >= need, "%lld bytes of work memory, %lld are needed", (long long)work_bytes,
                  (long long)need);
        rows::SampleArgs a;
        a.logits = static_cast<const char*>(logits);
        a.row_bytes = n_rows == 1 ? 0 : row_stride * bytes;
        a.type = static_cast<uint32_t>(type);
        a.rows = static_cast<int32_t>(n_rows);
        a.vocab = static_cast<int32_t>(vocab);
        a.temperature = temperature;
        a.top_k = top_k;
        a.top_p = top_p;
        a.min_p = min_p;
        a.u = u;
        a.tokens = tokens;
        a.logprobs = logprobs;
        a.work = static_cast<char*>(work);
        rows::Sample(a, static_cast<hipStream_t>(stream));
        return 0;
      },
      -1);
}

int64_t rpg_hip_sample_rows_work(int64_t n_rows, int64_t vocab) {
  return Guard(
      [&]() -> int64_t {
        RPG_CHECK(n_rows >= 0 && n_rows <= 65535, "%lld rows outside [0, 65535]", (long long)n_rows);
        RPG_CHECK(vocab >= 1 && vocab <= 262144, "%lld logits outside [1, 262144]", (long long)vocab);
        return rows::WorkBytes(n_rows, vocab);
      },
      -1);
}

int32_t rpg_hip_quant_append(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs, int32_t type,
                             const rpg_hip_rows* k, const rpg_hip_rows* v, const rpg_hip_rows* q,
                             const rpg_hip_rows* q_out, int32_t n_heads, const float* q_norm, const float* k_norm,
                             float eps, const float* rope, int64_t rope_rows, void* stream) {
  return Guard(
      [&] {
        paged::CodesAppendArgs a;
        a.a.c = QuantOf(cache, type, &a.scales);
        a.code = cache->code;
        a.a.s = SeqsOf(seqs, cache->page_size, true);
        if (Empty(a.a.s, true)) return 0;
        AppendRows(&a.a, k, v, q, q_out, n_heads, q_norm, k_norm, eps, rope, rope_rows);
        paged::AppendCodes(a, static_cast<hipStream_t>(stream));
        return 0;
      },
      -1);
}

int32_t rpg_hip_quant_read(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs, int32_t type,
                           const rpg_hip_rows* k, const rpg_hip_rows* v, void* stream) {
  return Guard(
      [&] {
        paged::CodesReadArgs a;
        a.c = QuantOf(cache, type, &a.scales);
        a.code = cache->code;
        a.s = SeqsOf(seqs, cache->page_size, true);
        if (Empty(a.s, true)) return 0;
        RPG_CHECK(a.c.n_kv <= 65536, "%d key heads", a.c.n_kv);
        a.k = RowsOf("k", k, a.c, a.s.n_tokens, a.c.n_kv, true);
        a.v = RowsOf("v", v, a.c, a.s.n_tokens, a.c.n_kv, true);
        RPG_CHECK(a.k.p != a.v.p, "k and v are the same rows");
        paged::ReadCodes(a, static_cast<hipStream_t>(stream));
        return 0;
      },
      -1);
}

int32_t rpg_hip_quant_decode(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs, int32_t type,
                             const rpg_hip_rows* q, const rpg_hip_rows* out, int32_t n_heads, float scale, void* work,
                             int64_t work_bytes, void* stream) {
  return Guard(
      [&] { return QuantAttention(cache, seqs, type, q, out, n_heads, scale, work, work_bytes, stream, false); }, -1);
}

int32_t rpg_hip_quant_prompt(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs, int32_t type,
                             const rpg_hip_rows* q, const rpg_hip_rows* out, int32_t n_heads, float scale, void* work,
                             int64_t work_bytes, void* stream) {
  return Guard(
      [&] { return QuantAttention(cache, seqs, type, q, out, n_heads, scale, work, work_bytes, stream, true); }, -1);
}

int64_t rpg_hip_quant_work(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs, int32_t type,
                           int32_t n_heads, int32_t prompt) {
  return Guard(
      [&]() -> int64_t {
        paged::Scales scales;
        const paged::Cache c = QuantSizes(cache, type, &scales);
        const paged::Seqs s = SeqSizes(seqs, cache->page_size);
        CheckHeads(c, s, n_heads);
        return AttentionWork(c, s, n_heads, prompt != 0, true);
      },
      -1);
}

int32_t rpg_hip_paged_shared(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs,
                             const rpg_hip_groups* groups, const rpg_hip_rows* q, const rpg_hip_rows* out,
                             int32_t n_heads, float scale, void* work, int64_t work_bytes, void* stream) {
  return Guard(
      [&] {
        paged::SharedArgs a;
        a.a.c = CacheOf(cache);
        a.a.s = SeqsOf(seqs, cache->page_size, false);
        if (Empty(a.a.s, false)) return 0;
        AttentionRows(&a.a, q, out, a.a.s.n_seqs, n_heads, scale);
        a.groups = GroupsOf(groups, &a.a, false, &a.prefix_splits, work, work_bytes);
        paged::Shared(a, static_cast<hipStream_t>(stream));
        return 0;
      },
      -1);
}

int64_t rpg_hip_paged_shared_work(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs, int32_t n_groups,
                                  int32_t n_heads) {
  return Guard(
      [&]() -> int64_t {
        const paged::Cache c = CacheSizes(cache);
        const paged::Seqs s = SeqSizes(seqs, cache->page_size);
        int64_t bytes;
        SharedSizes(c, s, n_groups, n_heads, false, &bytes);
        return Empty(s, false) ? 0 : bytes;
      },
      -1);
}

int32_t rpg_hip_quant_shared(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs,
                             const rpg_hip_groups* groups, int32_t type, const rpg_hip_rows* q,
                             const rpg_hip_rows* out, int32_t n_heads, float scale, void* work, int64_t work_bytes,
                             void* stream) {
  return Guard(
      [&] {
        paged::CodesSharedArgs a;
        a.c.a.c = QuantOf(cache, type, &a.c.scales);
        a.c.code = cache->code;
        a.c.a.s = SeqsOf(seqs, cache->page_size, false);
        if (Empty(a.c.a.s, false)) return 0;
        AttentionRows(&a.c.a, q, out, a.c.a.s.n_seqs, n_heads, scale);
        a.groups = GroupsOf(groups, &a.c.a, true, &a.prefix_splits, work, work_bytes);
        paged::SharedCodes(a, static_cast<hipStream_t>(stream));
        return 0;
      },
      -1);
}

int64_t rpg_hip_quant_shared_work(const rpg_hip_quant_cache* cache, const rpg_hip_sequences* seqs, int32_t n_groups,
                                  int32_t type, int32_t n_heads) {
  return Guard(
      [&]() -> int64_t {
        paged::Scales scales;
        const paged::Cache c = QuantSizes(cache, type, &scales);
        const paged::Seqs s = SeqSizes(seqs, cache->page_size);
        int64_t bytes;
        SharedSizes(c, s, n_groups, n_heads, true, &bytes);
        return Empty(s, false) ? 0 : bytes;
      },
      -1);
}

int32_t rpg_hip_edit_logits(int32_t type, const void* logits, int64_t n_rows, int64_t vocab, int64_t row_stride,
                            const rpg_hip_edits* edits, void* out, int64_t out_stride, void* stream) {
  return Guard(
      [&] {
        const int bytes = ElementBytes(type);
        RPG_CHECK(edits != nullptr, "the edits are null");
        const rpg_hip_edits& e = *edits;
        RPG_CHECK(n_rows >= 0 && n_rows <= 65535, "%lld rows outside [0, 65535]", (long long)n_rows);
        RPG_CHECK(vocab >= 1 && vocab <= 1 << 24, "%lld logits outside [1, 2^24]", (long long)vocab);
        if (n_rows == 0) return 0;
        CheckPointer("logits", logits, bytes);
        CheckPointer("out", out, bytes);
        RPG_CHECK(n_rows == 1 || (row_stride >= 0 && row_stride <= kMaxStride), "row_stride %lld",
                  (long long)row_stride);
        RPG_CHECK(n_rows == 1 || (out_stride >= vocab && out_stride <= kMaxStride), "out_stride %lld",
                  (long long)out_stride);
        RPG_CHECK(out != logits || n_rows == 1 || out_stride == row_stride, "out is logits with another stride");
        rows::EditArgs a;
        a.logits = static_cast<const char*>(logits);
        a.out = static_cast<char*>(out);
        a.row_bytes = n_rows == 1 ? 0 : row_stride * bytes;
        a.out_bytes = n_rows == 1 ? 0 : out_stride * bytes;
        a.type = static_cast<uint32_t>(type);
        a.rows = static_cast<int32_t>(n_rows);
        a.vocab = static_cast<int32_t>(vocab);
        CheckApart("out overlaps logits", out, a.out_bytes, logits, a.row_bytes, n_rows, vocab * bytes);
        for (const void* p : {static_cast<const void*>(e.history_lens), static_cast<const void*>(e.prompts),
                              static_cast<const void*>(e.repetition), static_cast<const void*>(e.presence),
                              static_cast<const void*>(e.frequency), static_cast<const void*>(e.mask_rows)})
          if (p != nullptr) CheckPointer("a row parameter", p, 4);
        if (e.history != nullptr) {
          CheckList("history", e.history, n_rows == 1 ? 0 : e.history_stride);
          RPG_CHECK(e.history_size >= 0 && e.history_size <= rows::kMaxHistory, "a history of %d tokens", e.history_size);
          a.history = e.history;
          a.history_stride = n_rows == 1 ? 0 : e.history_stride;
          a.history_size = e.history_size;
          a.history_lens = e.history_lens;
          a.prompts = e.prompts;
          a.repetition = e.repetition;
          a.presence = e.presence;
          a.frequency = e.frequency;
        } else {
          RPG_CHECK(e.history_lens == nullptr && e.prompts == nullptr && e.repetition == nullptr &&
                        e.presence == nullptr && e.frequency == nullptr,
                    "penalties without a history");
        }
        RPG_CHECK((e.bias_ids == nullptr) == (e.bias == nullptr), "bias_ids without bias, or bias without bias_ids");
        if (e.bias_ids != nullptr) {
          CheckList("bias_ids", e.bias_ids, n_rows == 1 ? 0 : e.bias_ids_stride);
          CheckList("bias", e.bias, n_rows == 1 ? 0 : e.bias_stride);
          RPG_CHECK(e.n_biases >= 0 && e.n_biases <= rows::kMaxBiases, "%d biases", e.n_biases);
          a.bias_ids = e.bias_ids;
          a.bias = e.bias;
          a.bias_ids_stride = n_rows == 1 ? 0 : e.bias_ids_stride;
          a.bias_stride = n_rows == 1 ? 0 : e.bias_stride;
          a.n_biases = e.n_biases;
        }
        if (e.mask != nullptr) {
          RPG_CHECK(e.n_masks >= 0, "%d masks", e.n_masks);
          CheckList("mask", e.mask, e.n_masks <= 1 ? 0 : e.mask_stride);
          a.mask = e.mask;
          a.mask_stride = e.n_masks <= 1 ? 0 : e.mask_stride;
          a.mask_rows = e.mask_rows;
          a.n_masks = e.n_masks;
        } else {
          RPG_CHECK(e.mask_rows == nullptr, "mask_rows without a mask");
        }
        rows::Edit(a, static_cast<hipStream_t>(stream));
        return 0;
      },
      -1);
}

}  // extern "C"
