// extern "C" entry points of the serving operators (include/rpg_hip.h): checks
// of the callers' arguments, then one enqueue. Nothing here touches the GPU
// before every check has passed.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.h"
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

paged::Cache CacheSizes(const rpg_hip_paged_cache* c) {
  RPG_CHECK(c != nullptr, "the cache is null");
  paged::Cache out;
  const int bytes = ElementBytes(c->type);
  RPG_CHECK(c->head_dim == 64 || c->head_dim == 128, "head_dim %d is neither 64 nor 128", c->head_dim);
  RPG_CHECK(c->page_size >= 16 && c->page_size <= 65536 && (c->page_size & (c->page_size - 1)) == 0,
            "page_size %d is not a power of two from 16 to 65536", c->page_size);
  RPG_CHECK(c->n_pages >= 1, "a cache of %d pages", c->n_pages);
  RPG_CHECK(c->n_kv >= 1, "%d key heads", c->n_kv);
  out.page_bytes = StrideBytes("page_stride", c->page_stride, bytes);
  out.head_bytes = StrideBytes("head_stride", c->head_stride, bytes);
  const int64_t row = StrideBytes("row_stride", c->row_stride, bytes);
  // positions of a page are addressed by 32-bit offsets; no two of them overlap
  RPG_CHECK(row >= c->head_dim * bytes && row * c->page_size < kMaxStride, "row_stride %lld",
            (long long)c->row_stride);
  RPG_CHECK((c->n_kv == 1 || std::abs(out.head_bytes) >= c->head_dim * bytes) &&
                (c->n_pages == 1 || std::abs(out.page_bytes) >= c->head_dim * bytes),
            "head_stride %lld or page_stride %lld is less than a row", (long long)c->head_stride,
            (long long)c->page_stride);
  out.row_bytes = static_cast<int32_t>(row);
  out.n_pages = c->n_pages;
  out.n_kv = c->n_kv;
  out.page_log2 = __builtin_ctz(static_cast<unsigned>(c->page_size));
  out.head_dim = c->head_dim;
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

paged::Seqs SeqSizes(const rpg_hip_sequences* s, const rpg_hip_paged_cache* c) {
  RPG_CHECK(s != nullptr, "the sequences are null");
  paged::Seqs out;
  RPG_CHECK(s->n_seqs >= 0 && s->n_tokens >= 0, "%d sequences of %d new tokens", s->n_seqs, s->n_tokens);
  RPG_CHECK(s->pages >= 0 && s->pages <= kMaxPositions / c->page_size,
            "%d pages of %d positions for a sequence", s->pages, c->page_size);
  out.n_seqs = s->n_seqs;
  out.n_tokens = s->n_tokens;
  out.capacity = s->pages * c->page_size;
  return out;
}

paged::Seqs SeqsOf(const rpg_hip_sequences* s, const rpg_hip_paged_cache* c, bool packed) {
  paged::Seqs out = SeqSizes(s, c);
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

int Splits(const paged::Cache& c, const paged::Seqs& s, int32_t n_heads, bool prompt) {
  const int bytes = ElementBytes(static_cast<int32_t>(c.type));
  if (prompt) return paged::PromptSplits(s.n_tokens, s.n_seqs, n_heads, c.n_kv, bytes, s.capacity);
  return paged::DecodeSplits(s.n_seqs, n_heads, c.n_kv, bytes, s.capacity);
}

// Calls without sequences or new tokens have nothing to do.
bool Empty(const paged::Seqs& s, bool packed) { return s.n_seqs == 0 || (packed && s.n_tokens == 0); }

int64_t AttentionWork(const paged::Cache& c, const paged::Seqs& s, int32_t n_heads, bool prompt) {
  if (Empty(s, prompt)) return 0;
  const int64_t rows = static_cast<int64_t>(prompt ? s.n_tokens : s.n_seqs) * n_heads;
  return paged::WorkBytes(rows, c.head_dim, Splits(c, s, n_heads, prompt));
}

int32_t Attention(const rpg_hip_paged_cache* cache, const rpg_hip_sequences* seqs, const rpg_hip_rows* q,
                  const rpg_hip_rows* out, int32_t n_heads, float scale, void* work, int64_t work_bytes, void* stream,
                  bool prompt) {
  paged::AttentionArgs a;
  a.c = CacheOf(cache);
  a.s = SeqsOf(seqs, cache, prompt);
  if (Empty(a.s, prompt)) return 0;
  CheckHeads(a.c, a.s, n_heads);
  const int n_tokens = prompt ? a.s.n_tokens : a.s.n_seqs;
  a.q = RowsOf("q", q, a.c, n_tokens, n_heads, false);
  a.out = RowsOf("out", out, a.c, n_tokens, n_heads, true);
  CheckInPlace("out is q", a.out, a.q, n_tokens, n_heads);
  RPG_CHECK(scale > 0.0f && std::isfinite(scale), "scale %g is not positive and finite", scale);
  a.n_heads = n_heads;
  a.scale = scale;
  a.splits = Splits(a.c, a.s, n_heads, prompt);
  const int64_t need = AttentionWork(a.c, a.s, n_heads, prompt);
  if (need > 0) {
    CheckPointer("work", work, 16);
    RPG_CHECK(work_bytes >= need, "%lld bytes of work memory, %lld are needed", (long long)work_bytes,
              (long long)need);
  }
  a.work = static_cast<float*>(work);
  if (prompt)
    paged::Prompt(a, static_cast<hipStream_t>(stream));
  else
    paged::Decode(a, static_cast<hipStream_t>(stream));
  return 0;
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
        a.s = SeqsOf(seqs, cache, true);
        if (Empty(a.s, true)) return 0;
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
        const paged::Seqs s = SeqSizes(seqs, cache);
        CheckHeads(c, s, n_heads);
        return AttentionWork(c, s, n_heads, prompt != 0);
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

}  // extern "C"
