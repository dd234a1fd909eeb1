// The extern "C" entry points of the paged cache and of beam search's selection (include/cudallm.h): argument checks,
// then the launchers of kernels/paged.h. Nothing is enqueued when a check fails.
#include <algorithm>
#include <array>
#include <climits>
#include <cmath>
#include <cstdint>
#include <exception>
#include <numeric>
#include <string>
#include <utility>

#include "common/check.h"
#include "cudallm.h"
#include "kernels/paged.h"

namespace cudallm {
int capi_report(const std::exception& ex);  // capi.cpp: sets cudallm_last_error, returns the code

namespace {

template <typename Body>
int invoke(Body&& body) noexcept {
    try {
        body();
        return CUDALLM_OK;
    } catch (const std::exception& ex) {
        return capi_report(ex);
    } catch (...) {
        return capi_report(InternalError("unknown exception"));
    }
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

size_t x_bytes(int x_dtype) { return x_dtype == CUDALLM_X_FP32 ? 4 : 2; }

// [p, p + n) and [q, q + m) share a byte.
bool overlap(const void* p, unsigned long long n, const void* q, unsigned long long m) {
    const auto a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return n != 0 && m != 0 && a < b + m && b < a + n;
}

// [q, q + m) and one of the rows [p + r * stride, + n) share a byte.
bool rows_meet(const void* p, long long rows, long long n, long long stride, const void* q, long long m) {
    if (!overlap(p, (rows - 1) * stride + n, q, m)) return false;
    if (rows == 1 || stride == 0) return true;
    const long long d = static_cast<long long>(reinterpret_cast<uintptr_t>(q)) - static_cast<long long>(reinterpret_cast<uintptr_t>(p));
    return std::min((d + m - 1) / stride, rows - 1) * stride + n > d;  // the last row that starts before the end of q
}

// Heads of n bytes at p + t * token + h * head, t < tokens.
struct Heads {
    const void* p;
    long long token, head, heads;
};

// a and b have a byte in common. Exact where their tokens are equally far apart (as they are in a packed projection) and the pairs of heads are few
// or equally spaced; otherwise only heads that the strides' common divisor keeps apart are known to be.
bool heads_meet(Heads a, Heads b, long long tokens, long long n) {
    for (Heads* x : {&a, &b}) {
        if (tokens == 1) x->token = 0;
        if (x->heads == 1) x->head = 0;
    }
    const long long in_a = (a.heads - 1) * a.head + n, in_b = (b.heads - 1) * b.head + n;  // a token spans
    if (!overlap(a.p, (tokens - 1) * a.token + in_a, b.p, (tokens - 1) * b.token + in_b)) return false;
    const long long d = static_cast<long long>(reinterpret_cast<uintptr_t>(b.p)) - static_cast<long long>(reinterpret_cast<uintptr_t>(a.p));
    if (a.token == b.token) {
        // [0, n_a) of one token meets [x, x + n_b) of another one (or the same).
        auto meet = [&](long long x, long long n_a, long long n_b) {
            if (a.token == 0) return x > -n_b && x < n_a;
            const long long most = x + (tokens - 1) * a.token, above = most + n_b - 1;  // take tokens off while it stays above -n_b
            if (above < 0) return false;
            return most - std::min(above / a.token, 2 * (tokens - 1)) * a.token < n_a;
        };
        if (!meet(d, in_a, in_b)) return false;
        if (a.head == b.head) {
            for (long long i = 1 - a.heads; i < b.heads; ++i)
                if (meet(d + i * a.head, n, n)) return true;
            return false;
        }
        if (a.heads * b.heads <= 65536) {
            for (long long i = 0; i < a.heads; ++i)
                for (long long j = 0; j < b.heads; ++j)
                    if (meet(d + j * b.head - i * a.head, n, n)) return true;
            return false;
        }
    }
    const long long step = std::gcd(std::gcd(a.token, b.token), std::gcd(a.head, b.head));
    if (step == 0) return true;
    const long long r = (d % step + step) % step;
    return r < n || step - r < n;
}

// Bytes that rows of `width` ints with a stride span.
unsigned long long table_bytes(int rows, int width, long long stride) {
    return rows < 1 || width < 1 ? 0 : 4 * (static_cast<unsigned long long>(rows - 1) * stride + width);
}

void check_pages(const cudallm_pages* p) {
    CLLM_REQUIRE(p != nullptr, "pages is null");
    CLLM_REQUIRE(p->struct_size == static_cast<int>(sizeof(cudallm_pages)), "cudallm_pages.struct_size must be sizeof(cudallm_pages)");
    CLLM_REQUIRE(p->kv_dtype == CUDALLM_KV_FP16 || p->kv_dtype == CUDALLM_KV_BF16, "kv_dtype must be 0 (fp16) or 1 (bf16)");
    CLLM_REQUIRE(p->n_layers > 0 && p->n_pages > 0 && p->n_kv_heads > 0 && p->page_size > 0,
                 "n_layers, n_pages, n_kv_heads and page_size must be positive");
    CLLM_REQUIRE(p->head_dim >= 8 && p->head_dim <= 256 && p->head_dim % 8 == 0, "head_dim must be a multiple of 8 in 8 .. 256");
    CLLM_REQUIRE(p->k != nullptr && p->v != nullptr && aligned(p->k, 16) && aligned(p->v, 16), "k and v must be 16-byte aligned device pointers");
    // In the order of their strides, each dimension must step over all of the smaller ones.
    std::array<std::pair<long long, long long>, 4> dims{{{p->token_stride, p->page_size},
                                                         {p->head_stride, p->n_kv_heads},
                                                         {p->page_stride, p->n_pages},
                                                         {p->layer_stride, p->n_layers}}};
    std::sort(dims.begin(), dims.end());
    long long span = p->head_dim;
    for (const auto& [stride, size] : dims) {
        if (size == 1) continue;
        CLLM_REQUIRE(stride % 8 == 0 && stride >= span, "page strides must be multiples of 8 elements, and elements must not overlap");
        span += stride * (size - 1);
    }
}

void check_layer(const cudallm_pages* p, int layer) {
    CLLM_REQUIRE(layer >= 0 && layer < p->n_layers, "layer out of range");
}

void check_x_dtype(int x) {
    CLLM_REQUIRE(x >= CUDALLM_X_FP32 && x <= CUDALLM_X_BF16, "x_dtype must be 0 (fp32), 1 (fp16) or 2 (bf16)");
}

void check_workspace(const void* w, unsigned long long got, size_t need) {
    CLLM_REQUIRE(w != nullptr && aligned(w, 256) && got >= need,
                 "workspace must be 256-byte aligned and hold at least " + std::to_string(need) + " bytes");
}

void check_table(const int* t, int rows, int width, long long stride) {
    CLLM_REQUIRE(rows >= 0 && rows <= kMaxPageRows && width >= 0, "rows must be in 0 .. 65536, table_width not negative");
    CLLM_REQUIRE(static_cast<long long>(rows) * width <= INT_MAX, "a table must have fewer than 2^31 entries");
    CLLM_REQUIRE(rows == 0 || width == 0 || (t != nullptr && aligned(t, 4)), "tables is null");
    CLLM_REQUIRE(rows <= 1 || stride >= width, "table_stride must be at least table_width");
}

}  // namespace
}  // namespace cudallm

using namespace cudallm;

extern "C" {

unsigned long long cudallm_attend_workspace_bytes(void) { return attend_workspace_bytes(); }

unsigned long long cudallm_pages_workspace_bytes(int n_pages, int rows) { return pages_workspace_bytes(n_pages, rows); }

unsigned long long cudallm_beam_workspace_bytes(int rows, int vocab, int keep) { return beam_workspace_bytes(rows, vocab, keep); }

int cudallm_paged_attend(const cudallm_pages* pages, const cudallm_attend_args* a, void* stream) {
    return invoke([&] {
        check_pages(pages);
        CLLM_REQUIRE(a != nullptr && a->struct_size == static_cast<int>(sizeof(cudallm_attend_args)),
                     "cudallm_attend_args.struct_size must be sizeof(cudallm_attend_args)");
        check_layer(pages, a->layer);
        check_x_dtype(a->x_dtype);
        check_table(a->tables, a->n_seq, a->table_width, a->table_stride);
        if (a->n_seq == 0) return;
        CLLM_REQUIRE(a->n_heads > 0 && a->n_heads % pages->n_kv_heads == 0, "n_heads must be a positive multiple of n_kv_heads");
        CLLM_REQUIRE(static_cast<long long>(a->n_seq) * a->n_heads <= INT_MAX, "n_seq * n_heads must be below 2^31");
        CLLM_REQUIRE(static_cast<long long>(a->table_width) * pages->page_size <= INT_MAX - 64, "a row must hold fewer than 2^31 - 64 tokens");
        CLLM_REQUIRE(a->window >= 0 && std::isfinite(a->scale), "window must not be negative, scale must be finite");
        const size_t es = x_bytes(a->x_dtype);
        CLLM_REQUIRE(a->q != nullptr && a->lens != nullptr && a->out != nullptr, "q, lens and out must be non-null");
        CLLM_REQUIRE(aligned(a->q, es) && aligned(a->out, es) && aligned(a->lens, 4) && aligned(a->lse, 4), "misaligned pointer");
        CLLM_REQUIRE(a->q_seq_stride >= 0 && a->q_head_stride >= 0, "q strides must not be negative");
        const unsigned long long span = (a->n_seq - 1) * a->q_seq_stride + (a->n_heads - 1) * a->q_head_stride + pages->head_dim;
        const unsigned long long heads = static_cast<unsigned long long>(a->n_seq) * a->n_heads, outs = es * heads * pages->head_dim;
        const unsigned long long lses = a->lse != nullptr ? 4 * heads : 0, table = table_bytes(a->n_seq, a->table_width, a->table_stride);
        CLLM_REQUIRE(!overlap(a->q, es * span, a->out, outs), "out must not overlap q");
        CLLM_REQUIRE(!overlap(a->tables, table, a->out, outs) && !overlap(a->lens, 4ull * a->n_seq, a->out, outs), "out must not overlap tables or lens");
        CLLM_REQUIRE(!overlap(a->q, es * span, a->lse, lses) && !overlap(a->out, outs, a->lse, lses) && !overlap(a->tables, table, a->lse, lses) &&
                         !overlap(a->lens, 4ull * a->n_seq, a->lse, lses),
                     "lse must not overlap q, out, tables or lens");
        check_workspace(a->workspace, a->workspace_bytes, attend_workspace_bytes());
        launch_paged_attend(*pages, *a, static_cast<cudaStream_t>(stream));
    });
}

int cudallm_paged_append(const cudallm_pages* pages, const cudallm_append_args* a, void* stream) {
    return invoke([&] {
        check_pages(pages);
        CLLM_REQUIRE(a != nullptr && a->struct_size == static_cast<int>(sizeof(cudallm_append_args)),
                     "cudallm_append_args.struct_size must be sizeof(cudallm_append_args)");
        check_layer(pages, a->layer);
        check_x_dtype(a->x_dtype);
        check_table(a->tables, a->n_rows, a->table_width, a->table_stride);
        CLLM_REQUIRE(a->n_tokens >= 0, "n_tokens must not be negative");
        if (a->n_tokens == 0) return;
        const size_t es = x_bytes(a->x_dtype);
        CLLM_REQUIRE(a->k != nullptr && a->v != nullptr && a->positions != nullptr, "k, v and positions must be non-null");
        CLLM_REQUIRE(aligned(a->k, es) && aligned(a->v, es) && aligned(a->q, es) && aligned(a->q_out, es) && aligned(a->positions, 4) &&
                         aligned(a->rows, 4) && aligned(a->inv_freq, 4),
                     "misaligned pointer");
        CLLM_REQUIRE(a->rotary >= 0 && a->rotary % 2 == 0 && a->rotary <= pages->head_dim, "rotary must be even and at most head_dim");
        CLLM_REQUIRE(a->rotary == 0 || a->inv_freq != nullptr, "inv_freq must be non-null");
        CLLM_REQUIRE(a->q == nullptr || (a->n_heads > 0 && a->q_out != nullptr), "q needs n_heads > 0 and q_out");
        CLLM_REQUIRE(a->q_token_stride >= 0 && a->q_head_stride >= 0 && a->k_token_stride >= 0 && a->k_head_stride >= 0 &&
                         a->v_token_stride >= 0 && a->v_head_stride >= 0,
                     "strides must not be negative");
        CLLM_REQUIRE(a->n_heads <= 65536 && pages->n_kv_heads <= 65536, "at most 65536 heads");
        if (a->q != nullptr) {
            const long long T = a->n_tokens, H = a->n_heads, hd = pages->head_dim, ts = a->out_token_stride, hs = a->out_head_stride;
            const bool token_outer = (H == 1 || hs >= hd) && (T == 1 || ts >= (H == 1 ? hd : hs * (H - 1) + hd));
            const bool head_outer = (T == 1 || ts >= hd) && (H == 1 || hs >= (T == 1 ? hd : ts * (T - 1) + hd));
            CLLM_REQUIRE(token_outer || head_outer, "heads of q_out must not overlap");
            const bool same = a->q_out == a->q && (T == 1 || ts == a->q_token_stride) && (H == 1 || hs == a->q_head_stride);
            const unsigned long long span = es * ((T - 1) * (T > 1 ? ts : 0) + (H - 1) * (H > 1 ? hs : 0) + hd);
            CLLM_REQUIRE(!overlap(a->positions, 4ull * T, a->q_out, span) && (a->rows == nullptr || !overlap(a->rows, 4ull * T, a->q_out, span)) &&
                             !overlap(a->tables, table_bytes(a->n_rows, a->table_width, a->table_stride), a->q_out, span) &&
                             !overlap(a->inv_freq, 2ull * a->rotary, a->q_out, span),
                         "q_out must not overlap positions, rows, tables or inv_freq");
            const long long b = es, head = hd * b;
            const Heads written{a->q_out, ts * b, hs * b, H};
            CLLM_REQUIRE(same || !heads_meet(written, {a->q, a->q_token_stride * b, a->q_head_stride * b, H}, T, head), "q_out must be q or not overlap it");
            CLLM_REQUIRE(!heads_meet(written, {a->k, a->k_token_stride * b, a->k_head_stride * b, pages->n_kv_heads}, T, head) &&
                             !heads_meet(written, {a->v, a->v_token_stride * b, a->v_head_stride * b, pages->n_kv_heads}, T, head),
                         "q_out must not overlap k or v");
        }
        CLLM_REQUIRE(std::isfinite(a->factor), "factor must be finite");
        launch_paged_append(*pages, *a, static_cast<cudaStream_t>(stream));
    });
}

int cudallm_paged_fork(const cudallm_pages* pages, const cudallm_fork_args* a, void* stream) {
    return invoke([&] {
        check_pages(pages);
        CLLM_REQUIRE(a != nullptr && a->struct_size == static_cast<int>(sizeof(cudallm_fork_args)),
                     "cudallm_fork_args.struct_size must be sizeof(cudallm_fork_args)");
        check_table(a->tables, a->n_rows, a->table_width, a->table_stride);
        check_table(a->tables_out, a->n_out, a->table_width, a->table_out_stride);
        CLLM_REQUIRE(static_cast<long long>(a->table_width) * pages->page_size <= INT_MAX, "a row must hold fewer than 2^31 tokens");
        CLLM_REQUIRE(a->room >= 0, "room must not be negative");
        CLLM_REQUIRE(a->n_rows == 0 || a->lens != nullptr, "lens is null");
        CLLM_REQUIRE(a->n_out == 0 || (a->parents != nullptr && a->lens_out != nullptr), "parents and lens_out must be non-null");
        CLLM_REQUIRE(a->refs != nullptr && a->refs_out != nullptr && a->missing != nullptr, "refs, refs_out and missing must be non-null");
        CLLM_REQUIRE(aligned(a->lens, 4) && aligned(a->parents, 4) && aligned(a->lens_out, 4) && aligned(a->refs, 4) &&
                         aligned(a->refs_out, 4) && aligned(a->missing, 4),
                     "misaligned pointer");
        const std::array<std::pair<const void*, unsigned long long>, 4> in{
            {{a->tables, table_bytes(a->n_rows, a->table_width, a->table_stride)},
             {a->lens, 4ull * a->n_rows},
             {a->refs, 4ull * pages->n_pages},
             {a->parents, 4ull * a->n_out}}};
        const std::array<std::pair<const void*, unsigned long long>, 4> out{
            {{a->tables_out, table_bytes(a->n_out, a->table_width, a->table_out_stride)},
             {a->lens_out, 4ull * a->n_out},
             {a->refs_out, 4ull * pages->n_pages},
             {a->missing, 4ull}}};
        for (size_t o = 0; o < out.size(); ++o) {
            for (const auto& i : in) CLLM_REQUIRE(!overlap(i.first, i.second, out[o].first, out[o].second), "outputs must not overlap inputs");
            for (size_t k = 0; k < o; ++k)
                CLLM_REQUIRE(!overlap(out[k].first, out[k].second, out[o].first, out[o].second), "outputs must not overlap each other");
        }
        check_workspace(a->workspace, a->workspace_bytes, pages_workspace_bytes(pages->n_pages, std::max(a->n_rows, a->n_out)));
        launch_paged_fork(*pages, *a, static_cast<cudaStream_t>(stream));
    });
}

int cudallm_paged_compact(const cudallm_pages* pages, const cudallm_compact_args* a, void* stream) {
    return invoke([&] {
        check_pages(pages);
        CLLM_REQUIRE(a != nullptr && a->struct_size == static_cast<int>(sizeof(cudallm_compact_args)),
                     "cudallm_compact_args.struct_size must be sizeof(cudallm_compact_args)");
        check_table(a->tables, a->n_rows, a->table_width, a->table_stride);
        check_table(a->tables_out, a->n_rows, a->table_width, a->table_out_stride);
        CLLM_REQUIRE(a->refs != nullptr && a->refs_out != nullptr && a->live != nullptr, "refs, refs_out and live must be non-null");
        CLLM_REQUIRE(aligned(a->refs, 4) && aligned(a->refs_out, 4) && aligned(a->live, 4), "misaligned pointer");
        const std::array<std::pair<const void*, unsigned long long>, 2> in{
            {{a->tables, table_bytes(a->n_rows, a->table_width, a->table_stride)}, {a->refs, 4ull * pages->n_pages}}};
        const std::array<std::pair<const void*, unsigned long long>, 3> out{
            {{a->tables_out, table_bytes(a->n_rows, a->table_width, a->table_out_stride)}, {a->refs_out, 4ull * pages->n_pages}, {a->live, 4ull}}};
        for (size_t o = 0; o < out.size(); ++o) {
            for (const auto& i : in) CLLM_REQUIRE(!overlap(i.first, i.second, out[o].first, out[o].second), "outputs must not overlap inputs");
            for (size_t k = 0; k < o; ++k)
                CLLM_REQUIRE(!overlap(out[k].first, out[k].second, out[o].first, out[o].second), "outputs must not overlap each other");
        }
        check_workspace(a->workspace, a->workspace_bytes, pages_workspace_bytes(pages->n_pages, a->n_rows));
        launch_paged_compact(*pages, *a, static_cast<cudaStream_t>(stream));
    });
}

int cudallm_beam_select(const cudallm_beam_args* a, void* stream) {
    return invoke([&] {
        CLLM_REQUIRE(a != nullptr && a->struct_size == static_cast<int>(sizeof(cudallm_beam_args)),
                     "cudallm_beam_args.struct_size must be sizeof(cudallm_beam_args)");
        check_x_dtype(a->x_dtype);
        CLLM_REQUIRE(a->beams >= 1 && a->beams <= kMaxBeams && a->keep >= 1 && a->keep <= kMaxKeep && a->vocab >= 1 && a->vocab <= kMaxVocab,
                     "beams and keep must be in 1 .. 64, vocab in 1 .. 2^24");
        CLLM_REQUIRE(a->keep <= static_cast<long long>(a->beams) * a->vocab, "keep must be at most beams * vocab");
        CLLM_REQUIRE(a->n_groups >= 0 && static_cast<long long>(a->n_groups) * a->beams <= kMaxPageRows, "n_groups * beams must be in 0 .. 65536");
        if (a->n_groups == 0) return;
        const int rows = a->n_groups * a->beams;
        const size_t es = x_bytes(a->x_dtype);
        CLLM_REQUIRE(a->logits != nullptr && a->scores != nullptr && a->out_scores != nullptr && a->out_parents != nullptr && a->out_tokens != nullptr,
                     "logits, scores and the outputs must be non-null");
        CLLM_REQUIRE(aligned(a->logits, es) && aligned(a->scores, 4) && aligned(a->finished, 4) && aligned(a->out_scores, 4) &&
                         aligned(a->out_parents, 4) && aligned(a->out_tokens, 4),
                     "misaligned pointer");
        CLLM_REQUIRE(rows == 1 || a->row_stride >= a->vocab || a->row_stride == 0, "row_stride must be at least vocab, or 0 for one shared row");
        CLLM_REQUIRE(a->finished == nullptr || (a->eos >= 0 && a->eos < a->vocab), "eos must be in [0, vocab)");
        const long long outs = 4LL * a->n_groups * a->keep;
        const std::array<const void*, 3> out{a->out_scores, a->out_parents, a->out_tokens};
        for (size_t o = 0; o < out.size(); ++o) {
            // A group's scores are read before its own are written, so that they may be written in place where each has as many.
            const bool in_place = o == 0 && a->out_scores == a->scores && a->keep == a->beams;
            CLLM_REQUIRE((in_place || !overlap(a->scores, 4ull * rows, out[o], outs)) && (a->finished == nullptr || !overlap(a->finished, 4ull * rows, out[o], outs)) &&
                             !rows_meet(a->logits, rows, es * a->vocab, es * a->row_stride, out[o], outs),
                         "outputs must not overlap inputs (but out_scores may be scores where keep is beams)");
            for (size_t k = 0; k < o; ++k) CLLM_REQUIRE(!overlap(out[k], outs, out[o], outs), "outputs must not overlap each other");
        }
        check_workspace(a->workspace, a->workspace_bytes, beam_workspace_bytes(rows, a->vocab, a->keep));
        launch_beam_select(*a, static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
