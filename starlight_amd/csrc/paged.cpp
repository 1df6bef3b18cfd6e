#include "paged.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

namespace slhip {
namespace {

constexpr uint64_t kTableWordsMost = 1ull << 22;  // u32 buffers that the device keeps a host copy of
constexpr uint64_t kPositionsMost = 0x7fffffffull;

bool fail(Error* err, const Error& e) {
    *err = e;
    return false;
}

// a b c ..., or UINT64_MAX when it does not fit.
uint64_t product(std::initializer_list<uint64_t> f) {
    unsigned __int128 p = 1;
    for (uint64_t x : f) {
        p *= x;
        if (p > UINT64_MAX) p = UINT64_MAX;  // (stays there unless a factor is 0)
    }
    return static_cast<uint64_t>(p);
}

bool overlap(const sl_buffer_ref& a, const sl_buffer_ref& b) {
    return a.buffer == b.buffer && a.len != 0 && b.len != 0 && a.offset < b.offset + b.len &&
           b.offset < a.offset + a.len;
}

}  // namespace

bool paged_argument_missing(const PagedCall& c) {
    const bool append = c.kind == SL_PAGED_APPEND;
    return c.op == nullptr || c.tokens == nullptr || c.kv == nullptr ||
           (append ? c.k == nullptr || c.v == nullptr : c.q == nullptr || c.out == nullptr);
}

bool check_paged_call(const BufferView& buffers, const PagedCall& given, Error* err) {
    PagedCall c = given;
    if (c.kind != SL_PAGED_APPEND) c.k = c.v = nullptr, c.rope = nullptr;  // (not the operator's)
    if (c.op->code != SL_OP_CAUSAL_ATTENTION) return fail(err, Error::unsupported_op(c.op->code));
    if (c.rope != nullptr && c.rope->code != SL_OP_ROPE) return fail(err, Error::unsupported_op(c.rope->code));
    const uint64_t H = c.op->heads, Hkv = c.op->kv_heads, D = c.op->head_dim;
    const uint64_t B = c.tokens->batch, T = c.tokens->tokens;
    const sl_paged_kv& kv = *c.kv;
    if (Hkv == 0 || H == 0 || H % Hkv != 0)
        return fail(err, Error::execution("heads must be a multiple of kv_heads"));
    if (D == 0 || D % 16 != 0 || D > 256)
        return fail(err, Error::unimplemented("paged operators need head_dim a multiple of 16 up to 256"));
    if (H > 1024) return fail(err, Error::unimplemented("paged operators take at most 1024 heads"));
    if (kv.layers == 0 || c.op->layer >= kv.layers) return fail(err, Error::execution("layer is out of range"));
    if (c.kind != SL_PAGED_APPEND && !std::isfinite(c.op->scale))
        return fail(err, Error::execution("attention scale must be finite"));
    if (c.rope != nullptr) {
        if (c.rope->rope_variant != SL_ROPE_NEOX && c.rope->rope_variant != SL_ROPE_GPTJ)
            return fail(err, Error::execution("rope variant is not known"));
        if (!(c.rope->theta > 0.f) || !std::isfinite(c.rope->theta))
            return fail(err, Error::execution("rope theta must be positive and finite"));
    }
    if (kv.page_size == 0 || kv.page_size % 16 != 0)
        return fail(err, Error::unimplemented("page_size must be a nonzero multiple of 16"));
    if (kv.num_pages == 0 || kv.pages_per_seq == 0) return fail(err, Error::execution("the page pool is empty"));
    if (product({kv.pages_per_seq, kv.page_size}) > kPositionsMost)
        return fail(err, Error::unimplemented("a block table covers more than 2^31 - 1 positions"));
    // (the launches' threads, at most (T H / 16 + B Hkv) 512 and 256 T, are counted in 32 bits)
    if (T >= 1u << 24 || product({T, H}) > 1u << 25 || product({B, Hkv}) > 1u << 22)
        return fail(err, Error::unimplemented("too many tokens or rows for one call"));
    const auto kind_of = [&](uint32_t id) -> uint32_t {
        const sl_buffer_desc* d = buffers.get(id);
        return d ? d->kind : static_cast<uint32_t>(SL_BUFFER_NONE);
    };
    if (kind_of(kv.pool) != SL_BUFFER_F32) return fail(err, Error::invalid_buffer(kv.pool));
    for (uint32_t id : {kv.block_table, kv.seq_lens, c.tokens->row_starts}) {
        if (kind_of(id) != SL_BUFFER_U32) return fail(err, Error::invalid_buffer(id));
        if (buffers.get(id)->elements > kTableWordsMost)
            return fail(err, Error::unimplemented("block table, lengths and row starts must be u32 buffers of at most "
                                                  "16 MiB"));
    }
    if (buffers.get(kv.pool)->elements != product({kv.layers, kv.num_pages, 2, kv.page_size, Hkv, D}))
        return fail(err, Error::execution("page pool size does not match its layout"));
    if (buffers.get(kv.block_table)->elements < product({B, kv.pages_per_seq}) ||
        buffers.get(kv.seq_lens)->elements < B)
        return fail(err, Error::execution("block table or lengths buffer is too small for the batch"));
    if (buffers.get(c.tokens->row_starts)->elements < B + 1)
        return fail(err, Error::execution("row starts buffer is too small for the batch"));
    // ports: f32 ranges of the stated sizes
    if (c.kind == SL_PAGED_APPEND && (c.q == nullptr) != (c.out == nullptr))
        return fail(err, Error::execution("queries and rotated queries are given together"));
    const struct {
        const sl_buffer_ref* r;
        uint64_t len;
    } ports[4] = {{c.q, product({T, H, D})}, {c.k, product({T, Hkv, D})}, {c.v, product({T, Hkv, D})},
                  {c.out, product({T, H, D})}};
    for (const auto& p : ports) {
        if (p.r == nullptr) continue;
        const sl_buffer_ref& r = *p.r;
        if (kind_of(r.buffer) != SL_BUFFER_F32) return fail(err, Error::invalid_buffer(r.buffer));
        if (r.len != p.len) return fail(err, Error::execution("paged operator port has the wrong length"));
        const uint64_t have = buffers.get(r.buffer)->elements;
        if (r.offset > have || r.len > have - r.offset)
            return fail(err, Error::invalid_range(r.buffer, r.offset, r.len));
    }
    for (const auto& p : ports) {
        if (p.r == nullptr) continue;
        if (p.r->buffer == kv.pool || (p.r != c.out && c.out != nullptr && overlap(*p.r, *c.out)))
            return fail(err, Error::execution("a command output aliases an overlapping input range"));
    }
    return true;
}

bool check_paged_contents(const PagedCall& c, const PagedTables& t, uint32_t few, PagedPlan* plan, Error* err) {
    const sl_paged_kv& kv = *c.kv;
    const uint64_t B = c.tokens->batch, T = c.tokens->tokens, ps = kv.page_size, per = kv.pages_per_seq;
    const uint64_t capacity = per * ps;
    *plan = PagedPlan{};
    const uint32_t* const starts = t.row_starts;
    bool ordered = starts[0] == 0 && starts[B] == T;
    for (uint64_t b = 0; b < B; ++b) ordered &= starts[b] <= starts[b + 1];
    if (!ordered) return fail(err, Error::execution("row starts must rise from 0 to the number of tokens"));
    for (uint64_t b = 0; b < B; ++b) {
        const uint64_t L = t.seq_lens[b], n = starts[b + 1] - starts[b];
        if (n != 0 && L + n > capacity)
            return fail(err, Error::execution("paged KV length exceeds the row's block table"));
    }
    // the ids of the pages from .. upto - 1 of row b are below num_pages
    const auto in_range = [&](uint64_t b, uint64_t from, uint64_t upto) {
        uint32_t most = 0;
        const uint32_t* const ids = t.block_table + b * per;
        for (uint64_t i = from; i < upto; ++i) most = most > ids[i] ? most : ids[i];
        return from >= upto || most < kv.num_pages;
    };
    const auto pages = [&](uint64_t positions) { return (positions + ps - 1) / ps; };
    const char* const bad_id = "page id out of range";
    const uint64_t group = c.op->heads / c.op->kv_heads;
    const uint32_t* shared = nullptr;  // the prefix's pages
    for (uint64_t b = 0; b < B; ++b) {
        const uint64_t L = t.seq_lens[b], n = starts[b + 1] - starts[b], end = L + n;
        if (n == 0) continue;
        const uint64_t rows = n * group;
        uint64_t keys = 0;  // that the row's queries see at most
        plan->rows_with_tokens += 1;
        if (rows <= few) plan->few_rows += (rows + 15) / 16 * 16;  // (each row's blocks counted up)
        else plan->many_rows += (rows + 15) / 16 * 16, plan->many_blocks += (rows + 255) / 256;
        if (c.kind == SL_PAGED_APPEND) {
            if (!in_range(b, L / ps, pages(end))) return fail(err, Error::execution(bad_id));
        } else if (c.kind == SL_PAGED_WINDOW) {
            // only pages with a position that one of the row's queries sees are read
            uint64_t first = 0, sinks = 0;
            if (c.window != 0) {
                first = L + 1 > c.window ? L + 1 - c.window : 0;
                sinks = std::min<uint64_t>(c.sinks, first);
            }
            if (!in_range(b, first / ps, pages(end)) || !in_range(b, 0, pages(sinks)))
                return fail(err, Error::execution(bad_id));
            keys = end - first + sinks;
        } else {
            if (L < c.prefix) return fail(err, Error::execution("a row is shorter than the shared prefix"));
            const uint32_t* const ids = t.block_table + b * per;
            if (shared == nullptr) {
                shared = ids;
                if (!in_range(b, 0, pages(c.prefix))) return fail(err, Error::execution(bad_id));
            } else if (c.prefix != 0 && std::memcmp(shared, ids, pages(c.prefix) * 4) != 0) {
                return fail(err, Error::execution("a row does not begin with the shared prefix's pages"));
            }
            if (!in_range(b, c.prefix / ps, pages(end))) return fail(err, Error::execution(bad_id));
            keys = end;
        }
        uint32_t& most = rows <= few ? plan->few_keys : plan->many_keys;
        most = std::max(most, static_cast<uint32_t>(keys));
        (rows <= few ? plan->few_keys_in_all : plan->many_keys_in_all) += keys;
    }
    if (c.kind == SL_PAGED_APPEND && T != 0) {
        // A page that a row writes belongs to that row alone: neither another row's
        // cached or new positions lie in it, nor a second page of the row itself.
        std::vector<uint64_t> written((kv.num_pages + 63) / 64, 0);
        const auto is_written = [&](uint32_t id) { return (written[id / 64] >> (id % 64) & 1) != 0; };
        const char* const twice = "a row appends into a page another row reads";
        for (uint64_t b = 0; b < B; ++b) {
            const uint64_t L = t.seq_lens[b], n = starts[b + 1] - starts[b];
            if (n == 0) continue;
            for (uint64_t i = L / ps; i < pages(L + n); ++i) {
                const uint32_t id = t.block_table[b * per + i];
                if (is_written(id)) return fail(err, Error::execution(twice));
                written[id / 64] |= 1ull << (id % 64);
            }
        }
        for (uint64_t b = 0; b < B; ++b) {
            // cached pages that the row does not append to: none of them is written
            // (an entry that names no page, such as SL_PAGE_NONE, is no page)
            const uint64_t L = t.seq_lens[b], n = starts[b + 1] - starts[b];
            const uint64_t upto = std::min(n != 0 ? L / ps : pages(L), per);
            bool hit = false;
            for (uint64_t i = 0; i < upto; ++i) {
                const uint32_t id = t.block_table[b * per + i];
                hit |= id < kv.num_pages && is_written(id);
            }
            if (hit) return fail(err, Error::execution(twice));
        }
    }
    return true;
}

}  // namespace slhip

namespace {

struct DescView : slhip::BufferView {
    const sl_buffer_desc* table = nullptr;
    size_t n = 0;
    size_t count() const override { return n; }
    const sl_buffer_desc* get(uint32_t id) const override { return id < n ? &table[id] : nullptr; }
};

}  // namespace

extern "C" sl_status sl_hip_validate_paged(const sl_buffer_desc* buffers, size_t n_buffers, uint32_t kind,
                                           const sl_op* op, const sl_op* rope, const sl_buffer_ref* q,
                                           const sl_buffer_ref* k, const sl_buffer_ref* v, const sl_buffer_ref* out,
                                           uint32_t window, uint32_t sinks, const sl_paged_tokens* tokens,
                                           const sl_paged_kv* kv, const uint32_t* row_starts,
                                           const uint32_t* seq_lens, const uint32_t* block_table, sl_error* err) {
    using slhip::Error;
    Error e;
    slhip::PagedPlan plan;
    slhip::PagedCall c;
    c.kind = kind;
    c.op = op;
    c.rope = rope;
    c.tokens = tokens;
    c.kv = kv;
    c.q = q;
    c.k = k;
    c.v = v;
    c.out = out;
    if (kind == SL_PAGED_WINDOW) {
        c.window = window;
        c.sinks = sinks;
    } else if (kind == SL_PAGED_PREFIX) {
        c.prefix = window;
    }
    DescView view;
    view.table = buffers;
    view.n = n_buffers;
    if (kind > SL_PAGED_PREFIX || slhip::paged_argument_missing(c) || row_starts == nullptr || seq_lens == nullptr ||
        block_table == nullptr) {
        e = Error::execution("paged operator received a null argument");
    } else {
        try {
            if (slhip::check_paged_call(view, c, &e))
                (void)slhip::check_paged_contents(c, {row_starts, seq_lens, block_table}, 0, &plan, &e);
        } catch (...) {  // (no memory for the page marks)
            e = Error::out_of_memory(kv->num_pages);
        }
    }
    if (err) {
        err->status = e.status;
        err->buffer = e.buffer;
        err->offset = e.offset;
        err->len = e.len;
        err->requested = e.requested;
        err->op = e.op;
        err->reserved = 0;
        err->message = e.message;
    }
    return e.status;
}
