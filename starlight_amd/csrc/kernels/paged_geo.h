// What the kernels over a paged cache with ragged new tokens share: the
// launch's geometry, how a block finds its row, which keys a block of queries
// reads, and how f32 operands become pairs of fp16 parts.
#pragma once

#include "common.h"
#include "kernels.h"

namespace slhip {
namespace {

// The new tokens of all rows lie one after the other: q and out are
// [tokens, heads, head_dim], row b's tokens are starts[b] .. starts[b + 1],
// the first of them at position lens[b]. The `group` query heads of one KV head
// are handled together, so a row's queries for that head are n * group "query
// rows": query row r is token r / group, head kvh * group + r % group.
struct PagedGeo {
    const uint32_t* starts;
    const uint32_t* lens;
    const uint32_t* table;
    const float* pool;  // the layer's first page: [page][K, V][slot][kv_head][head_dim]
    const float* q;
    float* out;
    float* part;   // partial results [token][head][slot][head_dim], not yet divided by their sums
    float2* ml;    // [token][head][slot]: the partial's largest score and sum of weights
    uint32_t batch, tokens, heads, kv_heads, group, head_dim;
    uint32_t page16, pages_per_seq, num_pages;  // page16: 16-position groups per page
    uint32_t window, sinks;                     // window 0xffffffff: none
    uint32_t kbegin, kend;                      // only keys kbegin <= j < kend
    uint32_t splits, slots, slot0;              // key splits of this launch; slots per query row, the launch's first
    uint32_t aligned;                           // q and out are 16-byte aligned
    uint32_t shared;                            // all tokens are one row's (the shared prefix)
    uint32_t rows_over, rows_upto;              // rows with rows_over < query rows <= rows_upto, the others exit
    float scale;
};

// One block's row and its first query row.
struct PagedItem {
    uint32_t b, len, n, t0, r0;
};

// Item x of a grid with M query rows per item. Row b has the items from
// starts[b] * group / M + b on: at least as many as its query rows need, and
// found from starts alone. Every wave of a block comes to the same answer.
// False: the item has no query rows.
__device__ __forceinline__ bool paged_item(const PagedGeo& g, uint32_t x, uint32_t M, PagedItem* it) {
    const uint32_t lane = threadIdx.x % kWave;
    if (g.shared) {
        // (the first row that has a token: its table names the shared pages)
        uint32_t row = 0;
        for (uint32_t b0 = 0; b0 < g.batch; b0 += kWave) {
            const uint32_t b = b0 + lane;
            const uint64_t some = __ballot(b < g.batch && g.starts[min(b, g.batch - 1) + 1] != 0);
            if (some != 0) {
                row = b0 + static_cast<uint32_t>(__builtin_ctzll(some));
                break;
            }
        }
        it->b = __builtin_amdgcn_readfirstlane(row);
        it->len = g.kend;
        it->n = g.tokens;
        it->t0 = 0;
        it->r0 = x * M;
        return it->r0 < it->n * g.group;
    }
    uint32_t row = 0, start = 0, next = 0, len = 0, base = 0;
    for (uint32_t b0 = 0; b0 < g.batch; b0 += kWave) {
        const uint32_t b = min(b0 + lane, g.batch - 1);
        const uint32_t s = g.starts[b], e = g.starts[b + 1], l = g.lens[b];
        const uint32_t at = s * g.group / M + b;
        const uint64_t below = __ballot(b0 + lane < g.batch && at <= x);
        if (below == 0) break;
        const int last = 63 - __builtin_clzll(below);
        row = b0 + last;
        start = __builtin_amdgcn_readlane(s, last);
        next = __builtin_amdgcn_readlane(e, last);
        len = __builtin_amdgcn_readlane(l, last);
        base = __builtin_amdgcn_readlane(at, last);
        if (below != ~0ull) break;
    }
    // (bounds that hold for checked buffers, and keep a replayed launch in
    // range whatever they hold then)
    next = min(next, g.tokens);
    start = min(start, next);
    const uint32_t capacity = g.pages_per_seq * g.page16 * 16;
    len = min(len, capacity);
    it->b = __builtin_amdgcn_readfirstlane(row);
    it->t0 = start;
    it->n = min(next - start, capacity - len);
    it->len = len;
    it->r0 = (x - base) * M;
    const uint32_t rows = it->n * g.group;
    return it->r0 < rows && rows > g.rows_over && rows <= g.rows_upto;
}

// The keys that the query rows r0 .. r0 + count - 1 of an item see, as a list of
// groups of 16 positions (position / 16), none of them without a visible key:
// the sinks' groups, then those from the first key of the first query's window
// to the last query's own.
struct PagedKeys {
    uint32_t sink_groups, first_group, groups, end;
    __device__ __forceinline__ uint32_t group(uint32_t x) const {
        return x < sink_groups ? x : first_group + (x - sink_groups);
    }
};
__device__ __forceinline__ PagedKeys paged_keys(const PagedGeo& g, const PagedItem& it, uint32_t r0, uint32_t count) {
    const uint32_t lo = it.len + r0 / g.group, hi = it.len + (r0 + count - 1) / g.group;
    PagedKeys k;
    k.end = min(hi + 1, g.kend);
    const uint32_t first = max(lo >= g.window ? lo - g.window + 1 : 0, g.kbegin);
    k.first_group = first / 16;
    k.sink_groups = min((g.sinks + 15) / 16, k.first_group);
    const uint32_t last = (k.end + 15) / 16;
    k.groups = k.sink_groups + (last > k.first_group ? last - k.first_group : 0);
    return k;
}

// Which keys a query at `position` sees: j < end and (j >= low or j < sinks).
struct PagedMask {
    uint32_t low, end;
};
__device__ __forceinline__ PagedMask paged_mask(const PagedGeo& g, uint32_t position) {
    return {max(position >= g.window ? position - g.window + 1 : 0, g.kbegin), min(position + 1, g.kend)};
}
__device__ __forceinline__ bool paged_sees(const PagedMask& m, uint32_t sinks, uint32_t j) {
    return j < m.end && (j >= m.low || j < sinks);
}

// First element of the K rows of group `grp` (positions 16 grp ..) of row b for
// KV head kvh; a position's row is kv_heads * head_dim further, V one page half.
__device__ __forceinline__ const float* paged_group(const PagedGeo& g, uint32_t b, uint32_t grp, uint32_t kvh) {
    const uint32_t pi = min(grp / g.page16, g.pages_per_seq - 1);
    const uint32_t page = min(g.table[static_cast<uint64_t>(b) * g.pages_per_seq + pi], g.num_pages - 1);
    const uint64_t row = static_cast<uint64_t>(g.kv_heads) * g.head_dim;
    return g.pool + (static_cast<uint64_t>(page) * 2 * g.page16 + grp % g.page16) * 16 * row +
           static_cast<uint64_t>(kvh) * g.head_dim;
}
__device__ __forceinline__ uint64_t paged_v_offset(const PagedGeo& g) {
    return static_cast<uint64_t>(g.page16) * 16 * g.kv_heads * g.head_dim;
}

// ---- f32 operands as two fp16 parts ----
//
// x 2^e = h + l with h and l in fp16, each rounded to nearest: 11 + 11
// significant bits, so a product of two such operands from the three products
// h h, h l, l h is off by about 2^-22 of itself at most and 2^-23.5 in the
// mean (the left-out l l and the roundings of l), like products of rounded f32
// numbers. fp16's range is met by the scale: e brings the largest value of a
// block of operands to 2^14 .. 2^15, and what lies 2^-39 below that is lost, as
// it would be in f32 sums. Three fp16 matrix products cost a third of what f32's
// matrix instructions do.
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kPartTop = 14;  // the largest value's exponent after scaling

// The scale's exponent for a block whose largest magnitude is `most` (finite):
// between -113 and 60, so that the scales of two operands can be multiplied.
__device__ __forceinline__ int part_exponent(float most) {
    const int e = static_cast<int>(__float_as_uint(most) >> 23) - 127;
    return max(min(kPartTop - e, 60), kPartTop - 127);
}
__device__ __forceinline__ float power2(int e) {  // 2^e, 0 and infinity outside f32's normal numbers
    return e < -126 ? 0.f : e > 127 ? INFINITY : __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
__device__ __forceinline__ void put_parts(float x, float y, float scale, v8h& h, v8h& l, int i) {
    const float a = x * scale, b = y * scale;
    const _Float16 ha = static_cast<_Float16>(a), hb = static_cast<_Float16>(b);
    h[i] = ha;
    h[i + 1] = hb;
    l[i] = static_cast<_Float16>(a - static_cast<float>(ha));
    l[i + 1] = static_cast<_Float16>(b - static_cast<float>(hb));
}
__device__ __forceinline__ float max_abs(float m, float4 v) {
    m = fmaxf(fmaxf(m, fabsf(v.x)), fabsf(v.y));
    return fmaxf(fmaxf(m, fabsf(v.z)), fabsf(v.w));
}

__device__ __forceinline__ float4 scaled4(float4 v, float f) { return make_float4(v.x * f, v.y * f, v.z * f, v.w * f); }
__device__ __forceinline__ void fma4(float4& acc, float f, float4 v) {
    acc.x = fmaf(v.x, f, acc.x);
    acc.y = fmaf(v.y, f, acc.y);
    acc.z = fmaf(v.z, f, acc.z);
    acc.w = fmaf(v.w, f, acc.w);
}
__device__ __forceinline__ float4 load4(const float* p, bool aligned) {
    if (aligned) return *reinterpret_cast<const float4*>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}
__device__ __forceinline__ void store4(float* p, float4 v, bool aligned) {
    if (aligned) {
        *reinterpret_cast<float4*>(p) = v;
    } else {
        p[0] = v.x;
        p[1] = v.y;
        p[2] = v.z;
        p[3] = v.w;
    }
}

}  // namespace
}  // namespace slhip
