// What the kernels over a paged cache with ragged new tokens share: the
// launch's geometry, how a block finds its row, which keys a block of queries
// reads, and how f32 operands become pairs of fp16 parts.
#pragma once

#include "common.h"
#include "kernels.h"

namespace slhip {

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
    float2* ml;    // [token][head][slot]: the partial's largest exponent and sum of weights
    uint32_t batch, tokens, heads, kv_heads, group, head_dim;
    uint32_t page16, pages_per_seq, num_pages;  // page16: 16-position groups per page,
    uint32_t page_shift;                        // its logarithm, or 32 where it is no power of two
    uint32_t window, sinks;                     // window 0xffffffff: none
    // A launch's units of work, kv_heads blocks each: own_items x splits (own_items at least as
    // many as there are), each row's queries over its positions from `prefix` on (first: their
    // lengths differ); then shared_items x
    // shared_splits, all tokens' queries over the positions below `prefix`, which lie in the same
    // pages for every row.
    uint32_t prefix, shared_items, shared_splits, own_items, splits;
    // Own items in whole rounds of round_items, the rest of them split by tail_splits (1: not).
    uint32_t round_items, tail_splits;
    // Partials a query row has room for, the shared first. A row that leaves the later of
    // them ends its list with a sum of -1 (not split and no prefix: at once, its result is written).
    uint32_t slots;
    uint32_t uneven;                            // rows have fewer partials than slots
    uint32_t aligned;                           // q and out are 16-byte aligned
    uint32_t rows_over, rows_upto;              // rows with rows_over < query rows <= rows_upto, the others exit
    float scale;
};

// paged_tiles.hip: the form for many query rows per KV head, kTileRows per block, head_dim up to
// 128.
constexpr uint32_t kTileRows = 256;
hipError_t launch_paged_tiles(const PagedGeo& g, hipStream_t s);

inline unsigned paged_blocks(const PagedGeo& g) {
    return (g.shared_items * g.shared_splits + g.own_items * g.splits) * g.kv_heads;
}

namespace {

// One block's row, its first query row, and which keys it takes: begin <= j < end, split
// number `split` of `splits`, whose partial is `slot`.
struct PagedItem {
    uint32_t b, len, n, t0, r0;
    uint32_t begin, end, splits, split, slot;
};

// The rows b0 .. b0 + 63, one per lane: a row's tokens and length, how many items of M query
// rows it makes here (none where its kind is another launch's), and how many the rows before it
// in the 64 make.
struct PagedRow {
    uint32_t start, n, len, items, before;
};
__device__ __forceinline__ PagedRow paged_row(const PagedGeo& g, uint32_t b0, uint32_t M) {
    const uint32_t lane = threadIdx.x % kWave, b = min(b0 + lane, g.batch - 1);
    // (bounds that hold for checked buffers, and keep a replayed launch in range whatever
    // they hold then)
    const uint32_t capacity = g.pages_per_seq * g.page16 * 16, next = min(g.starts[b + 1], g.tokens);
    PagedRow r;
    r.start = min(g.starts[b], next);
    r.len = min(g.lens[b], capacity);
    r.n = min(next - r.start, capacity - r.len);
    const uint32_t rows = r.n * g.group;
    const bool mine = b0 + lane < g.batch && rows > g.rows_over && rows <= g.rows_upto;
    r.items = mine ? (rows + M - 1) / M : 0;
    const uint64_t one = __ballot(r.items != 0);
    if (__ballot(r.items > 1) == 0) {  // wave-uniform
        r.before = __popcll(one & ((1ull << lane) - 1));
    } else {
        uint32_t sum = r.items;
#pragma unroll
        for (uint32_t d = 1; d < kWave; d *= 2) {
            const uint32_t below = __shfl_up(sum, d);
            sum += lane >= d ? below : 0;
        }
        r.before = sum - r.items;
    }
    return r;
}
__device__ __forceinline__ uint32_t paged_row_items(const PagedRow& r) {  // of the 64 rows
    return __builtin_amdgcn_readlane(r.before + r.items, kWave - 1);
}

// Unit `unit` of a launch with M query rows per item (LAST_FIRST: the own items from the last to
// the first). The items are counted from the row starts, so those that there are lie side by side
// whatever the rows: blocks without work between the others would leave some of the chip's
// shader engines, which are given blocks in turn, with one block more than they have CUs
// (256 blocks of paged_tiles 98 us, not 70). Every wave of a block comes to the same answer.
// False: nothing to do.
template <bool LAST_FIRST>
__device__ __forceinline__ bool paged_item(const PagedGeo& g, uint32_t unit, uint32_t M, PagedItem* it) {
    const uint32_t own_units = g.own_items * g.splits;
    if (unit >= own_units) {
        unit -= own_units;
        it->split = unit / g.shared_items;
        it->begin = 0;
        it->end = g.prefix;
        it->splits = g.shared_splits;
        it->slot = it->split;
        // (the first row that has a token: its table names the shared pages)
        uint32_t row = 0;
        for (uint32_t b0 = 0; b0 < g.batch; b0 += kWave) {
            const uint32_t b = b0 + threadIdx.x % kWave;
            const uint64_t some = __ballot(b < g.batch && g.starts[min(b, g.batch - 1) + 1] != 0);
            if (some != 0) {
                row = b0 + static_cast<uint32_t>(__builtin_ctzll(some));
                break;
            }
        }
        it->b = __builtin_amdgcn_readfirstlane(row);
        it->len = g.prefix;
        it->n = g.tokens;
        it->t0 = 0;
        it->r0 = (unit - it->split * g.shared_items) * M;
        return it->r0 < it->n * g.group;
    }
    PagedRow r = paged_row(g, 0, M);
    uint32_t x = unit, first = 0;
    it->split = 0;
    it->splits = g.splits;
    if (LAST_FIRST || g.splits != 1) {
        uint32_t total = paged_row_items(r);
        for (uint32_t b0 = kWave; b0 < g.batch; b0 += kWave) total += paged_row_items(paged_row(g, b0, M));
        if (LAST_FIRST && g.tail_splits > 1) {
            const uint32_t tail = total % g.round_items, whole = total - tail;
            if (unit >= whole + tail * g.tail_splits) return false;
            if (unit >= whole) {
                it->splits = g.tail_splits;
                it->split = (unit - whole) / tail;
                x -= it->split * tail;
            }
        } else if (unit >= total * g.splits) {
            return false;
        } else if (g.splits != 1) {
            it->split = unit / total;
            x -= it->split * total;
        }
        if (LAST_FIRST) x = total - 1 - x;
    }
    for (uint32_t here = paged_row_items(r); x >= here && first + kWave < g.batch; here = paged_row_items(r)) {
        x -= here;
        first += kWave;
        r = paged_row(g, first, M);
    }
    const uint64_t found = __ballot(x >= r.before && x < r.before + r.items);
    if (found == 0) return false;
    const int at = __builtin_ctzll(found);
    it->begin = g.prefix;
    it->end = 0xffffffffu;
    it->slot = (g.prefix != 0 ? g.shared_splits : 0) + it->split;
    it->b = first + at;
    it->t0 = __builtin_amdgcn_readlane(r.start, at);
    it->n = __builtin_amdgcn_readlane(r.n, at);
    it->len = __builtin_amdgcn_readlane(r.len, at);
    it->r0 = (x - __builtin_amdgcn_readlane(r.before, at)) * M;
    return true;
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
    k.end = min(hi + 1, it.end);
    const uint32_t first = max(lo >= g.window ? lo - g.window + 1 : 0, it.begin);
    k.first_group = first / 16;
    k.sink_groups = min((g.sinks + 15) / 16, k.first_group);
    const uint32_t last = (k.end + 15) / 16;
    k.groups = k.sink_groups + (last > k.first_group ? last - k.first_group : 0);
    return k;
}

// Whether the item's results are written, not partials.
__device__ __forceinline__ bool paged_direct(const PagedGeo& g, const PagedItem& it) {
    return it.splits == 1 && g.prefix == 0;
}
// The partial `slot` of a query row (token and head), its values written by the caller; `m` and
// `l` are not looked at for a result.
__device__ __forceinline__ void paged_state(const PagedGeo& g, const PagedItem& it, uint64_t row, float m, float l) {
    float2* const ml = g.ml + row * g.slots;
    if (paged_direct(g, it)) {
        if (g.slots > 1) ml[0] = make_float2(0.f, -1.f);
        return;
    }
    ml[it.slot] = make_float2(m, l);
    if (g.prefix == 0 && it.split == 0 && it.splits < g.slots) ml[it.splits] = make_float2(0.f, -1.f);
}

// Which keys a query at `position` sees: j < end and (j >= low or j < sinks).
struct PagedMask {
    uint32_t low, end;
};
__device__ __forceinline__ PagedMask paged_mask(const PagedGeo& g, const PagedItem& it, uint32_t position) {
    return {max(position >= g.window ? position - g.window + 1 : 0, it.begin), min(position + 1, it.end)};
}
__device__ __forceinline__ bool paged_sees(const PagedMask& m, uint32_t sinks, uint32_t j) {
    return j < m.end && (j >= m.low || j < sinks);
}

// The kernel's geometry, its only argument, read again: what only the end of a
// kernel needs would otherwise hold scalar registers through its loop.
__device__ __forceinline__ PagedGeo geometry_again() {
    typedef __attribute__((address_space(4))) const uint64_t word;
    word* p = (word*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    struct Words {
        uint64_t w[sizeof(PagedGeo) / 8];
    } words;
    static_assert(sizeof(PagedGeo) % 8 == 0, "whole words");
#pragma unroll
    for (size_t i = 0; i < sizeof(PagedGeo) / 8; ++i) words.w[i] = p[i];
    return __builtin_bit_cast(PagedGeo, words);
}

// Which keys an item takes, in one register through a kernel's loop, and again from it. (In six,
// more of the loop's were spilled: 1.5% of paged_tiles. All that its end needs in LDS: 1%.)
__device__ __forceinline__ uint32_t paged_pack(const PagedItem& it) {
    uint32_t part = it.slot | it.split << 8 | it.splits << 16 | (it.end != 0xffffffffu ? 1u << 31 : 0);
    asm volatile("" : "+s"(part));
    return part;
}
__device__ __forceinline__ void paged_unpack(const PagedGeo& g, uint32_t part, PagedItem* it) {
    const bool shared = part >> 31 != 0;
    it->slot = part & 255;
    it->split = part >> 8 & 255;
    it->splits = part >> 16 & 255;
    it->begin = shared ? 0 : g.prefix;
    it->end = shared ? g.prefix : 0xffffffffu;
}

// Word i of a table that no kernel writes, the same for the whole wave: a scalar load.
__device__ __forceinline__ uint32_t uniform_word(const uint32_t* table, uint64_t i) {
    typedef __attribute__((address_space(4))) const uint32_t word;
    const uint64_t at = reinterpret_cast<uint64_t>(table + i);
    // (the builtin returns a signed value: widened as it is, it would fill the upper half)
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at)),
                   hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32));
    return *reinterpret_cast<word*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// First element of the K rows of group `grp` (positions 16 grp ..) of row b for
// KV head kvh (all uniform over the wave); a position's row is kv_heads * head_dim further, V one page half.
__device__ __forceinline__ const float* paged_group(const PagedGeo& g, uint32_t b, uint32_t grp, uint32_t kvh) {
    const uint32_t whole = g.page_shift < 32 ? grp >> g.page_shift : grp / g.page16;
    const uint32_t pi = min(whole, g.pages_per_seq - 1);
    const uint32_t page = min(uniform_word(g.table, static_cast<uint64_t>(b) * g.pages_per_seq + pi), g.num_pages - 1);
    const uint64_t row = static_cast<uint64_t>(g.kv_heads) * g.head_dim;
    return g.pool + (static_cast<uint64_t>(page) * 2 * g.page16 + (grp - whole * g.page16)) * 16 * row +
           static_cast<uint64_t>(kvh) * g.head_dim;
}
// Of a buffer resource: 32-bit words, no swizzle.
constexpr int kBufferFlags = 0x00027000;
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
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

// So rows (one position's keys or values) that share a scale have to be of like magnitude, for a
// query may see the small ones and not the large, and so have the values' columns, each a result
// of its own: where one of them, not all zero, is kApart below the largest value beside it,
// the plain form takes over.
constexpr int kPartTop = 14;  // the largest value's exponent after scaling
constexpr float kApart = 0x1p-16f;
// O's unit is lowered as larger values come, and raised again by more than this.
constexpr int kUnitSlack = 8;
// Whether one of the rows that N lanes hold together is such a one; m: the largest of the lane's values.
template <int N>
__device__ __forceinline__ bool row_apart(float m, float most) {
    const uint64_t small = __ballot(m < most * kApart), zero = __ballot(m == 0.f);
    bool apart = false;
#pragma unroll
    for (int at = 0; at < 64; at += N) {
        const uint64_t lanes = ((1ull << N) - 1) << at;
        apart |= (small & lanes) == lanes && (zero & lanes) != lanes;
    }
    return apart;
}

// The scale's exponent for a block whose largest magnitude is `most` (finite):
// between -113 and 60, so that the scales of two operands can be multiplied.
__device__ __forceinline__ int part_exponent(float most) {
    const int e = static_cast<int>(__float_as_uint(most) >> 23) - 127;
    return max(min(kPartTop - e, 60), kPartTop - 127);
}
__device__ __forceinline__ float power2(int e) {  // 2^e, 0 and infinity outside f32's normal numbers
    return e < -126 ? 0.f : e > 127 ? INFINITY : __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
// Both parts of eight values: x scale - h is exact before it is rounded. (Packed
// conversions and mixed multiply-adds; one multiply-add per part that rounds to fp16
// itself, a mix instruction of half the rate, measured 2-3% slower throughout.)
struct Parts {
    v8h h, l;
};
__device__ __forceinline__ Parts to_parts(float x0, float x1, float x2, float x3, float x4, float x5, float x6, float x7,
                                          float scale) {
    const float x[8] = {x0, x1, x2, x3, x4, x5, x6, x7};
    Parts p;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const v2h hp = __builtin_convertvector(v2f{x[i] * scale, x[i + 1] * scale}, v2h);
        const v2h lp = __builtin_convertvector(
            v2f{fmaf(x[i], scale, -static_cast<float>(hp[0])), fmaf(x[i + 1], scale, -static_cast<float>(hp[1]))}, v2h);
        p.h[i] = hp[0];
        p.h[i + 1] = hp[1];
        p.l[i] = lp[0];
        p.l[i + 1] = lp[1];
    }
    return p;
}
__device__ __forceinline__ Parts to_parts(float4 a, float4 b, float scale) {
    return to_parts(a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, scale);
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
// N float4 of a row, `at(i)` elements in, zeros from element `dims` on: all loads
// together, under one branch (a branch each would wait for each).
template <int N, bool EXACT, typename At>
__device__ __forceinline__ void load_row(const float* row, bool aligned, uint32_t dims, float4 (&x)[N], At at) {
    if (aligned) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            x[i] = EXACT || at(i) < dims ? *reinterpret_cast<const float4*>(row + at(i)) : make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            x[i] = EXACT || at(i) < dims ? load4(row + at(i), false) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
}
// Whether a value of x is a NaN (max_abs passes over them).
template <int N>
__device__ __forceinline__ bool any_nan(const float4 (&x)[N]) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < N; ++i) nan |= (x[i].x != x[i].x) | (x[i].y != x[i].y) | (x[i].z != x[i].z) | (x[i].w != x[i].w);
    return nan;
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

// Exponents beyond this have no fraction worth the name, and the largest one's rounding
// error would reach the weights' range: left to the plain form.
constexpr float kExponentMost = 134217728.f;

constexpr int kWeightTop = 14;  // weights reach fp16 as up to 2^14

// One wave's tiles in plain f32: lane l works on query l % 16, in `o` (that
// query's row in LDS) on the dims 4 i + l / 16, which no other lane touches.
// m in units of the weights' exponents, as in the fast form.
__device__ __forceinline__ void slow_tiles(const PagedGeo& g, const PagedKeys& keys, uint32_t b, uint32_t kvh,
                                           uint32_t tile0, uint32_t tiles, uint32_t step, const float* qrow,
                                           PagedMask mask, float c2, float* o, float& m, float& l) {
    const int lane = threadIdx.x % kWave, c = lane % 16, kk = lane / 16;
    const uint64_t row = static_cast<uint64_t>(g.kv_heads) * g.head_dim;
    m = -INFINITY;
    l = 0.f;
    for (uint32_t d = kk; d < g.head_dim; d += 4) o[d] = 0.f;
    for (uint32_t tile = tile0; tile < tiles; tile += step) {
        float p[8];
        float tmax = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t x = 2 * tile + i / 4;
            p[i] = -INFINITY;
            if (x >= keys.groups) continue;
            if (!paged_sees(mask, g.sinks, keys.group(x) * 16 + 4 * kk + i % 4)) continue;
            const float* k = paged_group(g, b, keys.group(x), kvh) + (4 * kk + i % 4) * row;
            float dot = 0.f;
#pragma unroll 1
            for (uint32_t d = 0; d < g.head_dim; ++d) dot = fmaf(qrow[d], k[d], dot);
            p[i] = (g.scale < 0.f ? -dot : dot) * c2;
            tmax = fmaxf(tmax, p[i]);
        }
        tmax = fmaxf(tmax, lane_xor16(tmax));
        tmax = fmaxf(tmax, lane_xor32(tmax));
        const float before = m;
        m = fmaxf(before, tmax);
        const float corr = before == -INFINITY ? 0.f : exp2f(before - m);
        l *= corr;
        if (corr != 1.f)
            for (uint32_t d = kk; d < g.head_dim; d += 4) o[d] *= corr;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t x = 2 * tile + i / 4;
            const bool seen = x < keys.groups && paged_sees(mask, g.sinks, keys.group(x) * 16 + 4 * kk + i % 4);
            p[i] = seen ? exp2f(p[i] - m) : 0.f;
            l += p[i];
        }
#pragma unroll 1
        for (int i = 0; i < 32; ++i) {
            const uint32_t x = 2 * tile + i / 16;
            if (x >= keys.groups) break;
            // the weight of key i for query c, from the lane that holds it
            float w = 0.f;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const float v = __shfl(p[r], c + 16 * (i % 16 / 4));
                w = r == i / 16 * 4 + i % 4 ? v : w;
            }
            if (!paged_sees(mask, g.sinks, keys.group(x) * 16 + i % 16)) continue;
            const float* v = paged_group(g, b, keys.group(x), kvh) + paged_v_offset(g) + (i % 16) * row;
#pragma unroll 1
            for (uint32_t d = kk; d < g.head_dim; d += 4) o[d] = fmaf(w, v[d], o[d]);
        }
    }
}

}  // namespace
}  // namespace slhip
