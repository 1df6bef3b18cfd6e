// Attention of ragged new tokens over a paged cache (reference/attention.rs:
// 129-219 for the mathematics; the pages, window, sinks and shared prefix have
// no reference counterpart).
//
// A query at position p sees the keys j <= p that lie in its window (j > p - W)
// or among the sinks (j < S); o = sum_j softmax_j(scale q.k_j) v_j, in one pass over
// the keys with a running maximum.
//
// paged_rows serves up to 16 query rows (token, query head of one KV head) per
// block: its waves take 32-key tiles of their own, K and V going from the
// pages straight into registers in matrix operand order, and their states are
// combined at the end. Long key ranges are split over `splits` blocks, whose
// partials paged_merge combines.
//   S^T = K Q^T: 16 keys x 32 dims (A) by 32 dims x 16 queries (B). Lane l
//     holds key l % 16 and dims 32 j + 4 (l / 16) .. and 16 further (two float4
//     of one row), the queries alike: the order of the dims in the sum is free.
//   O^T += V^T P^T: 16 dims x 32 keys (A) by 32 keys x 16 queries (B). S^T leaves
//     lane l with the keys 4 (l / 16) + i of each group and query l % 16, which is B
//     as it stands; for A the lane loads the float4 at dims 64 J + 4 (l % 16) of those
//     same keys, its element e being column l % 16 of dim tile (J, e).
// Every operand is two fp16 parts (paged_geo.h). Bound by HBM: splitting costs
// about four vector instructions per K/V element, a fifth of the time the
// element takes to arrive. 16 rows of the 8B shape behind windows of 4,096 (493 MB): 89 us,
// more than the rate of a large copy (4.9 TB/s).
//
// A tile whose values are not finite, or a result that is not a number, sends
// the wave back over its tiles in plain f32 (slow_tiles), where a key that a query
// does not see contributes nothing whatever it holds.
#include <algorithm>

#include "paged_geo.h"

namespace slhip {
namespace {

// EXACT: head_dim is 64 DV; else it is smaller, a multiple of 16, and the dims past it
// are zeros. NW: waves (8 where LDS and registers have room for two blocks per CU's waves).
template <int DV, bool EXACT, int NW>
__global__ __launch_bounds__(64 * NW, DV <= 2 ? 2 : 1) void paged_rows(PagedGeo g) {
    prefetch_kernarg<arg_bytes<PagedGeo>()>();
    constexpr int KS = 2 * DV;     // 32-dim steps of a score
    constexpr int DT = 4 * DV;     // 16-dim tiles of the result
    constexpr uint32_t M = 16;     // query rows
    constexpr int OROW = 64 * DV + 4;
    __shared__ __align__(16) float so[NW][M][OROW];
    __shared__ float sml[NW][M][2];
    PagedItem it;
    if (!paged_item<false>(g, blockIdx.x / g.kv_heads, M, &it)) return;  // block-uniform
    const int tid = threadIdx.x, lane = tid % kWave, c = lane % 16, kk = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t kvh = blockIdx.x % g.kv_heads, D = g.head_dim, G = g.group;
    const uint32_t count = min(M, it.n * G - it.r0);
    const PagedKeys keys = paged_keys(g, it, it.r0, count);
    const uint32_t tiles = (keys.groups + 1) / 2;
    const uint32_t kv_bytes = g.kv_heads * D * 4;
    const bool aligned = g.aligned != 0;
    const uint32_t r = it.r0 + min(static_cast<uint32_t>(c), count - 1);  // query c (those past the last repeat it)
    const auto row_of = [&](uint32_t r) -> uint64_t {
        return static_cast<uint64_t>(it.t0 + r / G) * g.heads + kvh * G + r % G;
    };
    const float* const qrow = g.q + row_of(r) * D;
    const PagedMask mask = paged_mask(g, it, it.len + r / G);

    float4 kx[2][KS][2], vx[8][DV];
    // A missing second group re-reads the first (its scores are masked); rows past the last
    // key are out of the buffer's range and read as zeros.
    const auto group_rows = [&](uint32_t tile, int s, bool values) {
        const uint32_t grp = keys.group(min(2 * tile + s, keys.groups - 1));
        const float* const at = paged_group(g, it.b, grp, kvh);
        const uint32_t rows_in = min(keys.end - 16 * grp, 16u);
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(values ? at + paged_v_offset(g) : at), 0,
                                                 (rows_in - 1) * kv_bytes + 4 * D, kBufferFlags);
    };
    const auto load_k = [&](uint32_t tile) {
        const uint32_t own = c * kv_bytes + 16 * kk;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const auto rsrc = group_rows(tile, s, false);
#pragma unroll
            for (int j = 0; j < 2 * KS; ++j)
                kx[s][j / 2][j % 2] = EXACT || 16u * j < D
                                          ? __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, own + 64 * j, 0, 0))
                                          : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    const auto load_v = [&](uint32_t tile) {
        const uint32_t own = 4 * kk * kv_bytes + 16 * c;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const auto rsrc = group_rows(tile, s, true);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int J = 0; J < DV; ++J)
                    vx[4 * s + i][J] = EXACT || 64 * J + 4 * c < D
                                           ? __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, own + 256 * J, i * kv_bytes, 0))
                                           : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    // When a tile's rows are asked for: at head_dim 64 as soon as the registers of the tile
    // before are free, at 128 K and V together (any earlier and they would be spilled), above V
    // after the scores.
    constexpr bool kAhead = DV == 1, kTogether = DV <= 2;
    const uint32_t tile0 = it.split * NW + wave, step = NW * it.splits;
    if (kAhead && tile0 < tiles) {
        load_k(tile0);
        load_v(tile0);
    }
    v8h qh[KS], ql[KS];
    int qe;
    bool bad = false;
    float4 x[2 * KS];
    load_row<2 * KS, EXACT>(qrow, aligned, D, x, [&](int j) { return 16u * j + 4 * kk; });
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < 2 * KS; ++j) most = max_abs(most, x[j]);
    most = fmaxf(most, lane_xor16(most));
    most = fmaxf(most, lane_xor32(most));
    uint32_t flag = any_nan(x) || most == INFINITY;
    asm volatile("" : "+v"(flag));  // (here, not at the end: it would keep the row in registers)
    bad |= flag != 0;
    qe = part_exponent(most);
    // a negative factor goes into the queries, so that the largest score is the largest sum
    const float scale = g.scale < 0.f ? -power2(qe) : power2(qe);
#pragma unroll
    for (int j = 0; j < KS; ++j) {
        const Parts p = to_parts(x[2 * j], x[2 * j + 1], scale);
        qh[j] = p.h;
        ql[j] = p.l;
    }
    const float c2 = fabsf(g.scale) * 1.4426950408889634f;
    // The state: query c's largest exponent, this lane's keys' part of the sum, and O^T in units
    // of 2^-oexp: o[4 J + e][i] is dim 64 J + 16 kk + 4 i + e.
    float m = -INFINITY, l = 0.f;
    v4f o[DT];
    int oexp = 0;
    bool first = true;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = v4f{0.f, 0.f, 0.f, 0.f};
#define SL_F16(a, b, x) __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, x, 0, 0, 0)
    for (uint32_t tile = tile0; tile < tiles; tile += step) {
        const bool more = tile + step < tiles;  // wave-uniform
        if (!kAhead) {
            load_k(tile);
            if (kTogether) load_v(tile);
        }
        // scores
        float row[2] = {0.f, 0.f};  // the lane's two keys' largest values
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < KS; ++j) row[s] = max_abs(max_abs(row[s], kx[s][j][0]), kx[s][j][1]);
        float most = wave_max(fmaxf(row[0], row[1]));
        bad |= most == INFINITY;
        const auto small = [&](float x) { return x < most * kApart && x != 0.f; };
        if (__builtin_expect(__any(small(row[0]) || small(row[1])), 0)) {  // wave-uniform; seldom
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                row[s] = fmaxf(row[s], lane_xor16(row[s]));
                row[s] = fmaxf(row[s], lane_xor32(row[s]));
                bad |= small(row[s]);
            }
        }
        const int ke = part_exponent(most);
        const float kscale = power2(ke);
        v4f sc[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            Parts k[KS];
#pragma unroll
            for (int j = 0; j < KS; ++j) k[j] = to_parts(kx[s][j][0], kx[s][j][1], kscale);
            // the small products first, so that a large sum rounds once per step
            v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                x = SL_F16(k[j].l, qh[j], x);
                x = SL_F16(k[j].h, ql[j], x);
            }
#pragma unroll
            for (int j = 0; j < KS; ++j) x = SL_F16(k[j].h, qh[j], x);
            sc[s] = x;
        }
        if (kAhead && more) load_k(tile + step);
        if (!kTogether) load_v(tile);
        // Weights are 2^(x c2 - m), x in the tile's units (an exact power of two apart from q.k's):
        // m, the largest x c2 so far once rounded, is the same number in every tile and split. A
        // query may see none of the keys so far (m = -inf): weights and corr are 0.
        float p[8];
        const uint32_t ga = keys.group(2 * tile), gb = keys.group(min(2 * tile + 1, keys.groups - 1));
        const bool both = 2 * tile + 1 < keys.groups;
        float tmax = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t j = 16 * (i < 4 ? ga : gb) + 4 * kk + i % 4;
            p[i] = (i < 4 || both) && paged_sees(mask, g.sinks, j) ? sc[i / 4][i % 4] : -INFINITY;
            tmax = fmaxf(tmax, p[i]);
        }
        tmax = fmaxf(tmax, lane_xor16(tmax));
        tmax = fmaxf(tmax, lane_xor32(tmax));
        const float ct = ldexpf(c2, -qe - ke);
        const float m_new = tmax == -INFINITY ? m : fmaxf(m, tmax * ct);
        const float corr = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        bad |= fabsf(m_new) > kExponentMost && m_new != -INFINITY;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float w = p[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(fmaf(p[i], ct, -m_new));
            sum += w;
            p[i] = w;
        }
        l = l * corr + sum;
        // values
        most = 0.f;
        float least = INFINITY;
        const auto largest = [&](int i) {  // of the lane's values of one key
            float x = 0.f;
#pragma unroll
            for (int J = 0; J < DV; ++J) x = max_abs(x, vx[i][J]);
            return x;
        };
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = largest(i);
            most = fmaxf(most, x);
            least = fminf(least, x == 0.f ? INFINITY : x);  // (zeros: past the last key)
        }
        most = wave_max(most);
        bad |= most == INFINITY;
        if (__builtin_expect(__any(least < most * kApart), 0)) {  // wave-uniform; seldom
#pragma unroll
            for (int i = 0; i < 8; ++i) bad |= row_apart<16>(largest(i), most);
#pragma unroll
            for (int J = 0; J < DV; ++J) {
                const auto joined = [&](auto at) {  // of a column
                    float x = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) x = fmaxf(x, fabsf(at(vx[i][J])));
                    x = fmaxf(x, lane_xor16(x));
                    return fmaxf(x, lane_xor32(x));
                };
                const float x = joined([](float4 v) { return v.x; }), y = joined([](float4 v) { return v.y; }),
                            z = joined([](float4 v) { return v.z; }), w = joined([](float4 v) { return v.w; });
                const float limit = most * kApart;
                bad |= (x < limit && x != 0.f) || (y < limit && y != 0.f) || (z < limit && z != 0.f) ||
                       (w < limit && w != 0.f);
            }
        }
        // O's unit: the weights' 2^14 times the values' scale
        const int need = part_exponent(most), held = first ? need : oexp - kWeightTop;
        const int ve = most != 0.f && (need < held || need > held + kUnitSlack) ? need : held;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= corr;
        if (__builtin_expect(ve != held, 0)) {  // wave-uniform
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][i] = __builtin_ldexpf(o[d][i], ve - held);
        }
        first = false;
        oexp = ve + kWeightTop;
        const Parts w = to_parts(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], power2(kWeightTop));
        const float vscale = power2(ve);
#pragma unroll
        for (int J = 0; J < DV; ++J)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const auto at = [&](int i) { return reinterpret_cast<const float*>(&vx[i][J])[e]; };
                const Parts v = to_parts(at(0), at(1), at(2), at(3), at(4), at(5), at(6), at(7), vscale);
                v4f x = o[4 * J + e];
                x = SL_F16(v.l, w.h, x);
                x = SL_F16(v.h, w.l, x);
                o[4 * J + e] = SL_F16(v.h, w.h, x);
            }
        if (kAhead && more) load_v(tile + step);
    }
#undef SL_F16
    const float back = power2(-oexp);
    float check = 0.f;
    check += l;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        o[d] *= back;
        check += (o[d][0] + o[d][1]) + (o[d][2] + o[d][3]);
    }
    // (an infinite check of finite values, near f32's end, only costs time)
    bad |= !(fabsf(check) < INFINITY);
    if (__any(bad)) {  // wave-uniform
        slow_tiles(g, keys, it.b, kvh, tile0, tiles, step, qrow, mask, c2, so[wave][c], m, l);
    } else {
#pragma unroll
        for (int J = 0; J < DV; ++J)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(&so[wave][c][64 * J + 16 * kk + 4 * i]) =
                    make_float4(o[4 * J][i], o[4 * J + 1][i], o[4 * J + 2][i], o[4 * J + 3][i]);
    }
    l += lane_xor16(l);
    l += lane_xor32(l);
    if (kk == 0) {
        sml[wave][c][0] = m;
        sml[wave][c][1] = l;
    }
    __syncthreads();
    const uint32_t d4 = D / 4;
    for (uint32_t i = tid; i < count * d4; i += 64 * NW) {
        const uint32_t x = i / d4, d = 4 * (i % d4);
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) mm = fmaxf(mm, sml[w][x][0]);
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float mw = sml[w][x][0];
            // (an empty state weighs nothing; a NaN maximum keeps its sum's NaN)
            const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - mm);
            sum = fmaf(sml[w][x][1], f, sum);
            if (f != 0.f) fma4(acc, f, *reinterpret_cast<const float4*>(&so[w][x][d]));
        }
        const uint64_t at = row_of(it.r0 + x);
        if (paged_direct(g, it)) store4(g.out + at * D + d, scaled4(acc, 1.0f / sum), aligned);
        else *reinterpret_cast<float4*>(g.part + (at * g.slots + it.slot) * D + d) = acc;
        if (d == 0) paged_state(g, it, at, mm, sum);
    }
}

// Combines the partials of each query row. A block has up to 16 query rows, a
// thread one float4 of one of them. The (m, sum) pairs of its rows come
// to LDS while the first partials are on their way; the weights 2^(m - max) / sum
// are worked out once per row and partial.
constexpr uint32_t kMergeRows = 16, kMergeSlots = 128;

__global__ __launch_bounds__(256) void paged_merge(PagedGeo g) {
    prefetch_kernarg<arg_bytes<PagedGeo>()>();
    constexpr int U = 8;  // partials in flight
    __shared__ float2 ml[kMergeRows][kMergeSlots];
    const uint32_t tid = threadIdx.x, d4 = g.head_dim / 4, S = g.slots;
    const uint32_t rows = min(256 / d4, kMergeRows);
    const uint64_t all = static_cast<uint64_t>(g.tokens) * g.heads, row0 = static_cast<uint64_t>(blockIdx.x) * rows;
    const uint32_t here = static_cast<uint32_t>(min(all - row0, static_cast<uint64_t>(rows)));
    const uint32_t x = min(tid / d4, here - 1), c = tid % d4;
    const uint64_t at = row0 + x;
    const float* const part = g.part + at * S * g.head_dim + 4 * c;
    float4 v[U];
    uint32_t last = S - 1;
    const auto load = [&](uint32_t s0) {  // (past the last they re-read it, with weight 0)
#pragma unroll
        for (int u = 0; u < U; ++u)
            v[u] = *reinterpret_cast<const float4*>(part + static_cast<uint64_t>(min(s0 + u, last)) * g.head_dim);
    };
    for (uint32_t i = tid; i < here * S; i += 256) ml[i / S][i % S] = g.ml[row0 * S + i];
    if (g.uneven == 0) load(0);
    __syncthreads();
    float mm = -INFINITY;
    uint32_t count = S;  // the row's partials
    if (g.uneven != 0) {
        for (count = 0; count < S && !(ml[x][count].y < 0.f);) ++count;
        if (count != 0) {
            last = count - 1;
            load(0);
        }
    }
    for (uint32_t s = 0; s < count; ++s) mm = fmaxf(mm, ml[x][s].x);
    __syncthreads();
    // each of a row's threads its share of the weights (a NaN maximum keeps its sum's NaN)
    if (tid / d4 < here)
        for (uint32_t s = c; s < count; s += d4) {
            const float2 p = ml[x][s];
            const float f = p.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(p.x - mm);
            ml[x][s] = make_float2(f, p.y * f);
        }
    __syncthreads();
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t s0 = 0; s0 < count; s0 += U) {
        if (s0 != 0) load(s0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u >= count) continue;
            const float2 p = ml[x][s0 + u];
            l += p.y;
            // (an empty partial's values are zeros)
            fma4(o, p.x, v[u]);
        }
    }
    if (tid / d4 < here && count != 0)
        store4(g.out + at * g.head_dim + 4 * c, scaled4(o, 1.0f / l), g.aligned != 0);
}

}  // namespace

namespace {

PagedGeo paged_geometry(const PagedTokensArgs& a) {
    PagedGeo g{};
    g.starts = a.starts;
    g.lens = a.lens;
    g.table = a.table;
    const uint64_t page = 2ull * a.page_size * a.kv_heads * a.head_dim;
    g.pool = a.pool + static_cast<uint64_t>(a.layer) * a.num_pages * page;
    g.q = a.q;
    g.out = a.out;
    g.batch = a.batch;
    g.tokens = a.tokens;
    g.heads = a.heads;
    g.kv_heads = a.kv_heads;
    g.group = a.heads / a.kv_heads;
    g.head_dim = a.head_dim;
    g.page16 = a.page_size / 16;
    g.page_shift = (g.page16 & (g.page16 - 1)) == 0 ? static_cast<uint32_t>(__builtin_ctz(g.page16)) : 32;
    g.pages_per_seq = a.pages_per_seq;
    g.num_pages = a.num_pages;
    g.window = a.window == 0 ? 0xffffffffu : a.window;
    g.sinks = a.window == 0 ? 0 : a.sinks;
    g.splits = g.slots = g.tail_splits = 1;
    g.aligned = aligned16(a.q) && aligned16(a.out);
    g.rows_upto = 0xffffffffu;
    g.scale = a.scale;
    return g;
}

constexpr uint32_t kBlockRows = 16;  // query rows of a paged_rows block

// Items with `per` query rows each: of all tokens together, and row by row.
uint32_t items_together(const PagedGeo& g, uint64_t per) {
    return static_cast<uint32_t>((static_cast<uint64_t>(g.tokens) * g.group + per - 1) / per);
}
uint32_t items_by_row(const PagedGeo& g, uint64_t per) {
    return static_cast<uint32_t>(static_cast<uint64_t>(g.tokens) * g.group / per + g.batch);
}

hipError_t launch_rows(const PagedGeo& g, hipStream_t s) {
    const unsigned grid = paged_blocks(g);
    const bool exact = g.head_dim % 64 == 0;
#define SL_ROWS(DV, NW)                                               \
    do {                                                              \
        if (exact) paged_rows<DV, true, NW><<<grid, 64 * NW, 0, s>>>(g); \
        else paged_rows<DV, false, NW><<<grid, 64 * NW, 0, s>>>(g);      \
    } while (0)
    switch ((g.head_dim + 63) / 64) {
        case 1: SL_ROWS(1, 8); break;
        case 2: SL_ROWS(2, 8); break;
        case 3: SL_ROWS(3, 4); break;
        default: SL_ROWS(4, 4); break;
    }
#undef SL_ROWS
    return hipGetLastError();
}

hipError_t launch_merge(const PagedGeo& g, hipStream_t s) {
    const uint64_t rows = std::min<uint64_t>(1024 / g.head_dim, kMergeRows);
    const uint64_t blocks = (static_cast<uint64_t>(g.tokens) * g.heads + rows - 1) / rows;
    paged_merge<<<static_cast<unsigned>(blocks), 256, 0, s>>>(g);
    return hipGetLastError();
}

// Partials of `slots` key ranges per query row, at the workspace's start.
bool place_partials(PagedGeo* g, uint32_t slots, const Workspace& ws) {
    const uint64_t rows = static_cast<uint64_t>(g->tokens) * g->heads * slots;
    const uint64_t ml = (2 * rows + 63) / 64 * 64;
    if (ml + rows * g->head_dim > ws.floats) return false;
    g->slots = slots;
    g->ml = reinterpret_cast<float2*>(ws.data);
    g->part = ws.data + ml;
    return true;
}

// Key splits for `blocks` blocks of equal work, one per CU at a time, whose keys take `steps`
// steps (256 keys of paged_rows, 64 of paged_tiles), and the time they take: a round of blocks
// costs its steps and `fixed` more, partials a step, and `partial` for each block's. (1 for a
// batch that fills the chip by itself; 2 for blocks that would leave a second round half empty.)
// Of the launch's blocks, `launched` per split with those that find nothing to do, there may be
// 2^23.
struct SplitCosts {
    double step_us, fixed, partial;
};
struct Splits {
    uint32_t n;
    double us;
};
Splits splits_for(uint64_t blocks, uint64_t launched, uint64_t steps, const SplitCosts& cost) {
    const uint64_t cus = compute_units();
    Splits best{1, 0.0};
    for (uint32_t n = 1; n <= kMergeSlots / 2 && n <= std::max<uint64_t>(steps, 1) && n * launched < 1u << 23; ++n) {
        const double rounds = static_cast<double>((blocks * n + cus - 1) / cus);
        const double us = cost.step_us * (rounds * (static_cast<double>(steps) / n + cost.fixed) +
                                          (n > 1 ? 1.0 + static_cast<double>(blocks * n) * cost.partial : 0.0));
        if (n == 1 || us < best.us) best = {n, us};
    }
    return best;
}

// Measured at head_dim 128 (at 64 both steps take two thirds; what counts is their relation). Rows
// that read much from HBM take at least that long. What the choice between the two goes by, all
// rows to paged_rows (all to paged_tiles), 8B shape:
//   1 row of 32, 128, 256, 360 new tokens at 0: 7.8, 9.8, 21.0, 33.0 us (15.5, 26.8, 34.7, 37.9),
//   of 32, 64 at 2,000: 21.8, 32.2 (31.5, 38.0), of 8, 32 at 16,000: 40.5, 101 (52.4, 60.6);
//   8 rows of 4, 8, 16 at 2,000: 31.9, 39.6, 55.5 (48.7, 50.5, 53.0); 4 rows of 8 at 16,000: 120
//   (146), of 180 at 0: 51.0 (31.8); 16 rows of 40 at 0: 35.9 (20.8).
// (It takes the other one for 360 at 0, 64 at 2,000 and 16 rows of 20 at 100, 26.2 us and not 20.2.)
constexpr SplitCosts kRowsCosts{6.0, 0.5, 0.002}, kTilesCosts{4.5, 4.0, 0.006};
double read_us(const PagedGeo& g, uint64_t keys) {
    return static_cast<double>(keys) * g.kv_heads * g.head_dim * 8 / 4.9e6 * (g.head_dim > 64 ? 1.0 : 1.5);
}

// Splits of paged_rows for `query_rows` in blocks that see up to `keys` keys.
Splits rows_splits(const PagedGeo& g, uint64_t query_rows, uint64_t launched, uint64_t keys) {
    return splits_for((query_rows + kBlockRows - 1) / kBlockRows * g.kv_heads, launched * g.kv_heads, (keys + 255) / 256,
                      kRowsCosts);
}
Splits tiles_splits(const PagedGeo& g, uint64_t blocks, uint64_t launched, uint64_t keys) {
    return splits_for(blocks * g.kv_heads, launched * g.kv_heads, (keys + 63) / 64, kTilesCosts);
}

}  // namespace

hipError_t launch_paged_window(const PagedTokensArgs& a, const Workspace& ws, hipStream_t s) {
    if (a.tokens == 0) return hipSuccess;
    PagedGeo g = paged_geometry(a);
    // All of the call's rows to paged_rows, or those with up to kPagedFewRows query rows, the
    // others to paged_tiles: which launches there are, and their splits, follow the row starts of
    // this call; each launch takes the rows that are its own when it runs.
    PagedGeo r = g, t = g;
    // (a block's queries see their windows and the positions between them)
    const auto seen = [&](uint64_t keys, uint32_t rows) {
        return std::min<uint64_t>(keys, uint64_t{g.window} + rows / g.group + g.sinks);
    };
    r.own_items = items_by_row(g, kBlockRows);
    t.own_items = items_by_row(g, kTileRows);
    const uint32_t most_few = std::min(g.batch * (kPagedFewRows / kBlockRows), r.own_items);
    bool some = true, tiles = false;
    Splits rs = rows_splits(g, static_cast<uint64_t>(a.few_rows) + a.many_rows, r.own_items,
                            std::max<uint64_t>(a.few_keys, seen(a.many_keys, kBlockRows)));
    Splits ts{1, 0.0};
    if (a.many_rows != 0 && g.head_dim <= 128) {
        Splits few{1, 0.0};
        if (a.few_rows != 0) {
            few = rows_splits(g, a.few_rows, most_few, a.few_keys);
            few.us = std::max(few.us, read_us(g, a.few_keys_in_all));
        }
        const uint64_t keys = seen(a.many_keys, kTileRows);
        ts = tiles_splits(g, a.many_blocks, t.own_items, keys);
        // Not split, but the last round of blocks less than half full: those blocks alone. (376 blocks
        // of a prompt of 3,001 of the 1B shape: 134 -> 119 us.)
        const uint32_t round = static_cast<uint32_t>(compute_units()) / g.kv_heads;
        const uint32_t rest = round != 0 ? a.many_blocks % round : 0;
        if (ts.n == 1 && a.many_blocks > round && rest != 0 && 2 * rest <= round) {
            const Splits last = tiles_splits(g, rest, rest, keys);
            const double us = kTilesCosts.step_us * (a.many_blocks / round) *
                                  (static_cast<double>((keys + 63) / 64) + kTilesCosts.fixed) + last.us;
            if (last.n > 1 && us < ts.us) {
                t.round_items = round;
                t.tail_splits = last.n;
                ts.us = us;
            }
        }
        if (few.us + ts.us < std::max(rs.us, read_us(g, a.few_keys_in_all + a.many_keys_in_all))) {
            rs = few;
            tiles = true;
            some = a.few_rows != 0;
        } else {
            ts.n = t.tail_splits = 1;
        }
        if (tiles && some) {
            r.rows_upto = t.rows_over = kPagedFewRows;
            r.own_items = most_few;
        }
    }
    // (as many splits as the workspace has room for)
    const uint64_t room = ws.floats / (static_cast<uint64_t>(g.tokens) * g.heads * (g.head_dim + 2) + 64);
    const auto fit = [&](uint32_t n) { return static_cast<uint32_t>(std::min<uint64_t>(n, std::max<uint64_t>(room, 1))); };
    const uint32_t slots = fit(std::max({rs.n, ts.n, t.tail_splits}));
    t.tail_splits = fit(t.tail_splits);
    if (slots > 1 && place_partials(&g, slots, ws)) {
        r.splits = fit(rs.n);
        t.splits = fit(ts.n);
        g.uneven = t.tail_splits > 1 || (some && tiles && r.splits != t.splits);
        if (t.tail_splits > 1) t.own_items += t.round_items * (t.tail_splits - 1);
        r.slots = t.slots = slots;
        r.ml = t.ml = g.ml;
        r.part = t.part = g.part;
    } else {
        t.tail_splits = 1;
    }
    hipError_t e = hipSuccess;
    if (some) e = launch_rows(r, s);
    if (e == hipSuccess && tiles) e = launch_paged_tiles(t, s);
    if (e == hipSuccess && g.slots > 1) e = launch_merge(g, s);
    return e;
}

// Bytes of K and V that sharing has to save: 4 rows of the 8B shape over 500, 1,000, 2,000
// positions (12, 24, 48 MiB) take 14.2, 15.0, 16.4 us by themselves, 19.8, 15.3, 16.0 shared;
// 16 over 208 (25 MiB) 12.0 and 14.5; 16 over 2,000 33.0 and 23.0.
constexpr uint64_t kSharingPays = 32ull << 20;

hipError_t launch_paged_prefix(const PagedTokensArgs& a, uint32_t prefix, const Workspace& ws, hipStream_t s) {
    if (a.tokens == 0) return hipSuccess;
    PagedGeo g = paged_geometry(a);
    const uint64_t rows = static_cast<uint64_t>(g.tokens) * g.group;
    // Sharing costs partials of every query row: it does not pay where the rows read little more
    // on their own (what they share then comes from the caches).
    const uint64_t saved = static_cast<uint64_t>(prefix) * (a.rows_with_tokens - 1) * g.kv_heads * g.head_dim * 8;
    if (saved < kSharingPays) return launch_paged_window(a, ws, s);
    const uint32_t by_rows = items_together(g, kBlockRows), by_tiles = items_together(g, kTileRows);
    const Splits rs = rows_splits(g, rows, 2ull * by_rows, prefix), ts = tiles_splits(g, by_tiles, 2ull * by_tiles, prefix);
    const bool tiles = g.head_dim <= 128 && ts.us < rs.us;
    g.shared_splits = tiles ? ts.n : rs.n;
    g.own_items = items_by_row(g, kBlockRows);
    g.splits = rows_splits(g, static_cast<uint64_t>(a.few_rows) + a.many_rows, 2ull * g.own_items,
                           std::max(a.few_keys, a.many_keys) - prefix).n;
    if (!place_partials(&g, g.shared_splits + g.splits, ws)) return launch_paged_window(a, ws, s);
    g.prefix = prefix;
    hipError_t e = hipSuccess;
    if (tiles) {
        PagedGeo x = g;
        x.shared_items = by_tiles;
        x.own_items = 0;
        e = launch_paged_tiles(x, s);
    } else {
        g.shared_items = by_rows;  // both kinds beside one another
    }
    if (e == hipSuccess) e = launch_rows(g, s);
    if (e == hipSuccess) e = launch_merge(g, s);
    return e;
}

hipError_t load_code_paged_attention() {
    hipFuncAttributes attr;
    return hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&paged_merge));
}

}  // namespace slhip
