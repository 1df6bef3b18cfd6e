// Attention of ragged new tokens over a paged cache (reference/attention.rs:
// 129-219 for the mathematics; the pages, window, sinks and shared prefix have
// no reference counterpart).
//
// A query at position p sees the keys j <= p that lie in its window (j > p - W)
// or among the sinks (j < S); o = sum_j softmax_j(scale q.k_j) v_j, in one pass over
// the keys with a running maximum.
//
// paged_rows serves up to 16 query rows (token, query head of one KV head) per
// block: its four waves take 32-key tiles of their own, K and V going from the
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
// element takes to arrive.
//
// A tile whose values are not finite, or a result that is not a number, sends
// the wave back over its tiles in plain f32 (slow_tile), where a key that a query
// does not see contributes nothing whatever it holds.
#include "paged_geo.h"

namespace slhip {
namespace {

constexpr int kWeightTop = 14;  // weights reach fp16 as up to 2^14

// One wave's tiles in plain f32: lane l works on query l % 16, in `o` (that
// query's row in LDS) on the dims 4 i + l / 16, which no other lane touches.
// m in units of q.k (with the factor's sign), as in the fast form.
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
            p[i] = g.scale < 0.f ? -dot : dot;
            tmax = fmaxf(tmax, p[i]);
        }
        tmax = fmaxf(tmax, lane_xor16(tmax));
        tmax = fmaxf(tmax, lane_xor32(tmax));
        const float before = m;
        m = fmaxf(before, tmax);
        const float corr = before == -INFINITY ? 0.f : exp2f((before - m) * c2);
        l *= corr;
        if (corr != 1.f)
            for (uint32_t d = kk; d < g.head_dim; d += 4) o[d] *= corr;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t x = 2 * tile + i / 4;
            const bool seen = x < keys.groups && paged_sees(mask, g.sinks, keys.group(x) * 16 + 4 * kk + i % 4);
            p[i] = seen ? exp2f((p[i] - m) * c2) : 0.f;
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

// EXACT: head_dim is 64 DV; else it is smaller, a multiple of 16, and the dims past
// it are zeros.
template <int DV, bool EXACT>
__global__ __launch_bounds__(256, DV <= 2 ? 2 : 1) void paged_rows(PagedGeo g) {
    prefetch_kernarg<arg_bytes<PagedGeo>()>();
    constexpr int KS = 2 * DV;  // 32-dim steps of a score
    constexpr int DT = 4 * DV;  // 16-dim tiles of the result
    __shared__ __align__(16) float so[4][16][64 * DV + 4];
    __shared__ float sml[4][16][2];
    PagedItem it;
    if (!paged_item(g, blockIdx.x / g.kv_heads, 16, &it)) return;  // block-uniform
    const int tid = threadIdx.x, lane = tid % kWave, c = lane % 16, kk = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t kvh = blockIdx.x % g.kv_heads, D = g.head_dim, G = g.group;
    const uint32_t count = min(16u, it.n * G - it.r0);
    const PagedKeys keys = paged_keys(g, it, it.r0, count);
    const uint32_t tiles = (keys.groups + 1) / 2;
    const uint32_t r = it.r0 + min(static_cast<uint32_t>(c), count - 1);
    const uint32_t position = it.len + r / G;
    const float* const qrow = g.q + (static_cast<uint64_t>(it.t0 + r / G) * g.heads + kvh * G + r % G) * D;
    const PagedMask mask = paged_mask(g, position);
    const uint64_t row = static_cast<uint64_t>(g.kv_heads) * D, voff = paged_v_offset(g);
    const bool aligned = g.aligned != 0;

    float4 kx[2][KS][2], vx[8][DV];
    // Keys past the last one re-read it (their scores are masked); a missing second
    // group re-reads the first.
    const auto load_k = [&](uint32_t tile) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t grp = keys.group(min(2 * tile + s, keys.groups - 1));
            const float* const at = paged_group(g, it.b, grp, kvh) + min(static_cast<uint32_t>(c), keys.end - 1 - 16 * grp) * row;
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    kx[s][j][h] = EXACT || 32 * j + 16 * h < D
                                      ? *reinterpret_cast<const float4*>(at + 32 * j + 16 * h + 4 * kk)
                                      : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    const auto load_v = [&](uint32_t tile) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t grp = keys.group(min(2 * tile + s, keys.groups - 1));
            const float* const base = paged_group(g, it.b, grp, kvh) + voff;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float* const at = base + min(static_cast<uint32_t>(4 * kk + i), keys.end - 1 - 16 * grp) * row;
#pragma unroll
                for (int J = 0; J < DV; ++J)
                    vx[4 * s + i][J] = EXACT || 64 * J + 4 * c < D
                                           ? *reinterpret_cast<const float4*>(at + 64 * J + 4 * c)
                                           : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
    };
    // When a tile's rows are asked for: at head_dim 64 a tile ahead; at 128 its K and
    // V together (registers for a tile ahead would be spilled); above, V after the
    // scores.
    constexpr bool kAhead = DV == 1, kTogether = DV <= 2;
    const uint32_t tile0 = blockIdx.y * 4 + wave, step = 4 * gridDim.y;
    if (kAhead && tile0 < tiles) {
        load_k(tile0);
        load_v(tile0);
    }
    v8h qh[KS], ql[KS];
    int qe;
    bool bad;
    {
        float4 qx[KS][2];
        float most = 0.f;
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < KS; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                qx[j][h] = EXACT || 32 * j + 16 * h < D ? load4(qrow + 32 * j + 16 * h + 4 * kk, aligned)
                                                        : make_float4(0.f, 0.f, 0.f, 0.f);
                most = max_abs(most, qx[j][h]);
                // (a NaN is not seen by max_abs)
                const float4 v = qx[j][h];
                bits |= (v.x != v.x) | (v.y != v.y) | (v.z != v.z) | (v.w != v.w);
            }
        most = fmaxf(most, lane_xor16(most));
        most = fmaxf(most, lane_xor32(most));
        bad = bits != 0 || most == INFINITY;
        qe = part_exponent(most);
        // a negative factor goes into the queries, so that the largest score is the largest sum
        const float scale = g.scale < 0.f ? -power2(qe) : power2(qe);
#pragma unroll
        for (int j = 0; j < KS; ++j) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                put_parts(qx[j][h].x, qx[j][h].y, scale, qh[j], ql[j], 4 * h);
                put_parts(qx[j][h].z, qx[j][h].w, scale, qh[j], ql[j], 4 * h + 2);
            }
        }
    }
    const float c2 = fabsf(g.scale) * 1.4426950408889634f;
    // The state: query c's largest score (in units of q.k), this lane's keys' part of
    // the sum, and O^T in units of 2^-oexp: o[4 J + e][i] is dim 64 J + 16 kk + 4 i + e.
    float m = -INFINITY, l = 0.f;
    v4f o[DT];
    int oexp = 0;
    bool first = true;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = v4f{0.f, 0.f, 0.f, 0.f};
#define SL_F16(a, b, x) __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, x, 0, 0, 0)
    for (uint32_t tile = tile0; tile < tiles; tile += step) {
        if (!kAhead) {
            load_k(tile);
            if (kTogether) load_v(tile);
        }
        // scores
        float most = 0.f;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < KS; ++j) most = max_abs(max_abs(most, kx[s][j][0]), kx[s][j][1]);
        most = wave_max(most);
        bad |= most == INFINITY;
        const int ke = part_exponent(most);
        const float kscale = power2(ke);
        v4f sc[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            v8h kh[KS], kl[KS];
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    put_parts(kx[s][j][h].x, kx[s][j][h].y, kscale, kh[j], kl[j], 4 * h);
                    put_parts(kx[s][j][h].z, kx[s][j][h].w, kscale, kh[j], kl[j], 4 * h + 2);
                }
            // the small products first, so that a large sum rounds once per step
            v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                x = SL_F16(kl[j], qh[j], x);
                x = SL_F16(kh[j], ql[j], x);
            }
#pragma unroll
            for (int j = 0; j < KS; ++j) x = SL_F16(kh[j], qh[j], x);
            sc[s] = x;
        }
        const bool more = tile + step < tiles;  // wave-uniform
        if (kAhead && more) load_k(tile + step);
        if (!kTogether) load_v(tile);
        float p[8];
        float tmax = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t x = 2 * tile + i / 4;
            const uint32_t j = keys.group(min(x, keys.groups - 1)) * 16 + 4 * kk + i % 4;
            p[i] = x < keys.groups && paged_sees(mask, g.sinks, j) ? sc[i / 4][i % 4] : -INFINITY;
            tmax = fmaxf(tmax, p[i]);
        }
        tmax = fmaxf(tmax, lane_xor16(tmax));
        tmax = fmaxf(tmax, lane_xor32(tmax));
        // The weights' exponents are (x - m) c2, x and m in the tile's units (an exact
        // power of two apart from q.k's): exactly 0 for the largest, however large.
        // A query may see none of the keys so far (m = -inf): weights and corr are 0.
        const float unit = power2(-qe - ke);
        const float m_new = fmaxf(m, tmax * unit);
        const float mt = m_new * power2(qe + ke), ct = c2 * unit;
        const float corr = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m_new) * c2);
        m = m_new;
        // values
        most = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int J = 0; J < DV; ++J) most = max_abs(most, vx[i][J]);
        most = wave_max(most);
        bad |= most == INFINITY;
        const int need = part_exponent(most);
        const int ve = first ? need : min(need, oexp - kWeightTop);
        // O's unit: the weights' 2^14 times the values' scale, lowered when larger values come
        const float turn = first ? 0.f : corr * power2(ve + kWeightTop - oexp);
        first = false;
        oexp = ve + kWeightTop;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] *= turn;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float w = p[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((p[i] - mt) * ct);
            sum += w;
            p[i] = w;
        }
        l = l * corr + sum;
        v8h ph, pl;
#pragma unroll
        for (int i = 0; i < 8; i += 2) put_parts(p[i], p[i + 1], power2(kWeightTop), ph, pl, i);
        const float vscale = power2(ve);
#pragma unroll
        for (int J = 0; J < DV; ++J)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v8h vh, vl;
#pragma unroll
                for (int i = 0; i < 8; i += 2)
                    put_parts(reinterpret_cast<const float*>(&vx[i][J])[e],
                              reinterpret_cast<const float*>(&vx[i + 1][J])[e], vscale, vh, vl, i);
                v4f x = o[4 * J + e];
                x = SL_F16(vl, ph, x);
                x = SL_F16(vh, pl, x);
                o[4 * J + e] = SL_F16(vh, ph, x);
            }
        if (kAhead && more) load_v(tile + step);
    }
#undef SL_F16
    const float back = power2(-oexp);
    float check = l;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
        o[t] *= back;
        check += (o[t][0] + o[t][1]) + (o[t][2] + o[t][3]);
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
    for (uint32_t i = tid; i < count * d4; i += 256) {
        const uint32_t x = i / d4, d = 4 * (i % d4);
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sml[w][x][0]);
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float mw = sml[w][x][0];
            // (an empty state weighs nothing; a NaN maximum keeps its sum's NaN)
            const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw - mm) * c2);
            sum = fmaf(sml[w][x][1], f, sum);
            if (f != 0.f) fma4(acc, f, *reinterpret_cast<const float4*>(&so[w][x][d]));
        }
        const uint32_t rr = it.r0 + x;
        const uint64_t at = static_cast<uint64_t>(it.t0 + rr / G) * g.heads + kvh * G + rr % G;
        if (g.slots == 1) {
            store4(g.out + at * D + d, scaled4(acc, 1.0f / sum), aligned);
        } else {
            const uint64_t slot = at * g.slots + g.slot0 + blockIdx.y;
            *reinterpret_cast<float4*>(g.part + slot * D + d) = acc;
            if (d == 0) g.ml[slot] = make_float2(mm, sum);
        }
    }
}

// Combines the partials of each query row: thread per float4 of the result.
__global__ __launch_bounds__(256) void paged_merge(PagedGeo g) {
    prefetch_kernarg<arg_bytes<PagedGeo>()>();
    const uint32_t d4 = g.head_dim / 4;
    const uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= static_cast<uint64_t>(g.tokens) * g.heads * d4) return;
    const uint64_t at = i / d4;
    const uint32_t d = 4 * static_cast<uint32_t>(i % d4);
    const float c2 = fabsf(g.scale) * 1.4426950408889634f;
    const float2* const ml = g.ml + at * g.slots;
    const float* const part = g.part + at * g.slots * g.head_dim + d;
    float mm = -INFINITY;
    for (uint32_t s = 0; s < g.slots; ++s) mm = fmaxf(mm, ml[s].x);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t s = 0; s < g.slots; ++s) {
        const float2 x = ml[s];
        const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x.x - mm) * c2);
        l = fmaf(x.y, f, l);
        if (f == 0.f) continue;
        fma4(o, f, *reinterpret_cast<const float4*>(part + static_cast<uint64_t>(s) * g.head_dim));
    }
    store4(g.out + at * g.head_dim + d, scaled4(o, 1.0f / l), g.aligned != 0);
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
    g.pages_per_seq = a.pages_per_seq;
    g.num_pages = a.num_pages;
    g.window = a.window == 0 ? 0xffffffffu : a.window;
    g.sinks = a.window == 0 ? 0 : a.sinks;
    g.kbegin = 0;
    g.kend = 0xffffffffu;
    g.splits = g.slots = 1;
    g.aligned = aligned16(a.q) && aligned16(a.out);
    g.rows_upto = 0xffffffffu;
    g.scale = a.scale;
    return g;
}

// One launch over the geometry's keys, `splits` blocks per item.
hipError_t launch_rows(const PagedGeo& g, hipStream_t s) {
    const uint64_t rows = static_cast<uint64_t>(g.tokens) * g.group;
    const uint64_t items = g.shared ? (rows + 15) / 16 : rows / 16 + g.batch;
    const dim3 grid(static_cast<unsigned>(items * g.kv_heads), g.splits);
    const uint32_t dv = (g.head_dim + 63) / 64;
    const bool exact = g.head_dim % 64 == 0;
#define SL_ROWS(DV)                                           \
    if (exact) paged_rows<DV, true><<<grid, 256, 0, s>>>(g);  \
    else paged_rows<DV, false><<<grid, 256, 0, s>>>(g)
    switch (dv) {
        case 1: SL_ROWS(1); break;
        case 2: SL_ROWS(2); break;
        case 3: SL_ROWS(3); break;
        default: SL_ROWS(4); break;
    }
#undef SL_ROWS
    return hipGetLastError();
}

hipError_t launch_merge(const PagedGeo& g, hipStream_t s) {
    const uint64_t n = static_cast<uint64_t>(g.tokens) * g.heads * (g.head_dim / 4);
    paged_merge<<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(g);
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

// Key splits for `items` blocks per KV head that read up to `keys` keys each: until
// about two blocks per CU run, each wave having a tile of 32 keys.
uint32_t splits_for(uint64_t items, uint64_t kv_heads, uint64_t keys) {
    const uint64_t blocks = items * kv_heads, most = (keys + 127) / 128;
    uint64_t n = blocks ? (2 * compute_units() + blocks - 1) / blocks : 1;
    n = n < most ? n : most;
    return static_cast<uint32_t>(n < 1 ? 1 : n > 64 ? 64 : n);
}

}  // namespace

hipError_t launch_paged_window(const PagedTokensArgs& a, const Workspace& ws, hipStream_t s) {
    if (a.tokens == 0) return hipSuccess;
    PagedGeo g = paged_geometry(a);
    const uint64_t rows = static_cast<uint64_t>(g.tokens) * g.group;
    const uint32_t splits = splits_for(rows / 16 + g.batch, g.kv_heads, a.most_keys);
    if (splits > 1 && place_partials(&g, splits, ws)) g.splits = splits;
    hipError_t e = launch_rows(g, s);
    if (e == hipSuccess && g.slots > 1) e = launch_merge(g, s);
    return e;
}

hipError_t launch_paged_prefix(const PagedTokensArgs& a, uint32_t prefix, const Workspace& ws, hipStream_t s) {
    if (a.tokens == 0) return hipSuccess;
    PagedGeo g = paged_geometry(a);
    const uint64_t rows = static_cast<uint64_t>(g.tokens) * g.group;
    const uint32_t first = splits_for((rows + 15) / 16, g.kv_heads, prefix);
    const uint32_t second = splits_for(rows / 16 + g.batch, g.kv_heads, a.most_keys - prefix);
    if (prefix == 0 || !place_partials(&g, first + second, ws)) return launch_paged_window(a, ws, s);
    PagedGeo own = g;
    g.shared = 1;
    g.kend = prefix;
    g.splits = first;
    own.kbegin = prefix;
    own.splits = second;
    own.slot0 = first;
    hipError_t e = launch_rows(g, s);
    if (e == hipSuccess) e = launch_rows(own, s);
    if (e == hipSuccess) e = launch_merge(g, s);
    return e;
}

hipError_t load_code_paged_attention() {
    hipFuncAttributes attr;
    return hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&paged_merge));
}

}  // namespace slhip
