// Attention of many query rows over a paged cache: prompt chunks, and the shared
// prefix of a large batch (paged_attention.hip has the definition and the form for
// few query rows; paged_geo.h the geometry and the fp16 parts).
//
// A block of 8 waves owns 256 query rows (token, query head of one KV head), 32 per
// wave, and streams the keys they see in stages of 64. Every wave loads one group of
// 16 positions of a stage, half of the waves its keys, half its values, while the
// stage before is computed; it splits them into fp16 parts once for the block, under
// a scale of that group's own, and writes them to the other half of LDS: one
// barrier per stage.
//   K parts lie row by row (a row and 16 bytes apart, so that 16 rows' pieces meet 64
//     different banks) and are read as A of v_mfma_f32_32x32x16_f16: lane l holds key
//     l % 32 and dims 16 j + 8 (l / 32) ..; B is the queries, in registers.
//   S^T leaves lane l with query l % 32 and the keys 8 (i / 4) + 4 (l / 32) + i % 4, i < 16,
//     which in that order is B of the second product.
//   V parts lie in A's order for it: a lane that loads the 4 (head_dim 64: 2) dims at
//     4 (l % 32) of the keys 8 (i / 4) + 4 (l / 32) + i % 4, i < 8, of a group holds, for
//     each e, row l % 32 of the dim tile e whose row r is dim 4 r + e.
// The softmax state is per lane, the sum of a query's weights added up over its two
// lanes at the end. O^T is kept in units of 2^-oexp, which follows the groups' values,
// so that the weights' fp16 parts keep their bits whatever a query's other keys hold.
//
// Bound by the matrix cores and by the vector work between their products (splitting,
// and about 12 instructions per weight), which overlap only in part: a stage takes about
// 11,000 cycles where its products take 6,100. 2,048 tokens at 6,000 of the 8B shape behind
// a window of 4,096: 410 us, 1.0 PFLOP/s of fp16 products, three of them per product
// (hipBLASLt's 8192^3 reaches 1.08). The scores of a whole stage before its softmax, not of
// 32 keys at a time: 128 us, not 132, for a prompt of 3,001 of the 1B shape; 134 with the
// looks at how far the rows and groups lie apart; 119 with its last round's blocks split.
// No better: two tiles of 32 queries per wave, blocks of 4 waves, stages of 32 keys, raised wave
// priorities; four waves per SIMD at head_dim 64 spill and take 160 us for that prompt.
#include "paged_geo.h"

namespace slhip {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int NW = 8;  // waves per block

// Weights are up to 2^kSlack, 2^(kSlack + kTileTop) as fp16 parts.
constexpr float kSlack = 8.f;
constexpr int kTileTop = 7;
constexpr int kNoUnit = 1000;  // of a group whose values are all zero

template <int DV>
struct TileShape {
    static constexpr int SG = 4;                    // 16-position groups per stage
    static constexpr int KROW = 64 * DV * 2 + 16;   // bytes between K rows of one part
    static constexpr int KPART = 16 * SG * KROW;    // bytes of one part of a stage's K
    static constexpr int VGROUP = 2 * DV * 2 * 1024;  // bytes of a group's V: dim tiles x parts x 1 KB
    static constexpr int STAGE = 2 * KPART + SG * VGROUP;
};

template <int DV, bool EXACT>
__global__ __launch_bounds__(64 * NW, 2) void paged_tiles(PagedGeo g) {
    prefetch_kernarg<arg_bytes<PagedGeo>()>();
    using Shape = TileShape<DV>;
    constexpr int SG = Shape::SG, KS = 4 * DV, DT = 2 * DV, VW = 2 * DV;  // VW: dims of V per lane
    constexpr int KV4 = 4 * DV;                                          // float4 of K per lane and group
    __shared__ __align__(16) uint8_t lds[2 * Shape::STAGE];
    __shared__ int exps[2][2][SG];  // [stage half][K, V][group]
    __shared__ int flags;
    PagedItem it;
    // (the last query rows, which see the most keys, first)
    if (!paged_item<true>(g, blockIdx.x / g.kv_heads, kTileRows, &it)) return;  // block-uniform
    const int tid = threadIdx.x, lane = tid % kWave, c = lane % 32, hh = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t kvh = blockIdx.x % g.kv_heads, D = g.head_dim, G = g.group;
    const uint32_t rows = it.n * G, count = min(32u * NW, rows - it.r0);
    const PagedKeys keys = paged_keys(g, it, it.r0, count);
    // this split's stages
    const uint32_t all = (keys.groups + SG - 1) / SG, per = (all + it.splits - 1) / it.splits;
    const uint32_t stage0 = min(it.split * per, all), stages = min(stage0 + per, all);
    // the wave's queries (those past the last repeat it, unstored)
    const uint32_t w0 = it.r0 + min(32u * wave, count - 1), w1 = it.r0 + min(32u * wave + 31, count - 1);
    const bool idle = 32u * wave >= count;  // wave-uniform: only loads
    const uint32_t r = it.r0 + min(32u * wave + c, count - 1);
    const PagedMask mask = paged_mask(g, it, it.len + r / G);
    const PagedMask mask0 = paged_mask(g, it, it.len + w0 / G), mask1 = paged_mask(g, it, it.len + w1 / G);
    // Places in the block's list of groups: those that one of the wave's queries sees a key
    // of (sinks aside), and those that all of them see whole.
    const auto listed = [&](uint32_t grp) { return keys.sink_groups + (max(grp, keys.first_group) - keys.first_group); };
    const uint32_t seen0 = listed(mask0.low / 16), seen1 = listed((mask1.end + 15) / 16);
    const uint32_t whole0 = listed((mask1.low + 15) / 16), whole1 = listed(mask0.end / 16);
    // (the list begins with the sinks' groups, wherever its window part starts)
    const uint32_t seen_sinks = (g.sinks + 15) / 16, whole_sinks = g.sinks / 16;
    const float* const qrow = g.q + (static_cast<uint64_t>(it.t0 + r / G) * g.heads + kvh * G + r % G) * D;
    const uint64_t row = static_cast<uint64_t>(g.kv_heads) * D;
    const bool aligned = g.aligned != 0;
    const uint32_t part = paged_pack(it);
    if (tid == 0) flags = 0;
    __syncthreads();

    // ---- loading: wave w < SG takes group w's K, the others group w - SG's V ----
    const bool loads_k = wave < SG;
    const int mine = loads_k ? wave : wave - SG;
    constexpr int F = 16 * DV;  // float4 per K row
    float4 x[KV4];  // K: float4 u of the lane's; V: x[i * DV / 2 ..], key i's VW dims
    const uint32_t kv_bytes = static_cast<uint32_t>(row) * 4;
    // byte offsets from a group's first row: the lane's own, the rest the same for the wave
    const uint32_t place = loads_k ? lane / F * kv_bytes + 16 * (lane % F) : 4 * hh * kv_bytes + 4 * VW * c;
    const bool in = EXACT || (loads_k ? 4 * (lane % F) : VW * c) < D;
    const auto group_of = [&](uint32_t stage) { return keys.group(min(stage * SG + mine, keys.groups - 1)); };
    // (rows past the last key are out of the buffer's range and read as zeros)
    const auto load = [&](uint32_t grp, const float* base) {
        const uint32_t rows_in = min(keys.end - 16 * grp, 16u);
        uint32_t step = kv_bytes;  // (its multiples worked out here, not held in registers from the start)
        asm volatile("" : "+s"(step));
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<float*>(loads_k ? base : base + paged_v_offset(g)), 0, (rows_in - 1) * kv_bytes + 4 * D, kBufferFlags);
        if (loads_k) {
#pragma unroll
            for (int u = 0; u < KV4; ++u)
                x[u] = in ? __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, place, (64 / F) * u * step, 0))
                          : make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t at = (8 * (i / 4) + i % 4) * step;
                if constexpr (DV == 2) {
                    x[i] = in ? __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, place, at, 0))
                              : make_float4(0.f, 0.f, 0.f, 0.f);
                } else {
                    const float2 v = in ? __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(rsrc, place, at, 0))
                                        : make_float2(0.f, 0.f);
                    if (i % 2 == 0) x[i / 2].x = v.x, x[i / 2].y = v.y;
                    else x[i / 2].z = v.x, x[i / 2].w = v.y;
                }
            }
        }
    };
    const auto stage_out = [&](int half) {
        const auto value = [&](int i, int d) -> float {  // key i's dim d, of the lane's V
            const float4 q = x[VW * i / 4];
            const int e4 = DV == 2 ? d : 2 * (i % 2) + d;
            return e4 == 0 ? q.x : e4 == 1 ? q.y : e4 == 2 ? q.z : q.w;
        };
        float most = 0.f, least = INFINITY;
        // (two keys' values in one float4)
        const auto pair = [&](int u) { return make_float2(fmaxf(fabsf(x[u].x), fabsf(x[u].y)), fmaxf(fabsf(x[u].z), fabsf(x[u].w))); };
#pragma unroll
        for (int u = 0; u < KV4; ++u) {
            const float2 p = pair(u);
            const float both = fmaxf(p.x, p.y);
            most = fmaxf(most, both);
            least = fminf(least, DV == 1 && !loads_k ? fminf(p.x, p.y) : both);
        }
        most = wave_max(most);
        uint32_t apart = 0;
        if (__builtin_expect(__any(least < most * kApart), 0)) {  // wave-uniform; seldom, but for rows of zeros
#pragma unroll
            for (int u = 0; u < KV4; ++u) {
                const float2 p = pair(u);
                if (loads_k) apart |= row_apart<F>(fmaxf(p.x, p.y), most);
                else if constexpr (DV == 2) apart |= row_apart<32>(fmaxf(p.x, p.y), most);
                else apart |= row_apart<32>(p.x, most) || row_apart<32>(p.y, most);
            }
            if (!loads_k) {
#pragma unroll
                for (int d = 0; d < VW; ++d) {
                    float column = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) column = fmaxf(column, fabsf(value(i, d)));
                    column = fmaxf(column, lane_xor32(column));
                    apart |= __any(column < most * kApart && column != 0.f);
                }
            }
        }
        const int e = part_exponent(most);
        const float scale = power2(e);
        uint8_t* const base = lds + half * Shape::STAGE;
        if (loads_k) {
#pragma unroll
            for (int u = 0; u < KV4; u += 2) {
                const Parts p = to_parts(x[u], x[u + 1], scale);
                const uint4 h = __builtin_bit_cast(uint4, p.h), l = __builtin_bit_cast(uint4, p.l);
                uint8_t* const to = base + (16 * mine + lane / F + (64 / F) * u) * Shape::KROW + 8 * (lane % F);
                *reinterpret_cast<uint2*>(to) = make_uint2(h.x, h.y);
                *reinterpret_cast<uint2*>(to + Shape::KPART) = make_uint2(l.x, l.y);
                *reinterpret_cast<uint2*>(to + 64 / F * Shape::KROW) = make_uint2(h.z, h.w);
                *reinterpret_cast<uint2*>(to + 64 / F * Shape::KROW + Shape::KPART) = make_uint2(l.z, l.w);
            }
        } else {
            uint8_t* const to = base + 2 * Shape::KPART + mine * Shape::VGROUP + 16 * lane;
#pragma unroll
            for (int d = 0; d < VW; ++d) {
                const Parts p = to_parts(value(0, d), value(1, d), value(2, d), value(3, d), value(4, d), value(5, d),
                                         value(6, d), value(7, d), scale);
                *reinterpret_cast<v8h*>(to + (2 * d) * 1024) = p.h;
                *reinterpret_cast<v8h*>(to + (2 * d + 1) * 1024) = p.l;
            }
        }
        if (lane == 0) {
            exps[half][loads_k ? 0 : 1][mine] = loads_k || most != 0.f ? e : kNoUnit;
            if (apart || most == INFINITY) flags = 1;
        }
    };

    // the next stage's group and its place, looked up a stage before its rows are asked for
    uint32_t next = 0;
    const float* next_at = g.pool;
    const auto load_next = [&](uint32_t stage) {  // asks for `stage`'s rows, looks up the one after it
        load(next, next_at);
        next = group_of(stage + 1);
        next_at = paged_group(g, it.b, next, kvh);
    };
    if (stage0 < stages) {
        next = group_of(stage0);
        next_at = paged_group(g, it.b, next, kvh);
        load_next(stage0);
    }
    v8h qh[KS], ql[KS];
    int qe;
    bool bad;
    {
        float4 q[2 * KS];
        load_row<2 * KS, EXACT>(qrow, aligned, D, q, [&](int j) { return 16u * (j / 2) + 8 * hh + 4 * (j % 2); });
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < 2 * KS; ++j) most = max_abs(most, q[j]);
        most = fmaxf(most, lane_xor32(most));
        // (worked out here: put off to the end, where it is used, it would keep the rows
        // in registers through the loop)
        uint32_t flag = any_nan(q) || most == INFINITY;
        asm volatile("" : "+v"(flag));
        bad = flag != 0;
        qe = part_exponent(most);
        // a negative factor goes into the queries, so that the largest score is the largest sum
        const float scale = g.scale < 0.f ? -power2(qe) : power2(qe);
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            const Parts p = to_parts(q[2 * j], q[2 * j + 1], scale);
            qh[j] = p.h;
            ql[j] = p.l;
        }
    }
    const float c2 = fabsf(g.scale) * 1.4426950408889634f;
    float m = -INFINITY, l = 0.f;
    v16f o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
    int oexp = kNoUnit;  // (none yet)
    if (stage0 < stages) {
        stage_out(0);
        if (!loads_k && stage0 + 1 < stages) load_next(stage0 + 1);
    }
    __syncthreads();
#define SL_F16(a, b, x) __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, x, 0, 0, 0)
    for (uint32_t stage = stage0; stage < stages; ++stage) {
        const int half = (stage - stage0) & 1;
        const bool more = stage + 1 < stages;
        // The waves w and w + 4 split at the two ends of a stage. They share a SIMD, which prefers
        // the older one: its products run while the other splits, and the other's while it is at
        // its softmax or splits the next stage's keys. (All at the end: 9% slower.)
        if (loads_k) {
            if (more) load_next(stage + 1);
        } else {
            if (more) stage_out(half ^ 1);
            if (stage + 2 < stages) load_next(stage + 2);
        }
        int ke[SG], ve[SG];
#pragma unroll
        for (int v = 0; v < SG; ++v) {
            ke[v] = __builtin_amdgcn_readfirstlane(exps[half][0][v]);
            ve[v] = __builtin_amdgcn_readfirstlane(exps[half][1][v]);
        }
        const uint8_t* const base = lds + half * Shape::STAGE;
        const uint32_t gx = stage * SG;
        // wave-uniform: one of the stage's groups is visible to one of the wave's queries
        if (!idle && gx < seen1 && (gx + SG > seen0 || gx < seen_sinks)) {
            // scores: the small products first, so that a large sum rounds once per step
            v16f st[2];
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
                for (int i = 0; i < 16; ++i) st[sub][i] = 0.f;
                const uint8_t* const krow = base + (32 * sub + c) * Shape::KROW + 16 * hh;
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    const v8h kh = *reinterpret_cast<const v8h*>(krow + 32 * j);
                    const v8h kl = *reinterpret_cast<const v8h*>(krow + Shape::KPART + 32 * j);
                    st[sub] = SL_F16(kl, qh[j], st[sub]);
                    st[sub] = SL_F16(kh, ql[j], st[sub]);
                    st[sub] = SL_F16(kh, qh[j], st[sub]);
                }
            }
            if (!(gx + SG <= whole1 && (gx + SG <= whole_sinks || gx >= whole0))) {  // wave-uniform
#pragma unroll
                for (int v = 0; v < SG; ++v) {
                    const uint32_t key0 = 16 * keys.group(min(gx + v, keys.groups - 1)) + 4 * hh;
                    const bool there = gx + v < keys.groups;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (!there || !paged_sees(mask, g.sinks, key0 + 8 * (i / 4) + i % 4)) st[v / 2][8 * (v % 2) + i] = -INFINITY;
                }
            }
            // The weights are 2^(x c2 - m), x in its group's units (an exact power of two apart
            // from q.k's). m is the largest x c2, once rounded, at the time it was taken: it
            // follows only where that is kSlack beyond it, so that most tiles leave O as it is. A
            // query may see none of the keys so far (m = -inf): its weights and corr are 0.
            float f[SG], m_new = -INFINITY;
#pragma unroll
            for (int v = 0; v < SG; ++v) {
                f[v] = ldexpf(c2, -qe - ke[v]);
                const v16f& x = st[v / 2];
                const int i0 = 8 * (v % 2);
                float most = fmaxf(x[i0], x[i0 + 1]);
#pragma unroll
                for (int i = i0 + 2; i < i0 + 8; i += 2) most = fmaxf(fmaxf(most, x[i]), x[i + 1]);
                m_new = fmaxf(m_new, most * f[v]);
            }
            m_new = fmaxf(m_new, lane_xor32(m_new));
            if (__any(!(m_new - m <= kSlack))) {  // wave-uniform
                m_new = fmaxf(m, m_new);
                const float corr = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
#pragma unroll
                for (int t = 0; t < DT; ++t) o[t] *= corr;
                l *= corr;
                m = m_new;
                bad |= fabsf(m) > kExponentMost && m != -INFINITY;
            }
            const float from = m == -INFINITY ? 0.f : m;
            if (oexp >= kNoUnit) oexp = ve[0] + kTileTop;  // O is still zero
#pragma unroll
            for (int v = 0; v < SG; ++v) {
                v16f& x = st[v / 2];
                const int i = 8 * (v % 2);
#pragma unroll
                for (int e = i; e < i + 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], f[v], -from));
                    l += x[e];
                }
                const int unit = ve[v] + kTileTop;
                if (__builtin_expect(ve[v] != kNoUnit && (unit < oexp || unit > oexp + kUnitSlack), 0)) {  // wave-uniform
#pragma unroll
                    for (int t = 0; t < DT; ++t)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[t][e] = __builtin_ldexpf(o[t][e], unit - oexp);
                    oexp = unit;
                }
                const Parts w = to_parts(x[i], x[i + 1], x[i + 2], x[i + 3], x[i + 4], x[i + 5], x[i + 6], x[i + 7],
                                         power2(oexp - ve[v]));
                const uint8_t* const vat = base + 2 * Shape::KPART + v * Shape::VGROUP + 16 * lane;
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const v8h vh = *reinterpret_cast<const v8h*>(vat + (2 * t) * 1024);
                    const v8h vl = *reinterpret_cast<const v8h*>(vat + (2 * t + 1) * 1024);
                    o[t] = SL_F16(vl, w.h, o[t]);
                    o[t] = SL_F16(vh, w.l, o[t]);
                    o[t] = SL_F16(vh, w.h, o[t]);
                }
            }
        }
        if (loads_k && more) stage_out(half ^ 1);
        __syncthreads();
    }
#undef SL_F16
    // (the arguments again from here on: kept through the loop they would cost it registers)
    const PagedGeo e = geometry_again();
    paged_unpack(e, part, &it);
    const bool direct = paged_direct(e, it);
    const float back = oexp >= kNoUnit ? 0.f : power2(-oexp);
    float check = l;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
        o[t] *= back;
#pragma unroll
        for (int i = 0; i < 16; ++i) check += o[t][i];
    }
    bad |= flags != 0 || !(fabsf(check) < INFINITY);
    l += lane_xor32(l);
    // (LDS is free: the last stage ended with a barrier)
    constexpr int OROW = 64 * DV + 4;
    static_assert(2 * Shape::STAGE >= NW * 32 * OROW * 4, "room for every wave's rows");
    float* const so = reinterpret_cast<float*>(lds) + wave * 32 * OROW;
    const uint32_t mine_here = count > 32u * wave ? min(count - 32u * wave, 32u) : 0;  // the wave's query rows
    if (!__any(bad)) {  // wave-uniform
        // the wave's rows through LDS, so that they are written whole
        const float f = direct ? 1.0f / l : 1.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float* const to = so + c * OROW + VW * (8 * (i / 4) + 4 * hh + i % 4);
            if constexpr (DV == 2)
                *reinterpret_cast<float4*>(to) = make_float4(o[0][i] * f, o[1][i] * f, o[2][i] * f, o[3][i] * f);
            else *reinterpret_cast<float2*>(to) = make_float2(o[0][i] * f, o[1][i] * f);
        }
        const uint32_t d4 = D / 4;
        const bool al = !direct || aligned;
        const auto place_of = [&](uint32_t x) {
            const uint32_t rr = it.r0 + 32u * wave + x;
            return static_cast<uint64_t>(it.t0 + rr / G) * e.heads + kvh * G + rr % G;
        };
        for (uint32_t i = lane; i < mine_here * d4; i += kWave) {
            const uint32_t x = i / d4, d = 4 * (i % d4);
            const float4 v = *reinterpret_cast<const float4*>(so + x * OROW + d);
            const uint64_t to = place_of(x);
            store4(direct ? e.out + to * D + d : e.part + (to * e.slots + it.slot) * D + d, v, al);
        }
        if (static_cast<uint32_t>(lane) < mine_here)  // (lanes c of the lower half: query c)
            paged_state(e, it, place_of(lane), m, l);
        return;
    }
    // Values that are not finite somewhere: the wave's queries again, in f32, 16 at a time.
    for (uint32_t q0 = 32u * wave; q0 < min(count, 32u * wave + 32); q0 += 16) {
        const uint32_t rr = it.r0 + min(q0 + lane % 16, count - 1);
        const uint64_t to = static_cast<uint64_t>(it.t0 + rr / G) * e.heads + kvh * G + rr % G;
        float* const own = so + lane % 16 * OROW;
        const float* const qr = e.q + to * D;
        slow_tiles(e, keys, it.b, kvh, stage0 * SG / 2, min(stages * SG, keys.groups + 1) / 2, 1, qr,
                   paged_mask(e, it, it.len + rr / G), c2, own, m, l);
        l += lane_xor16(l);
        l += lane_xor32(l);
        if (q0 + lane % 16 >= count) continue;
        const float f = direct ? 1.0f / l : 1.f;
        float* const d0 = direct ? e.out + to * D : e.part + (to * e.slots + it.slot) * D;
        for (uint32_t d = lane / 16; d < D; d += 4) d0[d] = own[d] * f;
        if (lane < 16) paged_state(e, it, to, m, l);
    }
}

}  // namespace

hipError_t launch_paged_tiles(const PagedGeo& g, hipStream_t s) {
    const unsigned grid = paged_blocks(g);
    const bool exact = g.head_dim % 64 == 0;
    if (g.head_dim <= 64) {
        if (exact) paged_tiles<1, true><<<grid, 64 * NW, 0, s>>>(g);
        else paged_tiles<1, false><<<grid, 64 * NW, 0, s>>>(g);
    } else {
        if (exact) paged_tiles<2, true><<<grid, 64 * NW, 0, s>>>(g);
        else paged_tiles<2, false><<<grid, 64 * NW, 0, s>>>(g);
    }
    return hipGetLastError();
}

hipError_t load_code_paged_tiles() {
    hipFuncAttributes attr;
    return hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&paged_tiles<1, true>));
}

}  // namespace slhip
