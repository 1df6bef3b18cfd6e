// Storing new keys and values in a paged cache, rotated on the way (no
// reference counterpart; the rotation is reference/rope.rs:32-141, the copy
// reference/attention.rs:33-83 through a block table).
//
// Token t of row b, the i-th of its new ones, sits at position p = lens[b] + i:
// its keys are rotated by the angles p / theta^(2 pair / head_dim) and stored
// with its values in slot p % page_size of page table[b][p / page_size]; its
// queries, where given, are rotated into q_out. Angles, sines and cosines in
// f64, rounded once, the rotation in f32 without contraction, as the Rope
// operator has them.
//
// Bound by HBM: (2 heads + 4 kv_heads) head_dim floats per token. One block per
// token: its threads issue the loads of their first items, then work out the
// token's sines and cosines once for all heads while those are on their way.
// The powers theta^(2 pair / head_dim) come with the arguments, and the sines from
// sin_cos below: with the library's pow, sin and cos in every block, 8 tokens took
// 11.2 us and 2,000 (98 MB) 86 us.
#include "common.h"
#include "kernels.h"
#include "paged_geo.h"

namespace slhip {
namespace {

// Sine and cosine of an angle below 2^31: reduced to r in [-pi/4, pi/4] by
// multiples n of pi/2 in two parts (the first product is exact in its
// multiply-add, so r is off by 2^-53 or so), then the Taylor series, whose first
// terms left out, r^19 / 19! and r^20 / 20!, are below 2^-63. In f64's last bits they may
// differ from the library's, which after rounding to f32 shows about once in 2^28
// values.
__device__ __forceinline__ void sin_cos(double angle, float* sine, float* cosine) {
    const double n = rint(angle * 0.63661977236758134308);  // 2 / pi
    // pi / 2 = its f64 value + 6.123...e-17
    const double r = fma(-n, 6.123233995736766036e-17, fma(-n, 1.5707963267948965580, angle));
    const double z = r * r;
    constexpr auto inv_factorial = [](int k) {
        double f = 1.0;
        for (int i = 2; i <= k; ++i) f *= i;
        return 1.0 / f;
    };
    double s = inv_factorial(17), c = -inv_factorial(18);
    constexpr double s15 = -inv_factorial(15), s13 = inv_factorial(13), s11 = -inv_factorial(11),
                     s9 = inv_factorial(9), s7 = -inv_factorial(7), s5 = inv_factorial(5), s3 = -inv_factorial(3);
    constexpr double c16 = inv_factorial(16), c14 = -inv_factorial(14), c12 = inv_factorial(12),
                     c10 = -inv_factorial(10), c8 = inv_factorial(8), c6 = -inv_factorial(6), c4 = inv_factorial(4);
    s = fma(s, z, s15);
    c = fma(c, z, c16);
    s = fma(s, z, s13);
    c = fma(c, z, c14);
    s = fma(s, z, s11);
    c = fma(c, z, c12);
    s = fma(s, z, s9);
    c = fma(c, z, c10);
    s = fma(s, z, s7);
    c = fma(c, z, c8);
    s = fma(s, z, s5);
    c = fma(c, z, c6);
    s = fma(s, z, s3);
    c = fma(c, z, c4);
    s = fma(s * z, r, r);
    c = fma(fma(c, z, -0.5), z, 1.0);
    const int q = static_cast<int>(static_cast<int64_t>(n)) & 3;
    const double a = (q & 1) != 0 ? c : s, b = (q & 1) != 0 ? s : c;
    *sine = static_cast<float>((q & 2) != 0 ? -a : a);
    *cosine = static_cast<float>(q == 1 || q == 2 ? -b : b);
}

constexpr int kAppendIpt = 4;  // items whose loads a thread issues together

struct Item {
    uint32_t kind, head, c;  // 0: queries, 1: keys, 2: values
};
__device__ __forceinline__ Item item(uint32_t i, uint32_t nq, uint32_t nk, uint32_t per_head, uint32_t d4) {
    const uint32_t kind = i < nq ? 0 : i < nq + nk ? 1 : 2, x = i - (kind == 0 ? 0 : kind == 1 ? nq : nq + nk);
    const uint32_t per = kind == 2 ? d4 : per_head;
    return {kind, x / per, x % per};
}
// (by value: a choice among captured pointers would go through memory)
template <typename T>
__device__ __forceinline__ T* choose(uint32_t kind, T* q, T* k, T* v) {
    return kind == 0 ? q : kind == 1 ? k : v;
}

// An item is one float4 of pairs: NeoX the float4 c < head_dim / 8 with its
// partner head_dim / 2 further, GPT-J a float4 of two pairs; V items and
// unrotated ones are copies. Items of a token: q's, then k's, then v's.
template <bool ALIGNED>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a, RopePowers powers) {
    prefetch_kernarg<arg_bytes<PagedAppendArgs>()>();
    __shared__ float sc[256];  // [half] sine, [half] cosine; head_dim <= 256
    const uint32_t t = blockIdx.x, lane = threadIdx.x % kWave;
    uint32_t row = 0, start = 0, len = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += kWave) {
        const uint32_t b = min(b0 + lane, a.batch - 1);
        const uint32_t s = a.starts[b], l = a.lens[b];
        const uint64_t below = __ballot(b0 + lane < a.batch && s <= t);
        if (below == 0) break;
        const int last = 63 - __builtin_clzll(below);
        row = b0 + last;
        start = __builtin_amdgcn_readlane(s, last);
        len = __builtin_amdgcn_readlane(l, last);
        if (below != ~0ull) break;
    }
    const uint64_t position = static_cast<uint64_t>(len) + (t - start);
    // (no place for the token: cannot be with checked buffers)
    if (position >= static_cast<uint64_t>(a.pages_per_seq) * a.page_size) return;
    const uint32_t page_index = static_cast<uint32_t>(position / a.page_size);
    const uint32_t page = a.table[static_cast<uint64_t>(row) * a.pages_per_seq + page_index];
    if (page >= a.num_pages) return;
    const uint32_t D = a.head_dim, half = D / 2, d4 = D / 4;
    const bool rotated = a.rotate != 0, neox = a.interleaved == 0;
    // float4 items per head: NeoX pairs two float4s
    const uint32_t per_head = rotated && neox ? d4 / 2 : d4;
    const uint32_t nq = a.q != nullptr ? a.heads * per_head : 0, nk = a.kv_heads * per_head, nv = a.kv_heads * d4;
    const uint64_t kv_row = static_cast<uint64_t>(a.kv_heads) * D;
    const uint64_t slot = static_cast<uint64_t>(page) * 2 * a.page_size + position % a.page_size;
    float* const kdst = a.pool + slot * kv_row;
    float* const vdst = kdst + a.page_size * kv_row;
    const float* const qsrc = a.q + static_cast<uint64_t>(t) * a.heads * D;
    float* const qdst = a.q_out + static_cast<uint64_t>(t) * a.heads * D;
    const float* const ksrc = a.k + t * kv_row;
    const float* const vsrc = a.v + t * kv_row;
    const uint32_t total = nq + nk + nv;
    const uint32_t apart = rotated && neox ? half : 0;

    float4 v0[kAppendIpt], v1[kAppendIpt];
    const auto load = [&](uint32_t i0) {
#pragma unroll
        for (int u = 0; u < kAppendIpt; ++u) {
            const uint32_t i = i0 + u * 256;
            if (i >= total) continue;
            const Item x = item(i, nq, nk, per_head, d4);
            const float* const p = choose(x.kind, qsrc, ksrc, vsrc) + x.head * D + 4 * x.c;
            v0[u] = load4(p, ALIGNED);
            if (apart != 0 && x.kind != 2) v1[u] = load4(p + apart, ALIGNED);
        }
    };
    const auto store = [&](uint32_t i0) {
#pragma unroll
        for (int u = 0; u < kAppendIpt; ++u) {
            const uint32_t i = i0 + u * 256;
            if (i >= total) continue;
            const Item x = item(i, nq, nk, per_head, d4);
            const uint32_t c = x.c;
            float* const p = choose(x.kind, qdst, kdst, vdst) + x.head * D + 4 * c;
            const bool is_v = x.kind == 2;
            // (the pool is 16-byte aligned, q_out as ALIGNED says)
            const bool al = ALIGNED || x.kind != 0;
            if (is_v || !rotated) {
                store4(p, v0[u], al);
            } else if (neox) {
                const float4 x0 = v0[u], y0 = v1[u];
                const float s0 = sc[4 * c], s1 = sc[4 * c + 1], s2 = sc[4 * c + 2], s3 = sc[4 * c + 3];
                const float c0 = sc[half + 4 * c], c1 = sc[half + 4 * c + 1], c2 = sc[half + 4 * c + 2],
                            c3 = sc[half + 4 * c + 3];
                store4(p, make_float4(x0.x * c0 - y0.x * s0, x0.y * c1 - y0.y * s1, x0.z * c2 - y0.z * s2,
                                      x0.w * c3 - y0.w * s3), al);
                store4(p + half, make_float4(x0.x * s0 + y0.x * c0, x0.y * s1 + y0.y * c1, x0.z * s2 + y0.z * c2,
                                             x0.w * s3 + y0.w * c3), al);
            } else {
                const float4 z = v0[u];
                const float s0 = sc[2 * c], c0 = sc[half + 2 * c], s1 = sc[2 * c + 1], c1 = sc[half + 2 * c + 1];
                store4(p, make_float4(z.x * c0 - z.y * s0, z.x * s0 + z.y * c0, z.z * c1 - z.w * s1,
                                      z.z * s1 + z.w * c1), al);
            }
        }
    };
    load(threadIdx.x);
    if (rotated) {
        for (uint32_t pair = threadIdx.x; pair < half; pair += 256) {
            sin_cos(static_cast<double>(position) / powers.of[pair], &sc[pair], &sc[half + pair]);
        }
        __syncthreads();
    }
    store(threadIdx.x);
    for (uint32_t i0 = threadIdx.x + kAppendIpt * 256; i0 < total; i0 += kAppendIpt * 256) {
        load(i0);
        store(i0);
    }
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, const RopePowers& powers, hipStream_t s) {
    if (a.tokens == 0) return hipSuccess;
    const bool aligned = aligned16(a.k) && aligned16(a.v) && aligned16(a.q) && aligned16(a.q_out);
    if (aligned) paged_append_kernel<true><<<a.tokens, 256, 0, s>>>(a, powers);
    else paged_append_kernel<false><<<a.tokens, 256, 0, s>>>(a, powers);
    return hipGetLastError();
}

hipError_t load_code_paged_append() {
    hipFuncAttributes attr;
    return hipFuncGetAttributes(&attr, reinterpret_cast<const void*>(&paged_append_kernel<true>));
}

}  // namespace slhip
