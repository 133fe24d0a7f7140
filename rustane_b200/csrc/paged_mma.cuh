// The tensor-core form of paged attention, for 16-bit pools: mma.m16n8k16 with sixteen rows of a unit per warp.
//
// A warp takes sixteen entries at a time.  K and V go from global memory straight to registers in the order the products need, 16 bytes a lane:
// for q K^T the sum over hd may run in any order, so a lane's 16 bytes of a K row serve as the operand of two products (q lies in
// shared memory in the same order); for P V a lane has the same eight columns of four entries, whose halves one byte permutation
// pairs up, and which column a product's n stands for is undone when the result is stored.  Nothing is staged, no barrier is met
// inside the loop, and a warp's loads of both K and V (8 KB at hd 128) are in flight together.  With up to 64 rows a unit the
// row warps read the same entries; all but the first find them in the L1.
//
// mma.sync and not tcgen05: a token's unit has 1 to 16 rows, of a 64-row minimum there, and the work is bound by the bytes of K and V
// (two products a byte pair at eight q heads a kv head are a twentieth of what the tensor cores do in that time).
//
// Exactness: q of 32 bits is two fp16 parts (scaled by a power of two per row) or three bf16 parts, P two or three parts with an fp32
// result or a bf16 pool (a single bf16 P would cost 2^-9 a term, half the result's own rounding) and one with fp16 (2^-12).  Sums
// stay in 32 bits; with an fp32 result every step's product goes to fresh accumulators and is added by the CUDA cores, which round
// to nearest where the tensor cores cut off.
#pragma once
#include "paged_attn.cuh"

namespace cd {

template <typename KT> struct Bits16;
template <> struct Bits16<__half> { static constexpr uint32_t EXP = 0x7c007c00u; };
template <> struct Bits16<__nv_bfloat16> { static constexpr uint32_t EXP = 0x7f807f80u; };
// whether one of the two 16-bit numbers is infinite or NaN
template <typename KT> __device__ inline bool not_finite(uint32_t w) {
    const uint32_t e = w & Bits16<KT>::EXP;
    return (e & 0xffffu) == (Bits16<KT>::EXP & 0xffffu) || (e >> 16) == (Bits16<KT>::EXP >> 16);
}
// the finite ones of the two, zero for the others
template <typename KT> __device__ inline uint32_t finite_part(uint32_t w) {
    const uint32_t e = w & Bits16<KT>::EXP;
    return w & (((e & 0xffffu) == (Bits16<KT>::EXP & 0xffffu) ? 0u : 0xffffu) | ((e >> 16) == (Bits16<KT>::EXP >> 16) ? 0u : 0xffff0000u));
}
__device__ inline uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <typename KT, typename QT> struct MmaForm {
    static constexpr bool F16 = std::is_same<KT, __half>::value, WIDE = std::is_same<QT, float>::value;
    static constexpr int NQ = WIDE ? (F16 ? 2 : 3) : 1, NP = WIDE ? (F16 ? 2 : 3) : F16 ? 1 : 2;
    static constexpr int SHIFT = F16 ? (NP == 2 ? 12 : 8) : 0;  // P is times 2^SHIFT: fp16 parts of small ones keep their digits
};
template <int HD> constexpr int mma_ctas() { return HD == 128 ? 3 : 4; }

template <typename KT, typename QT, int HD> __global__ void __launch_bounds__(PA_THREADS, mma_ctas<HD>()) attn_mma_kernel(const __grid_constant__ AttnArgs p) {
    using X = Mma16<KT>;
    using F = MmaForm<KT, QT>;
    constexpr int NQ = F::NQ, NP = F::NP, NI = HD / 32, NH = HD / 64, RW = 16, PAD = 4;  // NI: 16-byte chunks of a K row a lane has; NH: of a V row
    extern __shared__ __align__(16) char dyn[];
    __shared__ long long sums[PA_WARPS];
    __shared__ float2 sml[PA_WARPS * RW];
    __shared__ float qscale[4 * RW];
    long long* pre = reinterpret_cast<long long*>(dyn);
    char* area = dyn + ((size_t)(p.c.nseq + 1) * 8 + 15) / 16 * 16;
    uint4* sq = reinterpret_cast<uint4*>(area);  // [row warps][NQ][NI][2 halves][32 lanes]; then, in the same place:
    float* so = reinterpret_cast<float*>(area);  // [warps][RW][HD + PAD]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int rw = warp % p.row_warps, tg = warp / p.row_warps, groups = PA_WARPS / p.row_warps;
    const KT* pool = static_cast<const KT*>(p.c.pool);
    const bool page16 = (p.c.page_tokens & 15) == 0;

    walk_line(p, pre, sums, [&](const SeqWork& w, int b, int kvh, int block, int tile, int tiles, bool whole, size_t slot) {
        const int valid_rows = min(p.ru, w.s.n * p.group - block * p.ru);
        __syncthreads();  // the unit before has been read
        for (int r = warp; r < p.row_warps * RW; r += PA_WARPS) {
            constexpr int EL = HD / 32;  // elements of a lane: EL lane .. EL lane + EL - 1
            float x[EL];
            float most = 0.f;
            if (r < valid_rows) {
                const int rho = block * p.ru + r, j = rho / p.group, head = kvh * p.group + rho % p.group;
                const QT* src = static_cast<const QT*>(p.q) + (size_t)(w.s.r0 + j) * p.q_stride + (size_t)head * HD + lane * EL;
#pragma unroll
                for (int e = 0; e < EL; ++e) x[e] = as_float(src[e]);
            } else {
#pragma unroll
                for (int e = 0; e < EL; ++e) x[e] = 0.f;
            }
            float back = 1.f;
            if (F::F16 && F::WIDE) {
#pragma unroll
                for (int e = 0; e < EL; ++e) most = fmaxf(most, fabsf(x[e]));
                most = warp_max(most);
                if (most > 0.f && most < INFINITY) {
                    const int ex = max(-100, ilogbf(most)) - 7;
                    back = __int_as_float((127 + ex) << 23);
                    const float by = __int_as_float((127 - ex) << 23);
#pragma unroll
                    for (int e = 0; e < EL; ++e) x[e] *= by;
                }
            }
            if (lane == 0) qscale[r] = back * p.scale_log2;
            const int d = lane * EL, ch = d / 8, at = (r / RW * NQ * NI + ch / 4) * 2 + (r % RW) / 8;
#pragma unroll
            for (int part = 0; part < NQ; ++part) {
                uint32_t* dst = reinterpret_cast<uint32_t*>(sq + (size_t)(at + part * NI * 2) * 32 + (r % 8) * 4 + ch % 4) + (d % 8) / 2;
#pragma unroll
                for (int e = 0; e < EL; e += 2) dst[e / 2] = X::part(x[e], x[e + 1]);
            }
        }
        __syncthreads();
        float o[NH][8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, scale[2];
        int last[2];
        float* srow[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = rw * RW + g + 8 * h, rho = block * p.ru + r, j = rho / p.group;
            last[h] = r < valid_rows ? w.s.len - w.s.n + j : -1;
            scale[h] = qscale[r];
            srow[h] = p.scores && r < valid_rows ? p.scores + ((size_t)(w.s.r0 + j) * p.heads + kvh * p.group + rho % p.group) * p.score_stride : nullptr;
        }
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[h][i][e] = 0.f;
        const uint4* q4 = sq + (size_t)rw * NQ * NI * 2 * 32 + lane;
        const int first = w.start + tile * PA_TILE, end = min(w.s.len, first + tiles * PA_TILE);
        const int all_see = w.s.len - w.s.n, none_out = p.window > 0 ? w.s.len - p.window : 0;  // every row sees entries none_out .. all_see
        const bool mixed = w.s.n > 1 || p.window > 0;
        const size_t v_off = (size_t)p.c.kv_heads * p.c.page_tokens * HD;

        int t0 = first + tg * 16;
        int page = page16 && t0 < end ? page_at(p.c, b, t0) : -1;
        for (; t0 < end; t0 += groups * 16) {
            uint4 k[2][NI], v[4][NH];
            uint32_t there = 0;  // of this lane's score columns t0 + 2c, 2c + 1, 2c + 8, 2c + 9: bit i
            if (page16) {
                const int now = page;
                if (t0 + groups * 16 < end) page = page_at(p.c, b, t0 + groups * 16);
                if (now >= 0) {
                    const KT* base = pool + row_at(p.c, now, 0, kvh, t0, HD);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < NI; ++i)
                            k[h][i] = t0 + 8 * h + g < end ? __ldg(reinterpret_cast<const uint4*>(base + (8 * h + g) * HD) + i * 4 + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = 2 * c + (e & 1) + (e >> 1) * 8;
                        const bool in = t0 + t < end;
                        there |= (uint32_t)in << e;
#pragma unroll
                        for (int h = 0; h < NH; ++h) v[e][h] = in ? __ldg(reinterpret_cast<const uint4*>(base + v_off + t * HD) + h * 8 + g) : make_uint4(0, 0, 0, 0);
                    }
                }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int t = t0 + 8 * h + g, pg = t < end ? page_at(p.c, b, t) : -1;
                    const KT* row = pool + (pg >= 0 ? row_at(p.c, pg, 0, kvh, t, HD) : 0);
#pragma unroll
                    for (int i = 0; i < NI; ++i) k[h][i] = pg >= 0 ? __ldg(reinterpret_cast<const uint4*>(row) + i * 4 + c) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = t0 + 2 * c + (e & 1) + (e >> 1) * 8, pg = t < end ? page_at(p.c, b, t) : -1;
                    const KT* row = pool + (pg >= 0 ? row_at(p.c, pg, 1, kvh, t, HD) : 0);
                    there |= (uint32_t)(pg >= 0) << e;
#pragma unroll
                    for (int h = 0; h < NH; ++h) v[e][h] = pg >= 0 ? __ldg(reinterpret_cast<const uint4*>(row) + h * 8 + g) : make_uint4(0, 0, 0, 0);
                }
            }
            if (!__any_sync(0xffffffffu, there)) {  // a page outside the pool
                if (p.scores)
                    for (int t = t0 + c; t < min(end, t0 + 16); t += 4) {
                        if (srow[0]) srow[0][t] = -INFINITY;
                        if (srow[1]) srow[1][t] = -INFINITY;
                    }
                continue;
            }
            // scores s[n][row half * 2 + column]
            float s[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
            for (int part = NQ - 1; part >= 0; --part)
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const uint4 a0 = q4[((part * NI + i) * 2) * 32], a1 = q4[((part * NI + i) * 2 + 1) * 32];
                    const uint32_t lo[4] = {a0.x, a1.x, a0.y, a1.y}, hi[4] = {a0.z, a1.z, a0.w, a1.w};
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        X::mma(s[n], lo, k[n][i].x, k[n][i].y);
                        X::mma(s[n], hi, k[n][i].z, k[n][i].w);
                    }
                }
            const bool edge = t0 + 15 > all_see || t0 < none_out || there != 15u;
            const bool masked = __any_sync(0xffffffffu, edge);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[n][e] *= scale[e >> 1];
                    if (masked) {
                        const int t = t0 + n * 8 + 2 * c + (e & 1);
                        const bool seen = (there >> (n * 2 + (e & 1)) & 1u) && t <= last[e >> 1] && (p.window == 0 || t > last[e >> 1] - p.window);
                        if (!seen) s[n][e] = -INFINITY;
                    }
                }
            if (p.scores)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int t = t0 + n * 8 + 2 * c;
                        if (srow[h] && t + 1 < end) *reinterpret_cast<float2*>(srow[h] + t) = make_float2(s[n][2 * h], s[n][2 * h + 1]);
                        else if (srow[h] && t < end) srow[h][t] = s[n][2 * h];
                    }
            float top[2];
            bool raise = false;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float x = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                top[h] = fmaxf(m[h], x);
                raise |= top[h] > m[h];
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float f = top[h] == -INFINITY ? 1.f : exp2f(m[h] - top[h]);
                    m[h] = top[h];
                    l[h] *= f;
#pragma unroll
                    for (int a = 0; a < NH; ++a)
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            o[a][i][2 * h] *= f;
                            o[a][i][2 * h + 1] *= f;
                        }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float base = (m[h] == -INFINITY ? 0.f : m[h]) - (float)F::SHIFT;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    s[n][2 * h] = exp2f(s[n][2 * h] - base);
                    s[n][2 * h + 1] = exp2f(s[n][2 * h + 1] - base);
                    l[h] += s[n][2 * h] + s[n][2 * h + 1];
                }
            }
            if (masked && mixed) {  // what some rows do not see must not reach them through 0 * inf
                bool odd = false;
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int h = 0; h < NH; ++h) odd |= not_finite<KT>(v[e][h].x) | not_finite<KT>(v[e][h].y) | not_finite<KT>(v[e][h].z) | not_finite<KT>(v[e][h].w);
                if (__any_sync(0xffffffffu, odd)) {  // rare: what is not finite goes, entry by entry, to the rows that see it
#pragma unroll 1
                    for (int t = t0; t < min(end, t0 + 16); ++t) {
                        const int at = t - t0, from = (lane & ~3) | (at & 7) >> 1, pg = page_at(p.c, b, t);
                        float e0 = at & 8 ? (at & 1 ? s[1][1] : s[1][0]) : (at & 1 ? s[0][1] : s[0][0]);
                        float e1 = at & 8 ? (at & 1 ? s[1][3] : s[1][2]) : (at & 1 ? s[0][3] : s[0][2]);
                        e0 = __shfl_sync(0xffffffffu, e0, from);
                        e1 = __shfl_sync(0xffffffffu, e1, from);
                        if (pg < 0) continue;
                        const bool see0 = t <= last[0] && (p.window == 0 || t > last[0] - p.window), see1 = t <= last[1] && (p.window == 0 || t > last[1] - p.window);
                        const KT* row = pool + row_at(p.c, pg, 1, kvh, t, HD);
#pragma unroll
                        for (int a = 0; a < NH; ++a)
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float v0 = as_float(row[a * 64 + c * 16 + i]), v1 = as_float(row[a * 64 + c * 16 + 8 + i]);
                                if (!isfinite(v0)) {
                                    if (see0) o[a][i][0] = fmaf(e0, v0, o[a][i][0]);
                                    if (see1) o[a][i][2] = fmaf(e1, v0, o[a][i][2]);
                                }
                                if (!isfinite(v1)) {
                                    if (see0) o[a][i][1] = fmaf(e0, v1, o[a][i][1]);
                                    if (see1) o[a][i][3] = fmaf(e1, v1, o[a][i][3]);
                                }
                            }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int h = 0; h < NH; ++h)
                            v[e][h] = make_uint4(finite_part<KT>(v[e][h].x), finite_part<KT>(v[e][h].y), finite_part<KT>(v[e][h].z), finite_part<KT>(v[e][h].w));
                }
            }
            uint32_t pp[NP][4];
#pragma unroll
            for (int part = 0; part < NP; ++part) {
                pp[part][0] = X::part(s[0][0], s[0][1]);
                pp[part][1] = X::part(s[0][2], s[0][3]);
                pp[part][2] = X::part(s[1][0], s[1][1]);
                pp[part][3] = X::part(s[1][2], s[1][3]);
            }
#pragma unroll
            for (int a = 0; a < NH; ++a)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t pick = i & 1 ? 0x7632u : 0x5410u;
                    const uint32_t b0 = __byte_perm(word(v[0][a], i / 2), word(v[1][a], i / 2), pick), b1 = __byte_perm(word(v[2][a], i / 2), word(v[3][a], i / 2), pick);
                    if constexpr (F::WIDE) {
                        float fresh[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int part = NP - 1; part >= 0; --part) X::mma(fresh, pp[part], b0, b1);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[a][i][e] += fresh[e];
                    } else {
#pragma unroll
                        for (int part = NP - 1; part >= 0; --part) X::mma(o[a][i], pp[part], b0, b1);
                    }
                }
        }
        __syncthreads();  // q has been read; its place takes the parts
        constexpr float DOWN = 1.0f / (1 << F::SHIFT);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            const int r = warp * RW + g + 8 * h;
            if (c == 0) sml[r] = make_float2(m[h], l[h] * DOWN);
#pragma unroll
            for (int a = 0; a < NH; ++a) {  // columns 64 a + 16 c + i and + 8: two runs of eight
                float* dst = so + (size_t)r * (HD + PAD) + a * 64 + c * 16;
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    *reinterpret_cast<float4*>(dst + i) = make_float4(o[a][i][2 * h] * DOWN, o[a][i + 1][2 * h] * DOWN, o[a][i + 2][2 * h] * DOWN, o[a][i + 3][2 * h] * DOWN);
                    *reinterpret_cast<float4*>(dst + 8 + i) =
                        make_float4(o[a][i][2 * h + 1] * DOWN, o[a][i + 1][2 * h + 1] * DOWN, o[a][i + 2][2 * h + 1] * DOWN, o[a][i + 3][2 * h + 1] * DOWN);
                }
            }
        }
        __syncthreads();
        finish_unit<QT, HD, PAD>(p, UnitParts<HD, PAD>{so, sml}, RW, w, kvh, block, whole, slot);
    });
}

template <typename KT, typename QT, int HD> inline size_t mma_shared(int nseq, int row_warps) {
    const size_t q = (size_t)row_warps * MmaForm<KT, QT>::NQ * (HD / 32) * 2 * 32 * 16, o = (size_t)PA_WARPS * 16 * (HD + 4) * 4;
    return ((size_t)(nseq + 1) * 8 + 15) / 16 * 16 + (q > o ? q : o);
}

}  // namespace cd
