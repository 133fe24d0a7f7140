// The tensor-core form of paged attention, for 16-bit pools: mma.m16n8k16 with sixteen rows of a unit per warp.
//
// The warps that have different rows of the same entries are a group with a ring of stages in shared memory: 8 KB of K and V each
// (sixteen entries at hd 128, 32 at hd 64), brought by cp.async 16 bytes at a time, two or more stages ahead of the products.  A row's 16-byte
// chunks are exchanged by the low bits of its place (chunk ^ place & 7), so that ldmatrix meets every bank once.  A group of one
// warp meets no barrier inside the loop at all.
//
// mma.sync and not tcgen05: a token's unit has 1 to 16 rows, of a 64-row minimum there, and the work is bound by the bytes of K and V.
// cp.async and not TMA tiles: pages may have any number of entries, places behind the last entry arrive as zeros, and the 64 KB an
// SM needs under way to keep HBM busy are there with two CTAs of four warps.  (K and V straight to registers, no ring: 774
// instructions per sixteen entries and 3.8 us between them at three CTAs an SM, 130001 entries of four heads 70 us.)
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
// 2^x to 2^-22 of itself; 0 for -inf
__device__ inline float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// (a, b) as a pair of 16-bit numbers; a and b become what is left
template <typename KT> __device__ inline uint32_t take_part(float& a, float& b);
template <> __device__ inline uint32_t take_part<__half>(float& a, float& b) {
    const __half2 p = __floats2half2_rn(a, b);
    const float2 f = __half22float2(p);
    a -= f.x;
    b -= f.y;
    return *reinterpret_cast<const uint32_t*>(&p);
}
template <> __device__ inline uint32_t take_part<__nv_bfloat16>(float& a, float& b) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&p);
    a -= __uint_as_float(w << 16);
    b -= __uint_as_float(w & 0xffff0000u);
    return w;
}
__device__ inline void copy16(uint32_t dst, const void* src, bool there) {  // zeros where not
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ inline void copies_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ inline void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ inline void ldsm(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ inline void ldsm_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

template <typename KT, typename QT> struct MmaForm {
    static constexpr bool F16 = std::is_same<KT, __half>::value, WIDE = std::is_same<QT, float>::value;
    static constexpr int NQ = WIDE ? (F16 ? 2 : 3) : 1, NP = WIDE ? (F16 ? 2 : 3) : F16 ? 1 : 2;
    static constexpr int SHIFT = F16 ? (NP == 2 ? 12 : 8) : 0;  // P is times 2^SHIFT: fp16 parts of small ones keep their digits
};
constexpr int MMA_STAGE = 8192, MMA_CTAS = 2;  // bytes of a stage: K, then V; CTAs an SM
// stages of a group's ring: with one row warp four groups of three (96 KB a CTA), with more row warps fewer groups of six
__host__ __device__ constexpr int mma_stages(int row_warps) { return row_warps == 1 ? 3 : 6; }
template <typename KT, typename QT, int HD, int ROW_WARPS> inline size_t mma_shared(int nseq) {
    const size_t q = (size_t)ROW_WARPS * MmaForm<KT, QT>::NQ * (HD / 16) * 32 * 16, ring = (size_t)PA_WARPS / ROW_WARPS * mma_stages(ROW_WARPS) * MMA_STAGE;
    const size_t o = (size_t)PA_WARPS * 16 * (HD + 4) * 4;  // (in the ring's place once it is empty)
    return ((size_t)(nseq + 1) * 4 + 127) / 128 * 128 + q + (ring > o ? ring : o);
}

template <typename KT, typename QT, int HD, int ROW_WARPS> __global__ void __launch_bounds__(PA_THREADS, MMA_CTAS) attn_mma_kernel(const __grid_constant__ AttnArgs p) {
    using X = Mma16<KT>;
    using F = MmaForm<KT, QT>;
    constexpr int NQ = F::NQ, NP = F::NP, RW = 16, PAD = 4, TS = MMA_STAGE / 4 / HD, CH = HD / 8, KS = HD / 16, HALVES = TS / 16;  // TS: entries of a stage
    constexpr int STAGES = mma_stages(ROW_WARPS), groups = PA_WARPS / ROW_WARPS, gsize = ROW_WARPS * 32, PASS = gsize / CH, PASSES = TS / PASS;  // PASS: rows a copy of the whole group brings
    extern __shared__ __align__(128) char dyn[];
    __shared__ int sums[PA_WARPS];
    __shared__ float2 sml[PA_WARPS * RW];
    __shared__ float qscale[4 * RW];
    int* pre = reinterpret_cast<int*>(dyn);
    uint4* sq = reinterpret_cast<uint4*>(dyn + ((size_t)(p.c.nseq + 1) * 4 + 127) / 128 * 128);  // [row warps][NQ][KS][32 lanes]
    char* ring_all = reinterpret_cast<char*>(sq + ROW_WARPS * NQ * KS * 32);
    float* so = reinterpret_cast<float*>(ring_all);  // [warps][RW][HD + PAD]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int rw = warp % ROW_WARPS, tg = warp / ROW_WARPS, gt = rw * 32 + lane;
    const uint32_t ring_base = (uint32_t)__cvta_generic_to_shared(ring_all), ring = ring_base + tg * STAGES * MMA_STAGE;
    const KT* pool = static_cast<const KT*>(p.c.pool);
    const bool page16 = (p.c.page_tokens & 15) == 0;
    const size_t v_off = (size_t)p.c.kv_heads * p.c.page_tokens * HD;
    auto group_sync = [&]() {
        if constexpr (ROW_WARPS == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(tg + 1), "r"(gsize) : "memory");
    };
    // ldmatrix: lane l points at row l % 8 of matrix l / 8
    const int mr = lane & 7, mj = lane >> 3;
    const uint32_t k_at = (uint32_t)((mj >> 1) * 8 + mr) * HD * 2, v_at = (uint32_t)((mj & 1) * 8 + mr) * HD * 2 + TS * HD * 2;

    pdl_launch_dependents();  // the joint's CTAs come in as these leave
    walk_line(p, pre, sums, [&](const SeqWork& w, int b, int kvh, int block, int tile, int tiles, bool whole, size_t slot) {
        const int valid_rows = min(p.ru, w.s.n * p.group - block * p.ru);
        const int first = w.start + tile * PA_TILE, end = min(w.s.len, first + tiles * PA_TILE);
        const int span = end - first - tg * TS, steps = span > 0 ? (span + groups * TS - 1) / (groups * TS) : 0;  // of this group
        __syncthreads();  // the unit before has been read
        // ---- the ring: page ids are looked up a step ahead of the copies
        int pages[HALVES];
        auto look_up = [&](int t0) {
            if (page16)
#pragma unroll
                for (int h = 0; h < HALVES; ++h) pages[h] = t0 + 16 * h < end ? page_at(p.c, b, t0 + 16 * h) : -1;
        };
        uint32_t gaps = 0;  // bit s: stage s lacks a page
        const int row0 = gt / CH, ch = gt % CH;  // this thread's place in a pass
        int next = 0, put = 0;                      // the step to issue, its stage
        auto issue = [&]() {
            if (next < steps) {
                const int t0 = first + (next * groups + tg) * TS;
                const uint32_t to = ring + put * MMA_STAGE + row0 * HD * 2;
                bool lacks = false;
                if (page16) {
                    const KT* half_at[HALVES];
#pragma unroll
                    for (int h = 0; h < HALVES; ++h) {
                        half_at[h] = pool + (pages[h] >= 0 ? row_at(p.c, pages[h], 0, kvh, t0 + 16 * h, HD) : 0) + row0 * HD + ch * 8;
                        lacks |= pages[h] < 0;
                    }
                    if (t0 + TS <= end && !lacks) {
#pragma unroll
                        for (int k = 0; k < PASSES; ++k) {
                            const KT* src = half_at[k * PASS / 16] + k * PASS % 16 * HD;
                            const uint32_t dst = to + k * PASS * HD * 2 + ((ch ^ ((row0 + k * PASS) & 7)) << 4);
                            copy16(dst, src, true);
                            copy16(dst + TS * HD * 2, src + v_off, true);
                        }
                    } else {
                        lacks = false;
#pragma unroll
                        for (int k = 0; k < PASSES; ++k) {
                            const bool there = pages[k * PASS / 16] >= 0 && t0 + row0 + k * PASS < end;
                            const KT* src = half_at[k * PASS / 16] + k * PASS % 16 * HD;
                            const uint32_t dst = to + k * PASS * HD * 2 + ((ch ^ ((row0 + k * PASS) & 7)) << 4);
                            copy16(dst, there ? src : pool, there);
                            copy16(dst + TS * HD * 2, there ? src + v_off : pool, there);
                        }
#pragma unroll
                        for (int h = 0; h < HALVES; ++h) lacks |= pages[h] < 0 && t0 + 16 * h < end;
                    }
                    look_up(t0 + groups * TS);
                } else {  // pages of odd sizes: lane r looks up row r (every warp of the group all of them: they agree on gaps)
                    const bool in = lane < TS && t0 + lane < end;
                    const int mine = in ? page_at(p.c, b, t0 + lane) : -1;
                    lacks = __any_sync(0xffffffffu, in && mine < 0);
#pragma unroll
                    for (int k = 0; k < PASSES; ++k) {
                        const int row = row0 + k * PASS, pg = __shfl_sync(0xffffffffu, mine, row);
                        const bool there = pg >= 0;
                        const KT* src = pool + (there ? row_at(p.c, pg, 0, kvh, t0 + row, HD) + ch * 8 : 0);
                        const uint32_t dst = to + k * PASS * HD * 2 + ((ch ^ (row & 7)) << 4);
                        copy16(dst, src, there);
                        copy16(dst + TS * HD * 2, src + (there ? v_off : 0), there);
                    }
                }
                gaps = (gaps & ~(1u << put)) | (uint32_t)lacks << put;
            }
            ++next;
            put = put + 1 == STAGES ? 0 : put + 1;
            copies_close();
        };
        look_up(first + tg * TS);
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) issue();
        // ---- q, as the products' operand
        for (int r = warp; r < ROW_WARPS * RW; r += PA_WARPS) {
            constexpr int EL = HD / 32;  // elements of a lane: EL lane .. EL lane + EL - 1
            float x[EL];
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
                float most = 0.f;
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
            // row r, column d: register (d % 16 / 8) * 2 + r % 16 / 8 of lane (r % 8) * 4 + d % 8 / 2, k-step d / 16
#pragma unroll
            for (int part = 0; part < NQ; ++part)
#pragma unroll
                for (int e = 0; e < EL; e += 2) {
                    const int d = lane * EL + e;
                    uint32_t* dst = reinterpret_cast<uint32_t*>(sq + ((size_t)(r / RW * NQ + part) * KS + d / 16) * 32 + (r % 8) * 4 + d % 8 / 2);
                    dst[d % 16 / 8 * 2 + r % RW / 8] = X::part(x[e], x[e + 1]);
                }
        }
        __syncthreads();
        float o[CH][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, scale[2];
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
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
        const uint4* q4 = sq + (size_t)rw * NQ * KS * 32 + lane;
        const int all_see = w.s.len - w.s.n, none_out = p.window > 0 ? w.s.len - p.window : 0;  // every row sees entries none_out .. all_see
        const bool mixed = w.s.n > 1 || p.window > 0;
        auto sees = [&](int t, int h) { return t <= last[h] && (p.window == 0 || t > last[h] - p.window); };

        int get = 0;
        for (int t0 = first + tg * TS; t0 < end; t0 += groups * TS) {
            copies_wait<STAGES - 2>();
            group_sync();  // the stage is complete, and the one behind it has been read
            const bool lacks = gaps >> get & 1u;
            issue();
            const uint32_t stage = ring + get * MMA_STAGE;
            get = get + 1 == STAGES ? 0 : get + 1;
            // scores s[n][row half * 2 + column] of entries t0 + 8 n + 2 c + column
            float s[TS / 8][4];
#pragma unroll
            for (int n = 0; n < TS / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t a[NQ][4];
#pragma unroll
                for (int part = 0; part < NQ; ++part) {
                    const uint4 x = q4[(part * KS + ks) * 32];
                    a[part][0] = x.x; a[part][1] = x.y; a[part][2] = x.z; a[part][3] = x.w;
                }
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    uint32_t k[4];
                    ldsm(k, stage + h * 16 * HD * 2 + k_at + (((ks * 2 + (mj & 1)) ^ mr) << 4));
#pragma unroll
                    for (int part = NQ - 1; part >= 0; --part) {
                        X::mma(s[2 * h], a[part], k[0], k[1]);
                        X::mma(s[2 * h + 1], a[part], k[2], k[3]);
                    }
                }
            }
            const bool masked = t0 + TS - 1 > all_see || t0 < none_out || t0 + TS > end || lacks;
            if (masked)
#pragma unroll
                for (int n = 0; n < TS / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = t0 + n * 8 + 2 * c + (e & 1);
                        if (!(sees(t, e >> 1) && t < end && (!lacks || page_at(p.c, b, t) >= 0))) s[n][e] = -INFINITY;
                    }
            if (p.scores)
#pragma unroll
                for (int n = 0; n < TS / 8; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int t = t0 + n * 8 + 2 * c;
                        if (srow[h] && t + 1 < end) *reinterpret_cast<float2*>(srow[h] + t) = make_float2(s[n][2 * h] * scale[h], s[n][2 * h + 1] * scale[h]);
                        else if (srow[h] && t < end) srow[h][t] = s[n][2 * h] * scale[h];
                    }
            float top[2];
            bool raise = false;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float x = fmaxf(s[0][2 * h], s[0][2 * h + 1]);
#pragma unroll
                for (int n = 1; n < TS / 8; ++n) x = fmaxf(x, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                top[h] = fmaxf(m[h], x * scale[h]);  // (scale is positive)
                raise |= top[h] > m[h];
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float f = top[h] == -INFINITY ? 1.f : ex2(m[h] - top[h]);
                    m[h] = top[h];
                    l[h] *= f;
#pragma unroll
                    for (int n = 0; n < CH; ++n) {
                        o[n][2 * h] *= f;
                        o[n][2 * h + 1] *= f;
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float base = (m[h] == -INFINITY ? 0.f : m[h]) - (float)F::SHIFT;
#pragma unroll
                for (int n = 0; n < TS / 8; ++n) {
                    s[n][2 * h] = ex2(fmaf(s[n][2 * h], scale[h], -base));
                    s[n][2 * h + 1] = ex2(fmaf(s[n][2 * h + 1], scale[h], -base));
                    l[h] += s[n][2 * h] + s[n][2 * h + 1];
                }
            }
            if (masked && mixed) {  // what some rows do not see must not reach them through 0 * inf
                const uint32_t* v = reinterpret_cast<const uint32_t*>(ring_all) + ((stage - ring_base) + TS * HD * 2) / 4;
                bool odd = false;
                for (int at = lane; at < TS * HD / 2; at += 32) odd |= not_finite<KT>(v[at]);
                if (__any_sync(0xffffffffu, odd)) {  // rare: what is not finite goes, entry by entry, to the rows that see it
#pragma unroll 1
                    for (int at = 0; at < TS; ++at) {
                        const int t = t0 + at, from = (lane & ~3) | (at & 7) >> 1;
                        float e0 = 0.f, e1 = 0.f;
#pragma unroll
                        for (int n = 0; n < TS / 8; ++n)
                            if (at >> 3 == n) {
                                e0 = at & 1 ? s[n][1] : s[n][0];
                                e1 = at & 1 ? s[n][3] : s[n][2];
                            }
                        e0 = __shfl_sync(0xffffffffu, e0, from);
                        e1 = __shfl_sync(0xffffffffu, e1, from);
                        if (t >= end) continue;
                        const bool see0 = sees(t, 0), see1 = sees(t, 1);
#pragma unroll
                        for (int n = 0; n < CH; ++n) {
                            const uint32_t word = v[at * HD / 2 + ((n ^ (at & 7)) << 2) + c];
                            if (!not_finite<KT>(word)) continue;
                            const float v0 = as_float(reinterpret_cast<const KT*>(&word)[0]), v1 = as_float(reinterpret_cast<const KT*>(&word)[1]);
                            if (!isfinite(v0)) {
                                if (see0) o[n][0] = fmaf(e0, v0, o[n][0]);
                                if (see1) o[n][2] = fmaf(e1, v0, o[n][2]);
                            }
                            if (!isfinite(v1)) {
                                if (see0) o[n][1] = fmaf(e0, v1, o[n][1]);
                                if (see1) o[n][3] = fmaf(e1, v1, o[n][3]);
                            }
                        }
                    }
                    group_sync();  // the group's warps have all read the stage: take what is not finite out of it
                    uint32_t* clean = const_cast<uint32_t*>(v);
                    for (int at = gt; at < TS * HD / 2; at += gsize) clean[at] = finite_part<KT>(clean[at]);
                    group_sync();
                }
            }
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                uint32_t pp[NP][4];
#pragma unroll
                for (int part = 0; part < NP; ++part) {
                    pp[part][0] = take_part<KT>(s[2 * h][0], s[2 * h][1]);
                    pp[part][1] = take_part<KT>(s[2 * h][2], s[2 * h][3]);
                    pp[part][2] = take_part<KT>(s[2 * h + 1][0], s[2 * h + 1][1]);
                    pp[part][3] = take_part<KT>(s[2 * h + 1][2], s[2 * h + 1][3]);
                }
#pragma unroll
                for (int n = 0; n < CH; n += 2) {
                    uint32_t v[4];
                    ldsm_t(v, stage + h * 16 * HD * 2 + v_at + (((n + (mj >> 1)) ^ mr) << 4));
                    if constexpr (F::WIDE) {
                        float f0[4] = {0.f, 0.f, 0.f, 0.f}, f1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int part = NP - 1; part >= 0; --part) {
                            X::mma(f0, pp[part], v[0], v[1]);
                            X::mma(f1, pp[part], v[2], v[3]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            o[n][e] += f0[e];
                            o[n + 1][e] += f1[e];
                        }
                    } else {
#pragma unroll
                        for (int part = NP - 1; part >= 0; --part) {
                            X::mma(o[n], pp[part], v[0], v[1]);
                            X::mma(o[n + 1], pp[part], v[2], v[3]);
                        }
                    }
                }
            }
        }
        copies_wait<0>();
        __syncthreads();  // the ring is empty; its place takes the parts
        constexpr float DOWN = 1.0f / (1 << F::SHIFT);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            const int r = warp * RW + g + 8 * h;
            if (c == 0) sml[r] = make_float2(m[h], l[h] * DOWN);
#pragma unroll
            for (int n = 0; n < CH; ++n)
                *reinterpret_cast<float2*>(so + (size_t)r * (HD + PAD) + n * 8 + 2 * c) = make_float2(o[n][2 * h] * DOWN, o[n][2 * h + 1] * DOWN);
        }
        __syncthreads();
        finish_unit<QT, HD, PAD>(p, UnitParts<HD, PAD>{so, sml}, RW, w, kvh, block, whole, slot);
    });
}

}  // namespace cd
