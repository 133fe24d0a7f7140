// The tensor-core form of paged attention, for 16-bit pools: mma.m16n8k16 with sixteen rows of a unit per warp.
//
// The warps that have different rows of the same entries (one, two or four, as the unit's rows need) are a group with a ring of stages in
// shared memory: 4 KB of K and 4 KB of V each (sixteen entries at hd 128, 32 at hd 64), brought by cp.async 16 bytes at a time.  K's
// half of a stage is filled again as soon as the scores are out, V's as soon as P V is.  A row's 16-byte chunks are exchanged by the low
// bits of its place (chunk ^ place & 7), so that ldmatrix meets every bank once and an address is one XOR.  A group of one warp meets no
// barrier inside the loop.
//
// What bounds it: HBM where one warp has a unit's rows (5.9 TB/s on a ragged batch of 48 over 1.6 GB, 272 us; 130001 entries of four heads, 266 MB,
// 56 us with their joint: 4.7 TB/s, the rest is the launch, the line and the ends of two kernels), the chain of a step's instructions, 5 to 9
// cycles each, where four do (48 rows over 167 MB 96 to 102 us), and the way to the first instruction of everything on a token of a few
// chats (11 us): a kernel's first pass waits for its code as well as for data, so copies stand in the code once and rare cases out of line.
//
// Forms measured on the way (the kernel alone, 130001 entries, where this one took 53): K and V straight to registers, no ring, 70 us; boxes by TMA,
// issued by a group's first thread, 59 (and 317 on the ragged batch of fp32 rows, then 290); by producer warps of their own, with the
// registers split, 64; three CTAs an SM with two stages and 168 registers 58, but the joint 6 us later, for which they leave no room.
//
// mma.sync and not tcgen05: a token's unit has 1 to 16 rows, of a 64-row minimum there, and the work is bound by the bytes of K and V.
//
// Exactness: q of 32 bits is two fp16 parts (scaled by a power of two per row) or three bf16 parts, P two parts or (bf16 pool, fp32 result)
// three: in one part every term would be off by 2^-12 (fp16) or 2^-9 (bf16) of itself, which terms that cancel leave of a small
// sum.  Sums stay in 32 bits; with an fp32 result every step's product goes to fresh accumulators and is added by the CUDA cores,
// which round to nearest where the tensor cores cut off.
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
    static constexpr int NQ = WIDE ? (F16 ? 2 : 3) : 1, NP = WIDE && !F16 ? 3 : 2;
    static constexpr int SHIFT = F16 ? 12 : 0;  // P is times 2^SHIFT: fp16 parts of small ones keep their digits
};
constexpr int MMA_STAGE = 8192;  // bytes of a stage: K, then V
// CTAs an SM, and stages of a CTA, which its groups share: two of twelve, at 224 registers a thread (they leave room for the joint's CTAs).
// Half the columns need half the sums: at hd 64, with units of one row warp, three CTAs of eight stages at 160 registers (48 sequences of up to
// 822 entries, 16 kv heads: 65 us for 69).  Drafted rows, whose units have several row warps, lose by it (106 us for 88; a group of four warps has
// four stages either way, so it is not the ring: fewer registers or fewer turns a CTA).  The parts of 32-bit q for several row warps take
// the room of four stages.
template <typename QT, int HD> struct MmaSize {
    static constexpr bool WIDE = std::is_same<QT, float>::value;
    static bool three(int row_warps) { return HD == 64 && !WIDE && row_warps == 1; }
    static int slots(int row_warps) { return three(row_warps) || (WIDE && row_warps > 1) ? 8 : 12; }
    // the most row warps that a build with so many stages meets
    __device__ static constexpr int most(int slots) { return (slots == 8) != WIDE && (WIDE || HD == 64) ? 1 : 4; }
};
template <typename KT, typename QT, int HD> inline size_t mma_shared(int nseq, int row_warps) {
    const size_t q = (size_t)row_warps * MmaForm<KT, QT>::NQ * (HD / 16) * 32 * 16, ring = (size_t)MmaSize<QT, HD>::slots(row_warps) * MMA_STAGE;
    const size_t o = (size_t)PA_WARPS * 16 * (HD + 4) * 4;  // (in the ring's place once it is empty)
    return (ring > o ? ring : o) + q + (size_t)(nseq + 1) * 4 + 1024;  // (1024: the ring's own alignment)
}
// Infinities and NaN.  A product in parts is not what the formula says of an infinity: q k with k infinite is NaN where a lower part of q is zero
// or of the other sign, p v likewise, and 0 * inf reaches rows that do not see the entry.  So (1) in tiles that some rows see only
// in part, what is not finite in V is taken out ahead of the products, and rows that see it are marked; (2) rows whose sums come out NaN
// are marked; (3) marked rows are worked out again, in fp32 FMAs, over all of the CTA's entries of the unit.  Rare, and therefore out of line.
//
// (1): which of this lane's rows (bit h: g + 8 h) see such an entry of the stage
template <typename KT, int HD, int TS> __device__ __noinline__ uint32_t odd_rows(const uint32_t* v, int t0, int end, int last0, int last1, int window) {
    const int lane = threadIdx.x & 31;
    uint32_t rows = 0;
    for (int at = 0; at < TS; ++at) {
        const int t = t0 + at;
        bool odd = false;
        for (int i = lane; i < HD / 2; i += 32) odd |= not_finite<KT>(v[at * HD / 2 + i]);
        if (__any_sync(0xffffffffu, odd) && t < end) rows |= (uint32_t)pa_sees(t, last0, window) | (uint32_t)pa_sees(t, last1, window) << 1;
    }
    return rows;
}
// (3): row r is in lane 4 (r % 8)'s bit of its row warp's marks, .x below 8 and .y from 8 on, of any of the groups.  All threads; ends with a barrier.
template <typename KT, typename QT, int HD, int PAD>
__device__ __noinline__ void rows_again(const AttnArgs& p, const SeqWork& w, int b, int kvh, int block, int first, int end, const uint2* marks, int row_warps, float2* ml, float* so) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = min(p.ru, w.s.n * p.group - block * p.ru);
    for (int r = warp; r < rows; r += PA_WARPS) {
        const int rw = r / 16, rr = r % 16;
        uint32_t marked = 0;
        for (int at = rw; at < PA_WARPS; at += row_warps) marked |= (rr < 8 ? marks[at].x : marks[at].y) >> 4 * (rr % 8) & 1u;
        if (!marked) continue;
        // a row with NaN in q is NaN already (a batch padded with rows of anything is not to pay for them)
        const int rho = block * p.ru + r;
        const QT* q = static_cast<const QT*>(p.q) + (size_t)(w.s.r0 + rho / p.group) * p.q_stride + (size_t)(kvh * p.group + rho % p.group) * HD;
        bool nan = false;
        for (int d = lane; d < HD; d += 32) nan |= isnan(as_float(q[d]));
        if (__any_sync(0xffffffffu, nan)) continue;
        float o[1][HD / 8], m[1], l[1];
        fma_rows<KT, QT, HD, 1>(p, w, b, kvh, block * p.ru + r, first, end, 4, m, l, o);
        fma_store<KT, HD, 1>(m, l, o, ml + rw * 16 + rr, so + (rw * 16 + rr) * (HD + PAD), HD + PAD);
        for (int at = rw + row_warps; at < PA_WARPS; at += row_warps) {  // the first group has all of it now
            if (lane == 0) ml[at * 16 + rr] = make_float2(-INFINITY, 0.f);
            for (int d = lane; d < HD; d += 32) so[(at * 16 + rr) * (HD + PAD) + d] = 0.f;
        }
    }
    __syncthreads();
}

template <int HD> struct MmaShared {
    float2 ml[PA_WARPS * 16];
    float qscale[4 * 16];
    uint2 marks[PA_WARPS];
};

// A run of one unit's tiles, its rows on ROW_WARPS warps.
template <typename KT, typename QT, int HD, int ROW_WARPS, int SLOTS>
__device__ __forceinline__ void mma_unit(const AttnArgs& p, char* ring_all, uint4* sq, MmaShared<HD>& sh, const SeqWork& w, int b, int kvh, int block, int tile, int tiles,
                                         bool whole, size_t slot) {
    using X = Mma16<KT>;
    using F = MmaForm<KT, QT>;
    constexpr int NQ = F::NQ, NP = F::NP, RW = 16, PAD = 4, TS = MMA_STAGE / 4 / HD, CH = HD / 8, KS = HD / 16, HALVES = TS / 16;  // TS: entries of a stage
    constexpr int groups = PA_WARPS / ROW_WARPS, gsize = ROW_WARPS * 32, STAGES = SLOTS / groups < 4 ? SLOTS / groups : 4;
    constexpr int PASS = gsize / CH, PASSES = TS / PASS, VOFF = MMA_STAGE / 2;  // PASS: rows that one copy of the whole group brings
    float* so = reinterpret_cast<float*>(ring_all);  // [warps][RW][HD + PAD]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    const int rw = warp % ROW_WARPS, tg = warp / ROW_WARPS, gt = rw * 32 + lane;
    const uint32_t ring_base = (uint32_t)__cvta_generic_to_shared(ring_all), ring = ring_base + tg * STAGES * MMA_STAGE;
    const KT* pool = static_cast<const KT*>(p.c.pool);
    const bool page16 = (p.c.page_tokens & 15) == 0;
    const size_t v_off = (size_t)p.c.kv_heads * p.c.page_tokens * HD, page_step = 2 * v_off;
    auto group_sync = [&]() {
        if constexpr (ROW_WARPS == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(tg + 1), "r"(gsize) : "memory");
    };
    // ldmatrix: lane l points at row l % 8 of matrix l / 8; a chunk's place is XORed in
    const int mr = lane & 7, mj = lane >> 3;
    const uint32_t k_at = (uint32_t)((mj >> 1) * 8 + mr) * HD * 2 + (((mj & 1) ^ mr) << 4), v_at = (uint32_t)((mj & 1) * 8 + mr) * HD * 2 + VOFF + (((mj >> 1) ^ mr) << 4);

    const int valid_rows = min(p.ru, w.s.n * p.group - block * p.ru);
    const int first = w.start + tile * PA_TILE, end = min(w.s.len, first + tiles * PA_TILE);
    __syncthreads();  // the unit before has been read
    // ---- the ring: page ids are looked up a step ahead of the copies
    int pages[HALVES];
    auto look_up = [&](int t0) {
        if (page16)
#pragma unroll
            for (int h = 0; h < HALVES; ++h) pages[h] = t0 + 16 * h < end ? page_word(p.c, b, t0 + 16 * h) : 0;
        else pages[0] = lane < TS && t0 + lane < end ? page_word(p.c, b, t0 + lane) : 0;  // of row `lane`
    };
    uint32_t gaps = 0;                                           // bit s: stage s lacks a page
    const int row0 = gt / CH, ch = gt % CH;                      // this thread's place in a pass
    const uint32_t put_at = ring + row0 * HD * 2 + ((ch ^ (row0 & 7)) << 4);
    const KT* head_at = pool + (size_t)kvh * p.c.page_tokens * HD + row0 * HD + ch * 8;
    int next = first + tg * TS, put = 0;                         // the step whose K is next, its stage
    const KT* from[HALVES];                                      // rows of the stage whose V is next: of each page
    uint32_t has = 0;                                            // bit k: this thread's row of pass k is there
    int odd_page = -1;                                           // (pages of odd sizes: of row `lane`)
    auto copy_half = [&](int half) {                             // 0: K, 1: V of the stage that `put` and the above describe
        const uint32_t to = put_at + put * MMA_STAGE + half * VOFF;
        const size_t off = half ? v_off : 0;
        constexpr uint32_t ALL = (1u << PASSES) - 1;
        if (page16 && has == ALL) {
#pragma unroll
            for (int k = 0; k < PASSES; ++k) copy16((to ^ ((k * PASS & 7) << 4)) + k * PASS * HD * 2, from[k * PASS / 16] + off + k * PASS % 16 * HD, true);
        } else if (page16) {
#pragma unroll
            for (int k = 0; k < PASSES; ++k) {
                const bool there = has >> k & 1u;
                copy16((to ^ ((k * PASS & 7) << 4)) + k * PASS * HD * 2, there ? from[k * PASS / 16] + off + k * PASS % 16 * HD : pool, there);
            }
        } else {
#pragma unroll 2
            for (int k = 0; k < PASSES; ++k) {
                const int row = row0 + k * PASS, pg = __shfl_sync(0xffffffffu, odd_page, row);
                copy16((to ^ ((k * PASS & 7) << 4)) + k * PASS * HD * 2, pg >= 0 ? pool + row_at(p.c, pg, 0, kvh, next + row, HD) + off + ch * 8 : pool, pg >= 0);
            }
        }
    };
    auto issue_k = [&]() {
        if (next < end) {
            bool lacks = false;
            if (page16) {
                has = 0;
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    const int t = next + 16 * h, off = p.c.page_shift >= 0 ? t & (p.c.page_tokens - 1) : t % p.c.page_tokens;
                    pages[h] = t < end ? checked_page(p.c, pages[h]) : -1;
                    from[h] = head_at + (size_t)max(pages[h], 0) * page_step + off * HD;
                    lacks |= pages[h] < 0 && t < end;
                }
                if (next + TS <= end && !lacks) has = (1u << PASSES) - 1;
                else
#pragma unroll
                    for (int k = 0; k < PASSES; ++k) has |= (uint32_t)(pages[k * PASS / 16] >= 0 && next + row0 + k * PASS < end) << k;
                look_up(next + groups * TS);
            } else {  // lane r looks up row r (every warp of the group all of them: they agree on gaps)
                const bool in = lane < TS && next + lane < end;
                odd_page = in ? checked_page(p.c, pages[0]) : -1;
                lacks = __any_sync(0xffffffffu, in && odd_page < 0);
                look_up(next + groups * TS);
            }
            gaps = (gaps & ~(1u << put)) | (uint32_t)lacks << put;
            copy_half(0);
        }
        copies_close();
    };
    auto issue_v = [&]() {
        if (next < end) copy_half(1);
        next += groups * TS;
        put = put + 1 == STAGES ? 0 : put + 1;
        copies_close();
    };
    look_up(next);
    // q comes ahead of the copies of K and V, which would otherwise be served first: as it is, into the place its parts will have
    constexpr int EL = HD / 32, QR = ROW_WARPS * RW / PA_WARPS;  // elements of a lane: EL lane .. EL lane + EL - 1; rows of a warp
    constexpr int QCH = HD * (int)sizeof(QT) / 16;
    for (int i = tid; i < ROW_WARPS * RW * QCH; i += PA_THREADS) {
        const int r = i / QCH, rho = block * p.ru + r, j = rho / p.group, head = kvh * p.group + rho % p.group;
        const bool there = r < valid_rows;
        copy16(smem_addr(sq) + i * 16, static_cast<const QT*>(p.q) + (there ? (size_t)(w.s.r0 + j) * p.q_stride + (size_t)head * HD + i % QCH * (16 / sizeof(QT)) : 0), there);
    }
    copies_close();
    float o[CH][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, scale[2];  // m: largest score before its scale, which is positive
    int last[2];
    float* srow[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = rw * RW + g + 8 * h, rho = block * p.ru + r, j = rho / p.group;
        last[h] = r < valid_rows ? w.s.len - w.s.n + j : -1;
        srow[h] = p.scores && r < valid_rows ? p.scores + ((size_t)(w.s.r0 + j) * p.heads + kvh * p.group + rho % p.group) * p.score_stride : nullptr;
    }
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    const uint4* q4 = sq + (size_t)rw * NQ * KS * 32 + lane;
    const int all_see = w.s.len - w.s.n, none_out = p.window > 0 ? w.s.len - p.window : 0;  // every row sees entries none_out .. all_see
    const bool mixed = w.s.n > 1 || p.window > 0;
    auto sees = [&](int t, int h) { return pa_sees(t, last[h], p.window); };

    uint32_t again = 0;  // marks of this lane's rows
    // Steps below 0 only issue copies: V of step it + STAGES - 1, K of step it + STAGES.  (One loop, so that the copies stand in the code
    // once: at its start a kernel waits for its instructions more than for anything else.)
    int get = 0, t0 = first + (tg - STAGES * groups) * TS;
#pragma unroll 1
    for (int it = -STAGES; it <= 0 || t0 < end; ++it, t0 += groups * TS) {
        const bool work = it >= 0 && t0 < end;
        if (it == 0) {  // ---- q, as the products' operand
            copies_wait<2 * STAGES - 1>();
            __syncthreads();
            float x[QR][EL];
#pragma unroll
            for (int qk = 0; qk < QR; ++qk)
#pragma unroll
                for (int e = 0; e < EL; ++e) x[qk][e] = as_float(reinterpret_cast<const QT*>(sq)[(warp + qk * PA_WARPS) * HD + lane * EL + e]);
            __syncthreads();
#pragma unroll
            for (int qk = 0; qk < QR; ++qk) {
                const int r = warp + qk * PA_WARPS;
                float back = 1.f;
                if (F::F16 && F::WIDE) {
                    float most = 0.f;
#pragma unroll
                    for (int e = 0; e < EL; ++e) most = fmaxf(most, fabsf(x[qk][e]));
                    most = warp_max(most);
                    if (most > 0.f && most < INFINITY) {
                        const int ex = max(-100, ilogbf(most)) - 14;  // the largest in [2^14, 2^15): two parts keep 2^-22 of elements down to 2^-18 of it
                        back = __int_as_float((127 + ex) << 23);
                        const float by = __int_as_float((127 - ex) << 23);
#pragma unroll
                        for (int e = 0; e < EL; ++e) x[qk][e] *= by;
                    }
                }
                if (lane == 0) sh.qscale[r] = fmaxf(back * p.scale_log2, 1e-37f);  // (0 times a masked score would be NaN)
                // row r, column d: register (d % 16 / 8) * 2 + r % 16 / 8 of lane (r % 8) * 4 + d % 8 / 2, k-step d / 16
#pragma unroll
                for (int part = 0; part < NQ; ++part)
#pragma unroll
                    for (int e = 0; e < EL; e += 2) {
                        const int d = lane * EL + e;
                        uint32_t* dst = reinterpret_cast<uint32_t*>(sq + ((size_t)(r / RW * NQ + part) * KS + d / 16) * 32 + (r % 8) * 4 + d % 8 / 2);
                        dst[d % 16 / 8 * 2 + r % RW / 8] = X::part(x[qk][e], x[qk][e + 1]);
                    }
            }
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h) scale[h] = sh.qscale[rw * RW + g + 8 * h];
        }
        if (work) {
            copies_wait<2 * STAGES - 2>();
            group_sync();  // K is there, and V of the step before has been read
        }
        if (it > -STAGES) issue_v();
        if (!work) {
            issue_k();
            continue;
        }
        const bool lacks = gaps >> get & 1u;
        const uint32_t stage = ring + get * MMA_STAGE;
        // scores s[n][row half * 2 + column] of entries t0 + 8 n + 2 c + column; two k-steps' operands at a time, into two sets of sums in turn
        float s[TS / 8][4], s2[TS / 8][4];
#pragma unroll
        for (int n = 0; n < TS / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = s2[n][e] = 0.f;
#pragma unroll
        for (int kb = 0; kb < KS / 2; ++kb) {
            constexpr int KB = 2;
            const uint32_t at = stage + k_at;
            uint32_t a[KB][NQ][4], k[KB][HALVES][4];
#pragma unroll
            for (int i = 0; i < KB; ++i) {
                const int ks = kb * KB + i;
#pragma unroll
                for (int h = 0; h < HALVES; ++h) ldsm(k[i][h], (at ^ (ks << 5)) + h * 16 * HD * 2);
#pragma unroll
                for (int part = 0; part < NQ; ++part) {
                    const uint4 x = q4[(part * KS + ks) * 32];
                    a[i][part][0] = x.x; a[i][part][1] = x.y; a[i][part][2] = x.z; a[i][part][3] = x.w;
                }
            }
#pragma unroll
            for (int i = 0; i < KB; ++i)
#pragma unroll
                for (int part = NQ - 1; part >= 0; --part)
#pragma unroll
                    for (int h = 0; h < HALVES; ++h) {
                        X::mma(kb & 1 ? s2[2 * h] : s[2 * h], a[i][part], k[i][h][0], k[i][h][1]);
                        X::mma(kb & 1 ? s2[2 * h + 1] : s[2 * h + 1], a[i][part], k[i][h][2], k[i][h][3]);
                    }
        }
#pragma unroll
        for (int n = 0; n < TS / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] += s2[n][e];
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
            top[h] = fmaxf(m[h], x);
            raise |= top[h] > m[h];
        }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float f = top[h] == -INFINITY ? 1.f : ex2((m[h] - top[h]) * scale[h]);
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
            // (the difference first: past 2^24 a rounded product of the maximum and the scale would be off by more than a power of two)
            const float base = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
            for (int n = 0; n < TS / 8; ++n) {
                s[n][2 * h] = ex2(fmaf(s[n][2 * h] - base, scale[h], (float)F::SHIFT));
                s[n][2 * h + 1] = ex2(fmaf(s[n][2 * h + 1] - base, scale[h], (float)F::SHIFT));
                l[h] += s[n][2 * h] + s[n][2 * h + 1];
            }
        }
        copies_wait<2 * STAGES - 2>();
        group_sync();  // V is there, and K has been read
        issue_k();
        get = get + 1 == STAGES ? 0 : get + 1;
        if (masked && mixed) {  // what some rows do not see must not reach them through 0 * inf
            const uint32_t* v = reinterpret_cast<const uint32_t*>(ring_all + (stage - ring_base) + VOFF);
            bool odd = false;
            for (int at = lane; at < TS * HD / 2; at += 32) odd |= not_finite<KT>(v[at]);
            if (__any_sync(0xffffffffu, odd)) {
                again |= odd_rows<KT, HD, TS>(v, t0, end, last[0], last[1], p.window);
                group_sync();  // the group's warps have all read the stage: take what is not finite out of it
                uint32_t* clean = const_cast<uint32_t*>(v);
                for (int at = gt; at < TS * HD / 2; at += gsize) clean[at] = finite_part<KT>(clean[at]);
                group_sync();
            }
        }
        const uint32_t at = stage + v_at;
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
            for (int nb = 0; nb < CH / 2; nb += 4) {  // 64 columns
                uint32_t v[4][4];
#pragma unroll
                for (int n = 0; n < 4; ++n) ldsm_t(v[n], (at ^ ((nb + n) << 5)) + h * 16 * HD * 2);
                if constexpr (F::WIDE) {
#pragma unroll
                    for (int n = 0; n < 4; n += 2) {
                        float f[4][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) f[i][e] = 0.f;
#pragma unroll
                        for (int part = NP - 1; part >= 0; --part)
#pragma unroll
                            for (int i = 0; i < 4; ++i) X::mma(f[i], pp[part], v[n + i / 2][i % 2 * 2], v[n + i / 2][i % 2 * 2 + 1]);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[2 * (nb + n) + i][e] += f[i][e];
                    }
                } else {
#pragma unroll
                    for (int part = NP - 1; part >= 0; --part)
#pragma unroll
                        for (int n = 0; n < 8; ++n) X::mma(o[2 * nb + n], pp[part], v[n / 2][n % 2 * 2], v[n / 2][n % 2 * 2 + 1]);
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
        bool nan = l[h] != l[h];
        if (c == 0) sh.ml[r] = make_float2(m[h] * scale[h], l[h] * DOWN);
#pragma unroll
        for (int n = 0; n < CH; ++n) {
            nan |= o[n][2 * h] != o[n][2 * h] || o[n][2 * h + 1] != o[n][2 * h + 1];
            *reinterpret_cast<float2*>(so + (size_t)r * (HD + PAD) + n * 8 + 2 * c) = make_float2(o[n][2 * h] * DOWN, o[n][2 * h + 1] * DOWN);
        }
        again |= (uint32_t)nan << h;
    }
    again |= __shfl_xor_sync(0xffffffffu, again, 1);
    again |= __shfl_xor_sync(0xffffffffu, again, 2);
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // (rows past the unit's, and those that see nothing, have no result to mend)
        const uint32_t x = __ballot_sync(0xffffffffu, again >> h & 1u && last[h] >= 0);
        if (lane == 0) (h ? sh.marks[warp].y : sh.marks[warp].x) = x;
    }
    __syncthreads();
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < PA_WARPS; ++i) any |= sh.marks[i].x | sh.marks[i].y;
    if (any) rows_again<KT, QT, HD, PAD>(p, w, b, kvh, block, first, end, sh.marks, ROW_WARPS, sh.ml, so);
    finish_unit<QT, HD, PAD>(p, UnitParts<HD, PAD>{so, sh.ml}, RW, ROW_WARPS, w, kvh, block, whole, slot);
}

template <typename KT, typename QT, int HD, int SLOTS, int REGS> __global__ void __maxnreg__(REGS) attn_mma_kernel(const __grid_constant__ AttnArgs p) {
    extern __shared__ char dyn[];
    __shared__ int sums[2 * PA_WARPS];
    __shared__ MmaShared<HD> sh;
    constexpr size_t RING = (size_t)SLOTS * MMA_STAGE, OUT = (size_t)PA_WARPS * 16 * (HD + 4) * 4;
    char* ring = dyn + ((1024 - (smem_addr(dyn) & 1023)) & 1023);
    uint4* sq = reinterpret_cast<uint4*>(ring + (RING > OUT ? RING : OUT));  // [row warps][NQ][KS][32 lanes]
    int* pre = reinterpret_cast<int*>(sq + (size_t)p.row_warps * MmaForm<KT, QT>::NQ * (HD / 16) * 32);
    pdl_launch_dependents();  // the joint's CTAs come in beside these
    int most;
    const int total = line_up(p, pre, sums, most);
    walk_line(p, pre, total, most, [&](const SeqWork& w, int b, int kvh, int block, int tile, int tiles, bool whole, size_t slot) {
        const int rows = min(p.ru, w.s.n * p.group - block * p.ru);
        if constexpr (MmaSize<QT, HD>::most(SLOTS) == 1) mma_unit<KT, QT, HD, 1, SLOTS>(p, ring, sq, sh, w, b, kvh, block, tile, tiles, whole, slot);
        else if (rows <= 16) mma_unit<KT, QT, HD, 1, SLOTS>(p, ring, sq, sh, w, b, kvh, block, tile, tiles, whole, slot);
        else if (rows <= 32) mma_unit<KT, QT, HD, 2, SLOTS>(p, ring, sq, sh, w, b, kvh, block, tile, tiles, whole, slot);
        else mma_unit<KT, QT, HD, 4, SLOTS>(p, ring, sq, sh, w, b, kvh, block, tile, tiles, whole, slot);
    });
}

}  // namespace cd
