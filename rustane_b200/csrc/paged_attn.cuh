// Attention of a batch's new rows over paged K and V (cd_paged_attention).
//
// o = sum_t p_t v_t, p = softmax(scale q k_t) over the entries a row sees.  A unit is (sequence, kv head, block of RU rows): its
// rows are the q heads of the kv head times the sequence's new rows, so K and V are read once for all of them.  A unit's entries are cut into tiles of 64 and
// all units' tiles lie on one line, which the CTAs share evenly: each of G = min(grid, T) CTAs takes T / G of them or one more, whatever the lengths are
// (they are known on the device only; every CTA adds them up for itself).  A unit that one CTA has whole is finished there;
// the others leave (max, sum, sum of p v) per CTA in slot CTA + unit (both only ever grow along the line, so no two meet),
// and join_kernel puts them together in the line's order.  Inside a CTA four warps share a unit: `row_warps` of them have different rows of
// the same entries, the rest other entries.  Statistics are fp32 in the log2 domain.
#pragma once
#include "paged_span.h"
#include "serve.cuh"

namespace cd {

constexpr int PA_THREADS = 128, PA_WARPS = 4, PA_MAX_CTAS = 640;

struct AttnArgs {
    PagedView c;
    const int* row_start;
    const void* q;
    void* out;
    float* lse;       // natural log, or nullptr
    float* part_o;    // [ctas + units][ru][hd]
    float2* part_ml;  // [ctas + units][ru] (max, sum)
    int2* unit_info;  // [units] first CTA, CTAs
    float* lse2;      // [nrows][heads] log2; with scores only
    float* scores;    // [nrows][heads][score_stride] log2 domain, or nullptr
    long long q_stride, score_stride;
    int weights[3];  // what a tile of a unit of up to 16, 32 and more rows costs on the line; the first is the least
    float scale_log2;
    int heads, group, nrows, max_rows, window, ru, row_warps, blocks;  // blocks: row blocks a sequence may have
};

struct SeqWork {
    BatchSeq s;
    int start, tiles, blocks, weight;
};
__device__ inline SeqWork seq_work(const AttnArgs& p, int b) {
    SeqWork w;
    w.s = batch_seq(p.c, p.row_start, b, p.nrows, p.max_rows);
    const PaSpan span = pa_span(w.s.len, w.s.n, p.window);
    w.start = span.start;
    w.tiles = span.tiles;
    const int rows = w.s.n * p.group;
    w.blocks = (rows + p.ru - 1) / p.ru;
    w.weight = p.weights[rows <= 16 ? 0 : rows <= 32 ? 1 : 2];
    return w;
}

// pre[b] = cost of the sequences before b (all threads; ends with a barrier), most = the dearest tile; returns the total (the host keeps
// it below 2^31).  sums: 2 PA_WARPS words.
__device__ inline int line_up(const AttnArgs& p, int* pre, int* sums, int& most) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int carry = 0;
    most = 1;
    if (tid == 0) pre[0] = 0;
    for (int base = 0; base < p.c.nseq; base += PA_THREADS) {
        const int b = base + tid;
        int v = 0, dear = 1;
        if (b < p.c.nseq) {
            const SeqWork w = seq_work(p, b);
            if (w.tiles) dear = w.weight;
            v = w.tiles * w.weight * w.blocks * p.c.kv_heads;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += x;
        }
        dear = __reduce_max_sync(0xffffffffu, dear);
        if (lane == 31) {
            sums[warp] = v;
            sums[PA_WARPS + warp] = dear;
        }
        __syncthreads();
        int before = carry;
#pragma unroll
        for (int i = 0; i < PA_WARPS; ++i) {
            if (i < warp) before += sums[i];
            carry += sums[i];
            most = max(most, sums[PA_WARPS + i]);
        }
        if (b < p.c.nseq) pre[b + 1] = before + v;
        __syncthreads();
    }
    return carry;
}

constexpr float LN2 = 0.69314718055994530942f;

// One row's end: o relative to 2^m with sum l.  l is 0 where nothing was seen.
template <typename QT> __device__ inline void store_out(const AttnArgs& p, size_t row_head, int hd, int col, float o, float l) {
    static_cast<QT*>(p.out)[row_head * hd + col] = from_float<QT>(l > 0.f || l != l ? o / l : 0.f);
}
template <typename QT> __device__ inline void store_out4(const AttnArgs& p, size_t row_head, int hd, int c4, const float4& o, float l) {
    const bool some = l > 0.f || l != l;
    const float x[4] = {some ? o.x / l : 0.f, some ? o.y / l : 0.f, some ? o.z / l : 0.f, some ? o.w / l : 0.f};
    struct alignas(4 * sizeof(QT)) Four { QT e[4]; } v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v.e[e] = from_float<QT>(x[e]);
    *reinterpret_cast<Four*>(static_cast<QT*>(p.out) + row_head * hd + c4 * 4) = v;
}
__device__ inline void store_lse(const AttnArgs& p, size_t row_head, float m, float l) {
    const float lse2 = l > 0.f || l != l ? m + log2f(l) : -INFINITY;
    if (p.lse) p.lse[row_head] = lse2 * LN2;
    if (p.scores) p.lse2[row_head] = lse2;
}

// What the warps of a CTA leave of a unit: o[w][rows][HD + PAD], (m, l)[w][rows], warp w = entry group * row_warps + row group.
template <int HD, int PAD> struct UnitParts {
    float* o;
    float2* ml;
};
// Merge the entry groups and store: the result where the unit is this CTA's alone, else this CTA's slot.  All threads.
template <typename QT, int HD, int PAD>
__device__ inline void finish_unit(const AttnArgs& p, const UnitParts<HD, PAD>& u, int rows_per_warp, int row_warps, const SeqWork& w, int kvh, int block, bool whole, size_t slot) {
    const int groups = PA_WARPS / row_warps, rows = min(p.ru, w.s.n * p.group - block * p.ru);
    for (int at = threadIdx.x; at < rows * (HD / 4); at += PA_THREADS) {
        const int r = at / (HD / 4), c4 = at % (HD / 4), rw = r / rows_per_warp, rr = r % rows_per_warp;
        float m = -INFINITY;
        for (int t = 0; t < groups; ++t) m = fmaxf(m, u.ml[(t * row_warps + rw) * rows_per_warp + rr].x);
        const float base = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int t = 0; t < groups; ++t) {
            const int at_w = (t * row_warps + rw) * rows_per_warp + rr;
            const float2 ml = u.ml[at_w];
            const float f = exp2f(ml.x - base);
            const float4 x = *reinterpret_cast<const float4*>(u.o + (size_t)at_w * (HD + PAD) + c4 * 4);
            l += ml.y * f;
            o.x += x.x * f; o.y += x.y * f; o.z += x.z * f; o.w += x.w * f;
        }
        if (whole) {
            const int rho = block * p.ru + r, j = rho / p.group, head = kvh * p.group + rho % p.group;
            const size_t row_head = (size_t)(w.s.r0 + j) * p.heads + head;
            store_out4<QT>(p, row_head, HD, c4, o, l);
            if (c4 == 0) store_lse(p, row_head, m, l);
        } else {
            *reinterpret_cast<float4*>(p.part_o + (slot * p.ru + r) * HD + c4 * 4) = o;
            if (c4 == 0) p.part_ml[slot * p.ru + r] = make_float2(m, l);
        }
    }
}

// Walk this CTA's share of the line; work(w, b, kvh, block, first tile, tiles, whole, slot) handles a run of one unit's tiles.
// A tile belongs to the CTA whose share its first point lies in; no share is shorter than a tile, so none is empty.
template <typename F> __device__ inline void walk_line(const AttnArgs& p, const int* pre, int total, int most, F&& work) {
    const int ctas = min((int)gridDim.x, max(1, total / most)), me = blockIdx.x;
    if (me >= ctas || total == 0) return;
    const int per = total / ctas, more = total - per * ctas, cut = more * (per + 1);  // the first `more` shares are one longer
    auto owner = [&](int t) { return t < cut ? t / (per + 1) : more + (t - cut) / per; };
    int t = me * per + min(me, more);
    const int end = t + per + (me < more);
    while (t < end) {
        int lo = 0, hi = p.c.nseq - 1;  // the last sequence that begins at t or before
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= t) lo = mid; else hi = mid - 1;
        }
        const SeqWork w = seq_work(p, lo);
        const int long_ = w.tiles * w.weight, in_seq = t - pre[lo], unit = in_seq / long_, in_unit = in_seq - unit * long_;
        const int kvh = unit / w.blocks, block = unit - kvh * w.blocks, u0 = t - in_unit;
        const int first = (in_unit + w.weight - 1) / w.weight, last = min(w.tiles, (end - u0 + w.weight - 1) / w.weight), n = last - first;
        if (n > 0) {
            const size_t slot_unit = ((size_t)lo * p.c.kv_heads + kvh) * p.blocks + block;
            const bool whole = n == w.tiles;
            if (first == 0 && threadIdx.x == 0) p.unit_info[slot_unit] = make_int2(me, whole ? 1 : owner(u0 + (w.tiles - 1) * w.weight) - me + 1);
            work(w, lo, kvh, block, first, n, whole, slot_unit + me);
        }
        t = u0 + long_;
    }
}

// ------------------------------------------------------------------------------------------------ fp32 FMAs
// RW rows of a unit (rho0 .. of all its blocks' rows) by one warp: eight lanes hold one entry's K (and V) row, a warp four entries side by side; each eight lanes keep
// (m, l, o) of their entries, here entries from + side, from + side + step .. of [first, end).
template <typename KT, typename QT, int HD, int RW>
__device__ __forceinline__ void fma_rows(const AttnArgs& p, const SeqWork& w, int b, int kvh, int rho0, int from, int end, int step, float (&m)[RW], float (&l)[RW], float (&o)[RW][HD / 8]) {
    constexpr int VEC = 16 / sizeof(KT), NC = HD / 8 / VEC;  // elements of a load, loads of a lane and row
    const int lane = threadIdx.x & 31, l8 = lane & 7, side = lane >> 3;
    const KT* pool = static_cast<const KT*>(p.c.pool);
    float q[RW][NC * VEC];
    int last[RW];        // the last entry a row sees, -1: none
    float* srow[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) {
        const int rho = rho0 + r, j = rho / p.group, head = kvh * p.group + rho % p.group;
        const bool valid = rho < w.s.n * p.group;
        last[r] = valid ? w.s.len - w.s.n + j : -1;
        m[r] = -INFINITY;
        l[r] = 0.f;
        srow[r] = p.scores && valid ? p.scores + ((size_t)(w.s.r0 + j) * p.heads + head) * p.score_stride : nullptr;
        const QT* src = static_cast<const QT*>(p.q) + (size_t)(valid ? w.s.r0 + j : 0) * p.q_stride + (size_t)(valid ? head : 0) * HD;
#pragma unroll
        for (int i = 0; i < NC * VEC; ++i) {
            q[r][i] = valid ? as_float(src[(i / VEC * 8 + l8) * VEC + i % VEC]) * p.scale_log2 : 0.f;
            o[r][i] = 0.f;
        }
    }
    // the next entries' rows are on their way while these are worked on; their page is looked up a step before that
    uint4 kn[NC], vn[NC];
    int page_n = -1, word = 0;
    auto look_up = [&](int t) { word = t < end ? page_word(p.c, b, t) : 0; };
    auto fetch = [&](int t) {
        page_n = t < end ? checked_page(p.c, word) : -1;
        if (page_n >= 0) {
            const KT *kr = pool + row_at(p.c, page_n, 0, kvh, t, HD), *vr = pool + row_at(p.c, page_n, 1, kvh, t, HD);
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                kn[i] = __ldg(reinterpret_cast<const uint4*>(kr) + i * 8 + l8);
                vn[i] = __ldg(reinterpret_cast<const uint4*>(vr) + i * 8 + l8);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NC; ++i) kn[i] = vn[i] = make_uint4(0, 0, 0, 0);
        }
    };
    int t0 = from + side;
    look_up(t0);
    fetch(t0);
    look_up(t0 + step);
    for (; __any_sync(0xffffffffu, t0 < end); t0 += step) {
        float k[NC * VEC], v[NC * VEC];
        const int page = page_n;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                k[i * VEC + e] = as_float(reinterpret_cast<const KT*>(&kn[i])[e]);
                v[i * VEC + e] = as_float(reinterpret_cast<const KT*>(&vn[i])[e]);
            }
        fetch(t0 + step);
        look_up(t0 + 2 * step);
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < NC * VEC; ++i) s = fmaf(q[r][i], k[i], s);
#pragma unroll
            for (int x = 1; x < 8; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            const bool seen = page >= 0 && pa_sees(t0, last[r], p.window);
            if (!seen) s = -INFINITY;
            if (srow[r] && l8 == r && t0 < end) srow[r][t0] = s;
            if (!seen) continue;  // what is masked does not reach the sums, whatever its V holds
            if (s > m[r] || s != s) {
                const float f = exp2f(m[r] - s);
                m[r] = s;
                l[r] *= f;
#pragma unroll
                for (int i = 0; i < NC * VEC; ++i) o[r][i] *= f;
            }
            const float e = exp2f(s - (m[r] == -INFINITY ? 0.f : m[r]));
            l[r] += e;
#pragma unroll
            for (int i = 0; i < NC * VEC; ++i) o[r][i] = fmaf(e, v[i], o[r][i]);
        }
    }
}
// Those rows' sums over the warp's four sides: (m, l) to ml[r], o to so[r * stride ..].
template <typename KT, int HD, int RW> __device__ __forceinline__ void fma_store(const float (&m)[RW], const float (&l)[RW], const float (&o)[RW][HD / 8], float2* ml, float* so, int stride) {
    constexpr int VEC = 16 / sizeof(KT);
    const int lane = threadIdx.x & 31, l8 = lane & 7;
#pragma unroll
    for (int r = 0; r < RW; ++r) {
        float top = m[r];
#pragma unroll
        for (int x = 8; x < 32; x <<= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, top, x);
            top = other > top || other != other ? other : top;
        }
        const float f = exp2f(m[r] - (top == -INFINITY ? 0.f : top));
        float sum = l[r] * f;
#pragma unroll
        for (int x = 8; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        if (lane == 0) ml[r] = make_float2(top, sum);
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
            float x = o[r][i] * f;
            x += __shfl_xor_sync(0xffffffffu, x, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 16);
            if (lane < 8) so[r * stride + (i / VEC * 8 + l8) * VEC + i % VEC] = x;
        }
    }
}

// For fp32 pools, where rounding K and V to 16 bits would cost what the pool is kept for.  Bound by the chain of an entry's
// instructions (hd / 8 FMAs, three shuffles and an exponential a row): 53 sequences of up to 953 entries, four heads, two rows,
// 140 MB, 82 us; 105 us with the rows asked for when they are needed.
template <typename QT, int HD> __global__ void __launch_bounds__(PA_THREADS, 2) attn_fma_kernel(const __grid_constant__ AttnArgs p) {
    constexpr int RW = 4, PAD = 4;
    extern __shared__ int pre[];
    __shared__ int sums[2 * PA_WARPS];
    __shared__ __align__(16) float so[PA_WARPS * RW * (HD + PAD)];
    __shared__ float2 sml[PA_WARPS * RW];
    const int warp = threadIdx.x >> 5, rw = warp % p.row_warps, tg = warp / p.row_warps, groups = PA_WARPS / p.row_warps;

    pdl_launch_dependents();
    int most;
    const int total = line_up(p, pre, sums, most);
    walk_line(p, pre, total, most, [&](const SeqWork& w, int b, int kvh, int block, int tile, int tiles, bool whole, size_t slot) {
        const int first = w.start + tile * PA_TILE, end = min(w.s.len, first + tiles * PA_TILE);
        float o[RW][HD / 8], m[RW], l[RW];
        fma_rows<float, QT, HD, RW>(p, w, b, kvh, block * p.ru + rw * RW, first + tg * 4, end, groups * 4, m, l, o);
        __syncthreads();  // the unit before has been read
        fma_store<float, HD, RW>(m, l, o, sml + warp * RW, so + warp * RW * (HD + PAD), HD + PAD);
        __syncthreads();
        finish_unit<QT, HD, PAD>(p, UnitParts<HD, PAD>{so, sml}, RW, p.row_warps, w, kvh, block, whole, slot);
    });
}

// ------------------------------------------------------------------------------------------------ the joint
// One row and q head of a unit that several CTAs shared: sum their parts in order.  Rows that see nothing get zeros here.  A chain of
// latencies (unit_info, then everything else at once): a warp has its parts' rows in registers before it knows their factors.
// PJ_THREADS: 64 where units have few parts (sixteen at once), 256 for the units of few long sequences.
constexpr int PJ_DEEP = 8;
template <typename QT, int HD, int PJ_THREADS> __global__ void __launch_bounds__(PJ_THREADS) attn_join_kernel(const __grid_constant__ AttnArgs p) {
    constexpr int PJ_WARPS = PJ_THREADS / 32;
    constexpr int MLS = (PA_MAX_CTAS + PJ_THREADS - 1) / PJ_THREADS, PER = 128 / HD;  // PER: parts a warp reads side by side, HD / 4 lanes each
    __shared__ float factor[PA_MAX_CTAS], red[32];
    __shared__ float4 acc[PJ_WARPS][HD / 4];
    const int b = blockIdx.x / p.blocks / p.c.kv_heads, kvh = blockIdx.x / p.blocks % p.c.kv_heads, block = blockIdx.x % p.blocks, r = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const SeqWork w = seq_work(p, b);
    const int rho = block * p.ru + r, j = rho / p.group, head = kvh * p.group + rho % p.group;
    const size_t row_head = (size_t)(w.s.r0 + j) * p.heads + head;
    pdl_wait();  // (ahead of every return: a grid that ends early would let the next one start before the kernel ahead has ended)
    if (p.scores) pdl_launch_dependents();
    if (rho >= w.s.n * p.group) return;
    if (w.tiles == 0) {
        for (int col = tid; col < HD; col += PJ_THREADS) store_out<QT>(p, row_head, HD, col, 0.f, 0.f);
        if (tid == 0) store_lse(p, row_head, 0.f, 0.f);
        return;
    }
    const int2 info = __ldcg(p.unit_info + blockIdx.x);
    const int n = info.y;
    if (n <= 1) return;
    const size_t slot0 = (size_t)blockIdx.x + info.x;
    float2 ml[MLS];
#pragma unroll
    for (int i = 0; i < MLS; ++i) ml[i] = tid + i * PJ_THREADS < n ? __ldcg(p.part_ml + (slot0 + tid + i * PJ_THREADS) * p.ru + r) : make_float2(-INFINITY, 0.f);
    const int c4 = lane % (HD / 4), first = warp * PER + lane / (HD / 4);
    const float4* rows = reinterpret_cast<const float4*>(p.part_o + (slot0 * p.ru + r) * HD) + c4;
    const size_t step = (size_t)p.ru * HD / 4;
    float4 x[PJ_DEEP];
#pragma unroll
    for (int d = 0; d < PJ_DEEP; ++d) {
        const int i = first + d * PJ_WARPS * PER;
        x[d] = i < n ? __ldcg(rows + i * step) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float m = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < MLS; ++i) {
        m = fmaxf(m, ml[i].x);
        nan |= ml[i].x != ml[i].x;
    }
    m = block_max(m, red);
    if (__syncthreads_or(nan)) m = NAN;
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < MLS; ++i) {
        const float f = exp2f(ml[i].x - (m == -INFINITY ? 0.f : m));
        if (tid + i * PJ_THREADS < n) factor[tid + i * PJ_THREADS] = f;
        l += ml[i].y * f;
    }
    l = block_sum(l, red);  // (its barriers: factor is complete)
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& v, float f) {
        a.x = fmaf(v.x, f, a.x); a.y = fmaf(v.y, f, a.y); a.z = fmaf(v.z, f, a.z); a.w = fmaf(v.w, f, a.w);
    };
#pragma unroll
    for (int d = 0; d < PJ_DEEP; ++d) {
        const int i = first + d * PJ_WARPS * PER;
        if (i < n) add(x[d], factor[i]);
    }
    for (int i = first + PJ_DEEP * PJ_WARPS * PER; i < n; i += PJ_WARPS * PER) add(__ldcg(rows + i * step), factor[i]);
    if (PER == 2) {
        a.x += __shfl_xor_sync(0xffffffffu, a.x, 16); a.y += __shfl_xor_sync(0xffffffffu, a.y, 16);
        a.z += __shfl_xor_sync(0xffffffffu, a.z, 16); a.w += __shfl_xor_sync(0xffffffffu, a.w, 16);
    }
    if (lane < HD / 4) acc[warp][c4] = a;
    __syncthreads();
    for (int col = tid; col < HD; col += PJ_THREADS) {
        float o = 0.f;
        for (int i = 0; i < PJ_WARPS; ++i) o += reinterpret_cast<const float*>(acc[i])[col];
        store_out<QT>(p, row_head, HD, col, o, l);
    }
    if (tid == 0) store_lse(p, row_head, m, l);
}

// weight[entry] += sum over the kv head's rows of 2^(score - lse): one thread per entry, rows in order
constexpr int PA_COLLECT = 512;
__global__ void __launch_bounds__(PA_THREADS) attn_collect_kernel(const __grid_constant__ AttnArgs p) {
    const int b = blockIdx.z, kvh = blockIdx.y;
    const SeqWork w = seq_work(p, b);
    const int first = blockIdx.x * PA_COLLECT, end = min(w.s.len, first + PA_COLLECT);
    pdl_wait();
    if (w.s.n == 0 || end <= max(first, w.start)) return;
    float sum[PA_COLLECT / PA_THREADS];
#pragma unroll
    for (int i = 0; i < PA_COLLECT / PA_THREADS; ++i) sum[i] = 0.f;
    for (int j = 0; j < w.s.n; ++j)
        for (int g = 0; g < p.group; ++g) {
            const size_t row_head = (size_t)(w.s.r0 + j) * p.heads + kvh * p.group + g;
            const float lse2 = __ldcg(p.lse2 + row_head);
            if (lse2 == -INFINITY) continue;
            const float* s = p.scores + row_head * p.score_stride;
#pragma unroll
            for (int i = 0; i < PA_COLLECT / PA_THREADS; ++i) {
                const int t = first + i * PA_THREADS + threadIdx.x;
                if (t >= w.start && t < end) sum[i] += exp2f(__ldcg(s + t) - lse2);
            }
        }
    float* weight = p.c.weight + ((size_t)b * p.c.kv_heads + kvh) * p.c.cap;
#pragma unroll
    for (int i = 0; i < PA_COLLECT / PA_THREADS; ++i) {
        const int t = first + i * PA_THREADS + threadIdx.x;
        if (t >= w.start && t < end) weight[t] += sum[i];
    }
}

}  // namespace cd
