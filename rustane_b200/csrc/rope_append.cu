// cd_rope_append: rotary positions of a batch's new rows, K and V into their pages, in one pass over q, k and v.
//
// A CTA has one row (or a part of its heads, where there are few rows): it asks for its first elements, finds the row's sequence and entry
// meanwhile, puts the row's cosines and sines into shared memory once for all heads, and moves eight elements a thread at a time,
// two such items under way: every element is read once and written once.  Bound by those bytes on a long prompt (8184 rows of 64
// heads, 469 MB, 74 us: 6.3 TB/s, 98 % of the copy rate; 99 us with one item at a time), by the launch and the chain of row_start,
// lens, page table and store on a token (four tokens 4.1 us).
//
// Angles: position * turns modulo 2^64 is the exact fraction of a turn; its upper half, brought into an eighth of a turn either
// way, is exact in 30 bits and rounds once to fp32 (off by at most 2^-24 of the reduced angle), at any position.
#include <algorithm>
#include <cmath>

#include "serve.cuh"

using namespace cd;

namespace {
const char* CALL = "cd_rope_append";
constexpr int RA_THREADS = 256;

struct AppendArgs {
    PagedView c;
    const int *row_start, *positions;
    const void *q, *k, *v;
    void* q_out;
    long long q_stride, k_stride, v_stride;
    const uint64_t* turns;
    float magnitude;
    int rot, heads, nrows, parts;  // parts: CTAs a row is cut into
};

__device__ inline float2 cos_sin(uint64_t turns, int position, float magnitude) {
    const uint32_t t = (uint32_t)((uint64_t)(int64_t)position * turns >> 32);  // of a turn, 2^32
    const uint32_t n = (t + (1u << 29)) >> 30;                                   // the nearest quarter
    float s, c;
    sincospif((float)(int32_t)(t - (n << 30)) * 4.656612873077392578125e-10f, &s, &c);  // 2^-31: half turns
    if (n & 1) { const float x = c; c = -s; s = x; }
    if (n & 2) { c = -c; s = -s; }
    return make_float2(c * magnitude, s * magnitude);
}

// E elements; 16-byte accesses where they fill some
template <typename T, int E> __device__ inline void load(const T* p, float (&x)[E]) {
    if constexpr (E * sizeof(T) % 16 == 0) {
#pragma unroll
        for (int i = 0; i < (int)(E * sizeof(T) / 16); ++i) {
            const uint4 w = *(reinterpret_cast<const uint4*>(p) + i);
#pragma unroll
            for (int e = 0; e < (int)(16 / sizeof(T)); ++e) x[i * (16 / sizeof(T)) + e] = as_float(reinterpret_cast<const T*>(&w)[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = as_float(p[e]);
    }
}
template <typename T, int E> __device__ inline void store(T* p, const float (&x)[E]) {
    if constexpr (E * sizeof(T) % 16 == 0) {
#pragma unroll
        for (int i = 0; i < (int)(E * sizeof(T) / 16); ++i) {
            uint4 w;
#pragma unroll
            for (int e = 0; e < (int)(16 / sizeof(T)); ++e) reinterpret_cast<T*>(&w)[e] = from_float<T>(x[i * (16 / sizeof(T)) + e]);
            *(reinterpret_cast<uint4*>(p) + i) = w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) p[e] = from_float<T>(x[e]);
    }
}

// One item: E elements of a rotated head and, in halves, their partners; or E elements that pass.  Loaded and stored apart, so that a thread
// has the loads of several items under way.
template <bool HALF, int E> struct Item {
    float a[E], b[E];
    int at = 0;
    bool turns = false;
    template <typename TI> __device__ inline void get(const TI* in, int item, int rot) {
        const int turned = HALF ? rot / 2 / E : rot / E;
        turns = item < turned;
        at = turns ? item * E : rot + (item - turned) * E;
        load<TI, E>(in + at, a);
        if (HALF && turns) load<TI, E>(in + rot / 2 + at, b);
    }
    template <typename TO> __device__ inline void put(TO* out, int rot, const float2* cs) {
        if (turns) {
            if constexpr (HALF) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float2 t = cs[at + e];
                    const float x = a[e], y = b[e];
                    a[e] = x * t.x - y * t.y;
                    b[e] = x * t.y + y * t.x;
                }
                store<TO, E>(out + rot / 2 + at, b);
            } else {
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const float2 t = cs[(at + e) / 2];
                    const float x = a[e], y = a[e + 1];
                    a[e] = x * t.x - y * t.y;
                    a[e + 1] = x * t.y + y * t.x;
                }
            }
        }
        store<TO, E>(out + at, a);
    }
};

template <typename QT, typename KT, int HD, bool HALF, int E> __global__ void __launch_bounds__(RA_THREADS) rope_append_kernel(const __grid_constant__ AppendArgs p) {
    __shared__ float2 cs[HD / 2];
    __shared__ int found, s_entry[2];
    const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts, tid = threadIdx.x;
    if (tid == 0) found = 0x7fffffff;
    const int position = p.positions[row];
    const int per = HALF ? p.rot / 2 / E + (HD - p.rot) / E : HD / E;  // items of a rotated head
    const int rotated = (p.heads + p.c.kv_heads) * per, all = rotated + p.c.kv_heads * (HD / E);
    const QT *q = static_cast<const QT*>(p.q) + row * p.q_stride, *k = static_cast<const QT*>(p.k) + row * p.k_stride, *v = static_cast<const QT*>(p.v) + row * p.v_stride;
    QT* q_out = static_cast<QT*>(p.q_out) + (size_t)row * p.heads * HD;
    KT* pool = static_cast<KT*>(p.c.pool);
    // the first items are asked for before anything else is known of the row
    constexpr int DEEP = 2;
    Item<HALF, E> x[DEEP];
    int vec[DEEP];  // q heads, k heads, v heads; -1: nothing
    auto fetch = [&](int i0) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const int i = i0 + d * p.parts * RA_THREADS;
            vec[d] = -1;
            if (i < rotated) {
                vec[d] = i / per;
                const QT* src = vec[d] < p.heads ? q + (size_t)vec[d] * HD : k + (size_t)(vec[d] - p.heads) * HD;
                x[d].get(src, i - vec[d] * per, p.rot);
            } else if (i < all) {
                const int h = (i - rotated) / (HD / E);
                vec[d] = p.heads + p.c.kv_heads + h;
                x[d].get(v + (size_t)h * HD, i - rotated - h * (HD / E), 0);
            }
        }
    };
    const int step = p.parts * RA_THREADS * DEEP;
    int i0 = part * RA_THREADS + tid;
    fetch(i0);
    if (tid < p.rot / 2) cs[tid] = cos_sin(p.turns[tid], position, p.magnitude);
    __syncthreads();
    // the row's sequence (the first that claims it), its entry and page: by the thread that finds it
    for (int b = tid; b < p.c.nseq; b += RA_THREADS) {
        const int r0 = p.row_start[b], r1 = p.row_start[b + 1];
        if (r0 <= row && row < r1) atomicMin(&found, b);
    }
    __syncthreads();
    const int b = found;
    if (b == 0x7fffffff) return;
    if (tid == b % RA_THREADS) {
        const BatchSeq s = batch_seq(p.c, p.row_start, b, p.nrows, p.nrows);
        const int at = s.len - s.n + row - s.r0;
        if (s.n > 0 && at < 0) report(p.c.status, CD_STATUS_BATCH);
        s_entry[0] = s.n > 0 ? max(at, -1) : -2;
        s_entry[1] = s.n > 0 && at >= 0 ? page_at(p.c, b, at) : -1;
    }
    __syncthreads();
    const int entry = s_entry[0], page = s_entry[1];
    if (entry == -2) return;  // the sequence is left out
    while (true) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const int h = vec[d] - p.heads;
            if (vec[d] >= 0 && h < 0) x[d].put(q_out + (size_t)vec[d] * HD, p.rot, cs);
            else if (vec[d] >= 0 && page >= 0) {
                const bool is_v = h >= p.c.kv_heads;
                x[d].put(pool + row_at(p.c, page, is_v, is_v ? h - p.c.kv_heads : h, entry, HD), is_v ? 0 : p.rot, cs);
            }
        }
        i0 += step;
        if (i0 >= all) break;
        fetch(i0);
    }
    if (p.c.weight && entry >= 0 && part == 0)
        for (int h = tid; h < p.c.kv_heads; h += RA_THREADS) {
            const size_t at = ((size_t)b * p.c.kv_heads + h) * p.c.cap + entry;
            p.c.weight[at] = 0.f;
            p.c.position[at] = position;
        }
}

template <typename QT, typename KT, int HD> cudaError_t launch(const AppendArgs& a, bool half, cudaStream_t s) {
    const unsigned grid = (unsigned)a.nrows * a.parts;
    const bool wide = (half ? a.rot / 2 : a.rot) % 8 == 0;
    if (half) {
        if (wide) rope_append_kernel<QT, KT, HD, true, 8><<<grid, RA_THREADS, 0, s>>>(a);
        else rope_append_kernel<QT, KT, HD, true, 1><<<grid, RA_THREADS, 0, s>>>(a);
    } else {
        if (wide) rope_append_kernel<QT, KT, HD, false, 8><<<grid, RA_THREADS, 0, s>>>(a);
        else rope_append_kernel<QT, KT, HD, false, 2><<<grid, RA_THREADS, 0, s>>>(a);
    }
    return cudaGetLastError();
}
template <typename QT, typename KT> cudaError_t launch_hd(int hd, const AppendArgs& a, bool half, cudaStream_t s) {
    return hd == 128 ? launch<QT, KT, 128>(a, half, s) : launch<QT, KT, 64>(a, half, s);
}
}  // namespace

extern "C" int cd_rope_frequencies(int rot_dim, double base, int scaling, double factor, int original, uint64_t* turns, float* magnitude) {
    const char* call = "cd_rope_frequencies";
    if (!turns || !magnitude) return refuse(CD_ERR_INVALID, call, "null argument");
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > 65536) return refuse(CD_ERR_INVALID, call, "rot_dim must be even, 2..65536");
    if (!(base >= 1.0) || !std::isfinite(base)) return refuse(CD_ERR_INVALID, call, "base must be at least 1");
    if (scaling < CD_ROPE_PLAIN || scaling > CD_ROPE_YARN) return refuse(CD_ERR_INVALID, call, "unknown scaling");
    if (!(factor >= 1.0) || !std::isfinite(factor)) return refuse(CD_ERR_INVALID, call, "factor must be at least 1");
    if (scaling == CD_ROPE_YARN && (original < 1 || base <= 1.0)) return refuse(CD_ERR_INVALID, call, "yarn needs the original number of positions and a base above 1");
    const double two_pi = 6.283185307179586476925286766559;
    if (scaling == CD_ROPE_NTK && rot_dim > 2) base *= std::pow(factor, (double)rot_dim / (rot_dim - 2));
    double low = 0.0, high = 0.0;
    *magnitude = 1.0f;
    if (scaling == CD_ROPE_YARN) {
        auto pair = [&](double t) { return rot_dim * std::log(original / (t * two_pi)) / (2.0 * std::log(base)); };
        low = std::max(std::floor(pair(32.0)), 0.0);
        high = std::min(std::ceil(pair(1.0)), (double)rot_dim - 1);
        *magnitude = (float)(0.1 * std::log(factor) + 1.0);
    }
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (scaling == CD_ROPE_LINEAR) f /= factor;
        if (scaling == CD_ROPE_YARN) {
            const double ramp = std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 0.001)));
            f = f / factor * ramp + f * (1.0 - ramp);
        }
        turns[i] = (uint64_t)std::llround(f / two_pi * 9223372036854775808.0) * 2;  // f <= 1: below 2^62
    }
    return CD_OK;
}

extern "C" int cd_rope_append(const cd_paged_cache* c, const cd_rope* rope, int dtype, int heads, int nrows, const void* q, int64_t q_stride, const void* k,
                              int64_t k_stride, const void* v, int64_t v_stride, const int32_t* positions, const int32_t* row_start, void* q_out,
                              void* stream) {
    if (int rc = check_cache(c, CALL)) return rc;
    if (!rope || !rope->turns) return refuse(CD_ERR_INVALID, CALL, "null rope");
    if (rope->rot_dim < 2 || rope->rot_dim % 2 || rope->rot_dim > c->hd) return refuse(CD_ERR_INVALID, CALL, "rot_dim must be even and in 2..hd");
    if (rope->layout != CD_ROPE_INTERLEAVED && rope->layout != CD_ROPE_HALF) return refuse(CD_ERR_INVALID, CALL, "unknown rope layout");
    if (!std::isfinite(rope->magnitude)) return refuse(CD_ERR_INVALID, CALL, "magnitude must be finite");
    if (dtype != CD_DTYPE_F32 && dtype != c->dtype) return refuse(CD_ERR_INVALID, CALL, "q, k and v are f32 or of the pool's type");
    if (heads <= 0 || heads > 65536) return refuse(CD_ERR_INVALID, CALL, "heads must be in 1..65536");
    if (nrows < 0 || nrows > 1 << 22) return refuse(CD_ERR_INVALID, CALL, "nrows must be in 0..4194304");
    if (nrows == 0 || c->nseq == 0) return CD_OK;
    const int64_t qp = (int64_t)heads * c->hd, kp = (int64_t)c->kv_heads * c->hd;
    if (q_stride == 0) q_stride = qp;
    if (k_stride == 0) k_stride = kp;
    if (v_stride == 0) v_stride = kp;
    if (int rc = check_rows(q, q_stride, qp, dtype, CALL)) return rc;
    if (int rc = check_rows(k, k_stride, kp, dtype, CALL)) return rc;
    if (int rc = check_rows(v, v_stride, kp, dtype, CALL)) return rc;
    if (int rc = check_rows(q_out, qp, qp, dtype, CALL)) return rc;
    if (q_out == q && q_stride != qp) return refuse(CD_ERR_INVALID, CALL, "q_out may be q only where q is packed");
    if (!positions || !row_start) return refuse(CD_ERR_INVALID, CALL, "null argument");
    if (!aligned(positions, 4) || !aligned(row_start, 4) || !aligned(rope->turns, 8))
        return refuse(CD_ERR_INVALID, CALL, "positions and row_start start on 4-byte boundaries, turns on an 8-byte one");
    AppendArgs a;
    a.c = view_of(c);
    a.row_start = row_start;
    a.positions = positions;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.turns = rope->turns;
    a.magnitude = rope->magnitude;
    a.rot = rope->rot_dim;
    a.heads = heads;
    a.nrows = nrows;
    // few rows: a CTA for every pass over its items, so that no load waits behind another
    const int passes = (int)std::min<long long>(64, ((long long)(heads + 2 * c->kv_heads) * c->hd / 8 + RA_THREADS - 1) / RA_THREADS);
    a.parts = nrows >= 1024 ? 1 : std::max(1, std::min(passes, 1024 / nrows));
    DeviceGuard guard(c->device);
    if (guard.err != cudaSuccess) return cuda_status(guard.err, CALL);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool half = rope->layout == CD_ROPE_HALF;
    cudaError_t e;
    if (c->dtype == CD_DTYPE_F32) e = launch_hd<float, float>(c->hd, a, half, s);
    else if (c->dtype == CD_DTYPE_F16) e = dtype == CD_DTYPE_F32 ? launch_hd<float, __half>(c->hd, a, half, s) : launch_hd<__half, __half>(c->hd, a, half, s);
    else e = dtype == CD_DTYPE_F32 ? launch_hd<float, __nv_bfloat16>(c->hd, a, half, s) : launch_hd<__nv_bfloat16, __nv_bfloat16>(c->hd, a, half, s);
    return cuda_status(e, CALL);
}
