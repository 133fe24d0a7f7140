// cd_verify_drafts: which drafted tokens of a batch stay, and the token drawn behind them.
//
// verify_rows_kernel reads every logit row once: a CTA leaves (max, sum of exp, arg-max) of a chunk of a row.  Bound by its instructions
// and exponentials (0.6 instructions a cycle and scheduler; 254 rows of 128000 bf16 logits, 65 MB, 19 us).  verify_pick_kernel, a cluster
// of CTAs per sequence, puts the chunks together, tests the drafts, and draws from the one row (pair of rows) it ended at, which it reads
// again.  Bound by the 64-bit exponentials, four a token (44 us for 32 sequences; 92 us with exp() and every logit asked for when it
// was needed), on one sequence by five barriers of the cluster and the loads between them (11 us).
//
// What is decided there are comparisons with given random numbers, so sums must not blur them.  The test u q(x) < p(x) goes by row sums of
// fp32 terms (16-byte loads' worth at a time, then over a thread's loads, in fp32; over threads in 64 bits), and where u q(x) is nearer to p(x)
// than those can tell (VerifyArgs::near, some 3e-5 of it) by sums in 64 bits over both rows, a few microseconds in one call out of a hundred.
// The draw, where every one of `vocab` running sums is a border, is in 64 bits throughout, its row sums included.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <utility>

#include "serve.cuh"

namespace cg = cooperative_groups;
using namespace cd;

namespace {
const char* CALL = "cd_verify_drafts";
constexpr int VD_THREADS = 256, VD_WARPS = VD_THREADS / 32, VD_PICK_THREADS = 512, VD_PICK_WARPS = VD_PICK_THREADS / 32, VD_CHUNKS = 32, VD_CLUSTER = 8, VD_TILE = 256, VD_KEEP = 16, VD_VOCAB = 1 << 22;

struct Part {
    float m;   // NaN: the chunk holds NaN
    int at;    // lowest place of m
    double s;  // sum of exp((x - m) / temperature)
};
struct VerifyArgs {
    const void *target, *draft;
    long long target_stride, draft_stride;
    const int *tokens, *row_start;
    const float *uniforms, *draws;
    int *accepted, *out, *status;
    Part* parts;  // [2 nrows][VD_CHUNKS]: target rows, then draft rows
    double inv_t, near;  // near: what the row pass's sums may be off by, of themselves, p's and q's together
    int nseq, nrows, max_rows, vocab, chunks, chunk;  // chunk: elements, a multiple of 8
};

// e^x in 64 bits for x <= 0 (or a little above): e^x = 2^(n / 256) e^r with |r| <= ln 2 / 512, e^r by its series up to r^4 / 24 (the next
// term is below 4e-17), 2^(j / 256) from a table.  Off by some 1e-16, and by x times 1e-16.  What the draw costs is the 64-bit pipe:
// eight operations here against about twice that in exp().
constexpr int EXP_TABLE = 256;
__device__ inline double exp_neg(double x, const double* two_to) {
    constexpr double ROUND = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is the integer
    const double t = fma(x, 369.32993046757462, ROUND);  // 256 / ln 2
    const int n = __double2loint(t);
    const double r = fma(t - ROUND, -0.0027076061740622863, x);  // ln 2 / 256
    double e = fma(r, 1.0 / 24.0, 1.0 / 6.0);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    const double y = e * two_to[n & (EXP_TABLE - 1)];
    const double v = __hiloint2double(__double2hiint(y) + ((n >> 8) << 20), __double2loint(y));
    return x > -708.0 ? v : x != x ? x : 0.0;  // (no branch: a lane's terms go through the pipe together)
}
__device__ inline uint4 load_once(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ inline bool rows_fit(const VerifyArgs& p, int r0, int r1) { return r0 >= 0 && r1 >= r0 && r1 <= p.nrows && r1 - r0 <= p.max_rows; }

// (m, at, s) of one chunk.  GREEDY: no sums.
template <typename T, bool GREEDY> __global__ void __launch_bounds__(VD_THREADS) verify_rows_kernel(const __grid_constant__ VerifyArgs p) {
    constexpr int VEC = 16 / sizeof(T), DEEP = 4;
    __shared__ float red_m[VD_WARPS];
    __shared__ int red_at[VD_WARPS];
    __shared__ double red_s[VD_WARPS];
    const int row = blockIdx.x / p.chunks, ch = blockIdx.x % p.chunks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool is_draft = row >= p.nrows;
    const int r = is_draft ? row - p.nrows : row;
    const T* x = is_draft ? static_cast<const T*>(p.draft) + r * p.draft_stride : static_cast<const T*>(p.target) + r * p.target_stride;
    const int head = (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T);  // elements before the first 16-byte boundary
    const int e0 = ch == 0 ? 0 : min(p.vocab, head + ch * p.chunk), e1 = ch == p.chunks - 1 ? p.vocab : min(p.vocab, head + (ch + 1) * p.chunk);
    const int v0 = min(e1, max(e0, head)), vecs = (e1 - v0) / VEC;
    const uint4* body = reinterpret_cast<const uint4*>(x + v0);
    uint4 w[DEEP];
    auto fetch = [&](int i) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
            if (i + d * VD_THREADS < vecs) w[d] = load_once(body + i + d * VD_THREADS);
    };
    // target rows are all there and asked for at once; a draft row only if a draft is behind it, as there need not be memory for others
    if (!is_draft) fetch(tid);
    bool used = false;
    for (int b = tid; b < p.nseq; b += VD_THREADS) {
        const int r0 = p.row_start[b], r1 = p.row_start[b + 1];
        used |= r0 <= r && r + is_draft < r1 && rows_fit(p, r0, r1);
    }
    if (!__syncthreads_or(used)) {
        if (!is_draft && ch == 0 && tid == 0 && r < p.row_start[p.nseq]) p.out[r] = -1;  // a row that no sequence took
        return;
    }
    if (is_draft) fetch(tid);
    const float scale = (float)(p.inv_t * 1.4426950408889634074);
    float m = -INFINITY, s = 0.f;
    int at = 0x7fffffff;
    bool nan = false;
    auto one = [&](int i) {  // a ragged end
        const float v = as_float(x[i]);
        if (GREEDY) {
            nan |= v != v;
            if (v > m || (v == m && i < at)) { m = v; at = i; }
        } else {
            if (v > m) {
                s *= ex2(m == -INFINITY ? 0.f : (m - v) * scale);
                m = v;
            }
            s += ex2((v - (m == -INFINITY ? 0.f : m)) * scale);
        }
    };
    for (int i = e0 + tid; i < v0; i += VD_THREADS) one(i);
    for (int i = tid; i < vecs; i += VD_THREADS * DEEP) {
        float v[DEEP][VEC];
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[d][e] = as_float(reinterpret_cast<const T*>(&w[d])[e]);
        if (i + (DEEP - 1) * VD_THREADS >= vecs)
#pragma unroll
            for (int d = 0; d < DEEP; ++d)
                if (i + d * VD_THREADS >= vecs)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) v[d][e] = -INFINITY;
        if (i + VD_THREADS * DEEP < vecs) fetch(i + VD_THREADS * DEEP);
        if (GREEDY) {
#pragma unroll
            for (int d = 0; d < DEEP; ++d)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    nan |= v[d][e] != v[d][e];
                    if (v[d][e] > m) { m = v[d][e]; at = v0 + (i + d * VD_THREADS) * VEC + e; }
                }
        } else {
            float top = m;
#pragma unroll
            for (int d = 0; d < DEEP; ++d)
#pragma unroll
                for (int e = 0; e < VEC; ++e) top = fmaxf(top, v[d][e]);
            if (top > m) {
                s *= ex2(m == -INFINITY ? 0.f : (m - top) * scale);
                m = top;
            }
            const float base = (m == -INFINITY ? 0.f : m);
            float some = 0.f;
#pragma unroll
            for (int d = 0; d < DEEP; ++d)
#pragma unroll
                for (int e = 0; e < VEC; ++e) some += ex2((v[d][e] - base) * scale);
            s += some;
        }
    }
    for (int i = v0 + vecs * VEC + tid; i < e1; i += VD_THREADS) one(i);

    if (GREEDY) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float om = __shfl_xor_sync(0xffffffffu, m, o);
            const int oa = __shfl_xor_sync(0xffffffffu, at, o);
            if (om > m || (om == m && oa < at)) { m = om; at = oa; }
        }
        if (lane == 0) { red_m[warp] = m; red_at[warp] = at; }
        nan = __syncthreads_or(nan);
        if (tid == 0) {
            for (int i = 1; i < VD_WARPS; ++i)
                if (red_m[i] > m || (red_m[i] == m && red_at[i] < at)) { m = red_m[i]; at = red_at[i]; }
            p.parts[(size_t)row * VD_CHUNKS + ch] = Part{nan ? NAN : m, at, 0.0};
        }
    } else {
        const float top = warp_max(m);
        double sum = (double)s * (double)ex2((m - (top == -INFINITY ? 0.f : top)) * scale);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) { red_m[warp] = top; red_s[warp] = sum; }
        __syncthreads();
        if (tid == 0) {
            float all = red_m[0];
            for (int i = 1; i < VD_WARPS; ++i) all = fmaxf(all, red_m[i]);
            sum = 0.0;
            for (int i = 0; i < VD_WARPS; ++i) sum += red_s[i] * (double)ex2((red_m[i] - (all == -INFINITY ? 0.f : all)) * scale);
            p.parts[(size_t)row * VD_CHUNKS + ch] = Part{all, 0, sum};
        }
    }
}

__device__ inline double warp_sum_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct RowStat {
    float m;
    int at;
    double z;
    __device__ bool good() const { return isfinite(m) && isfinite(z); }
};
__device__ inline Part load_part(const VerifyArgs& p, int row) {  // this lane's chunk of a row
    const int lane = threadIdx.x & 31;
    Part q{-INFINITY, 0x7fffffff, 0.0};
    if (lane < p.chunks) {
        const Part* src = p.parts + (size_t)row * VD_CHUNKS + lane;
        q.m = __ldcg(&src->m);
        q.at = __ldcg(&src->at);
        q.s = __ldcg(&src->s);
    }
    return q;
}
// a row's chunks together (all lanes of a warp)
template <bool GREEDY> __device__ inline RowStat row_stat(const VerifyArgs& p, const Part& q, const double* two_to) {
    RowStat r;
    if (GREEDY) {
        const bool nan = __any_sync(0xffffffffu, q.m != q.m);
        float m = q.m;
        int at = q.at;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float om = __shfl_xor_sync(0xffffffffu, m, o);
            const int oa = __shfl_xor_sync(0xffffffffu, at, o);
            if (om > m || (om == m && oa < at)) { m = om; at = oa; }
        }
        r.m = nan ? NAN : m;
        r.at = at;
        r.z = 1.0;
    } else {
        r.m = warp_max(q.m);
        r.at = 0;
        r.z = warp_sum_d(isfinite(r.m) ? q.s * exp_neg(((double)q.m - (double)r.m) * p.inv_t, two_to) : NAN);
    }
    return r;
}

struct PickShared {
    int first_bad, first_near, stays, valid, at;  // of a sequence's drafts: the first turned down, the first that the row pass's sums cannot decide
    double total[3];  // of this CTA: p's sum, q's sum, what is drawn from
    double red[2][VD_PICK_WARPS];
    float pm, qm;
    RowStat rows[2][VD_KEEP];  // of the sequence's first rows, target and draft, as the tests found them
};

// Whether the draft behind `row` stays, by sums in 64 bits (all threads of a CTA; the same in every CTA of a cluster).
template <typename T> __device__ __noinline__ bool stays_by_64_bits(const VerifyArgs& p, int row, PickShared& sh, const double* two_to) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, x = p.tokens[row + 1];
    const T *target = static_cast<const T*>(p.target) + row * p.target_stride, *draft = p.draft ? static_cast<const T*>(p.draft) + row * p.draft_stride : nullptr;
    if (warp == 0) {
        const RowStat t = row_stat<false>(p, load_part(p, row), two_to);
        const RowStat q = draft ? row_stat<false>(p, load_part(p, p.nrows + row), two_to) : RowStat{0.f, 0, 1.0};
        if (lane == 0) {
            sh.pm = t.m;
            sh.qm = q.m;
        }
    }
    __syncthreads();
    const double pm = sh.pm, qm = sh.qm;
    double sp = 0.0, sq = 0.0;
    for (int i = tid; i < p.vocab; i += VD_PICK_THREADS) {
        sp += exp_neg(((double)as_float(target[i]) - pm) * p.inv_t, two_to);
        if (draft) sq += exp_neg(((double)as_float(draft[i]) - qm) * p.inv_t, two_to);
    }
    sp = warp_sum_d(sp);
    sq = warp_sum_d(sq);
    if (lane == 0) { sh.red[0][warp] = sp; sh.red[1][warp] = sq; }
    __syncthreads();
    if (tid == 0) {
        sp = sq = 0.0;
        for (int i = 0; i < VD_PICK_WARPS; ++i) {
            sp += sh.red[0][i];
            sq += sh.red[1][i];
        }
        const double px = exp_neg(((double)as_float(target[x]) - pm) * p.inv_t, two_to) / sp;
        const double qx = draft ? exp_neg(((double)as_float(draft[x]) - qm) * p.inv_t, two_to) / sq : 1.0;
        sh.stays = (double)p.uniforms[row] * qx < px;
    }
    __syncthreads();
    return sh.stays;
}

template <typename T, bool GREEDY> __global__ void __launch_bounds__(VD_PICK_THREADS, 2) verify_pick_kernel(const __grid_constant__ VerifyArgs p) {
    extern __shared__ double tiles[];  // sums of this CTA's tiles
    __shared__ PickShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), b = blockIdx.x / size;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r0 = p.row_start[b], r1 = p.row_start[b + 1], n = (int)((unsigned)r1 - (unsigned)r0);  // (looked at where the rows fit)
    pdl_wait();
    const bool fits = rows_fit(p, r0, r1);
    if (!fits || n == 0) {
        if (rank == 0 && tid == 0) {
            p.accepted[b] = fits ? 0 : -1;
            if (!fits) report(p.status, CD_STATUS_BATCH);
        }
        return;
    }
    __shared__ double two_to[EXP_TABLE];
    if (!GREEDY && tid < EXP_TABLE) two_to[tid] = exp2((double)tid / EXP_TABLE);
    if (tid == 0) {
        sh.first_bad = sh.first_near = n - 1;
        sh.valid = 1;
    }
    __syncthreads();
    const T *target = static_cast<const T*>(p.target), *draft = static_cast<const T*>(p.draft);
    for (int from = 0;;) {
        for (int j = from + warp; j < n - 1; j += VD_PICK_WARPS) {  // (every load that does not hang on another is asked for at once)
            const int x = p.tokens[r0 + j + 1];
            const Part tp = load_part(p, r0 + j), qp = draft ? load_part(p, p.nrows + r0 + j) : Part{};
            const float u = GREEDY ? 0.f : p.uniforms[r0 + j];
            const bool in = (unsigned)x < (unsigned)p.vocab;
            const float tx = in && !GREEDY ? as_float(target[(r0 + j) * p.target_stride + x]) : 0.f, qx_logit = in && draft ? as_float(draft[(r0 + j) * p.draft_stride + x]) : 0.f;
            const RowStat t = row_stat<GREEDY>(p, tp, two_to);
            if (lane == 0 && j < VD_KEEP) sh.rows[0][j] = t;
            bool stays = t.good() && in;
            if (GREEDY) stays = stays && t.at == x;
            else {
                const double px = exp_neg(((double)tx - (double)t.m) * p.inv_t, two_to) / t.z;
                double qx = 1.0;
                if (draft) {
                    const RowStat q = row_stat<GREEDY>(p, qp, two_to);
                    if (lane == 0 && j < VD_KEEP) sh.rows[1][j] = q;
                    qx = q.good() ? exp_neg(((double)qx_logit - (double)q.m) * p.inv_t, two_to) / q.z : NAN;
                }
                const double uq = (double)u * qx;
                // (above 0 on both sides: 0 < 0 and NaN are decided)
                if (stays && uq > 0.0 && fabs(uq - px) <= p.near * px && lane == 0) atomicMin(&sh.first_near, j);
                stays = stays && uq < px;
            }
            if (!stays && lane == 0) atomicMin(&sh.first_bad, j);
        }
        __syncthreads();
        if (GREEDY) break;
        // A draft turned down by fp32 sums alone is one of the near ones.  The first of them goes first: what is behind a refused one does not count.
        const int near = sh.first_near;
        if (near > sh.first_bad || near == n - 1) break;
        const bool stays = stays_by_64_bits<T>(p, r0 + near, sh, two_to);
        if (!stays || near + 1 >= n - 1) {
            __syncthreads();
            if (tid == 0) sh.first_bad = stays ? n - 1 : near;
            __syncthreads();
            break;
        }
        __syncthreads();
        if (tid == 0) sh.first_bad = sh.first_near = n - 1;
        __syncthreads();
        from = near + 1;
    }
    const int end = sh.first_bad, row = r0 + end;
    const bool left = end < n - 1;  // a draft was turned down: draw from what p has over q
    if (warp == 0) {
        RowStat t, q;
        if (left && end < VD_KEEP) {
            t = sh.rows[0][end];
            if (draft) q = sh.rows[1][end];
        } else {
            const Part tp = load_part(p, row), qp = left && draft ? load_part(p, p.nrows + row) : Part{};
            t = row_stat<GREEDY>(p, tp, two_to);
            if (left && draft) q = row_stat<GREEDY>(p, qp, two_to);
        }
        if (lane == 0) {
            sh.pm = t.m;
            sh.at = t.at;
            sh.qm = left && draft ? q.m : 0.f;
            if (!t.good() || (!GREEDY && left && draft && !q.good())) sh.valid = 0;
        }
    }
    __syncthreads();
    if (rank == 0) {
        for (int j = tid; j < n; j += VD_PICK_THREADS)
            if (j != end) p.out[r0 + j] = j < end ? p.tokens[r0 + j + 1] : -1;
        if (tid == 0) p.accepted[b] = end;
    }
    if (!sh.valid || GREEDY) {  // the same in every CTA of the cluster
        if (rank == 0 && tid == 0) {
            p.out[row] = sh.valid ? sh.at : -1;
            if (!sh.valid) report(p.status, CD_STATUS_LOGITS);
        }
        return;
    }
    const T *pt = target + row * p.target_stride, *pd = left && draft ? draft + row * p.draft_stride : nullptr;
    const int gone = left && !draft ? p.tokens[row + 1] : -1;
    // e^((logit - largest) / temperature), the difference first: it is 0 for the largest whatever its size, where a rounded product of the
    // largest and 1 / temperature would leave what exceeds 64 bits of it
    const double pm = sh.pm, qm = sh.qm;
    double pb = 0.0, qb = 0.0;
    auto ep = [&](float x) { return exp_neg(fma((double)x - pm, p.inv_t, pb), two_to); };
    auto eq = [&](float x) { return exp_neg(fma((double)x - qm, p.inv_t, qb), two_to); };
    constexpr int PER = VD_TILE / 32;  // tokens of a tile a lane has
    auto logits = [&](const T* row_, int first, int step, float (&x)[PER]) {  // all of them asked for before one is used
#pragma unroll
        for (int e = 0; e < PER; ++e) x[e] = first + e * step < p.vocab ? as_float(row_[first + e * step]) : -INFINITY;
    };
    const int all_tiles = (p.vocab + VD_TILE - 1) / VD_TILE, per = (all_tiles + size - 1) / size;
    const int t0 = min(all_tiles, rank * per), t1 = min(all_tiles, t0 + per);
    if (pd) {
        double sp = 0.0, sq = 0.0;
        for (int t = t0 + warp; t < t1; t += VD_PICK_WARPS) {
            float a[PER], d[PER];
            logits(pt, t * VD_TILE + lane, 32, a);
            logits(pd, t * VD_TILE + lane, 32, d);
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                sp += ep(a[e]);
                sq += eq(d[e]);
            }
        }
        sp = warp_sum_d(sp);
        sq = warp_sum_d(sq);
        if (lane == 0) { sh.red[0][warp] = sp; sh.red[1][warp] = sq; }
        __syncthreads();
        if (tid < 2) {
            double v = 0.0;
            for (int i = 0; i < VD_PICK_WARPS; ++i) v += sh.red[tid][i];
            sh.total[tid] = v;
        }
        cluster.sync();
        sp = sq = 0.0;
#pragma unroll
        for (int r = 0; r < VD_CLUSTER; ++r) {
            const double* o = cluster.map_shared_rank(sh.total, r);
            sp += o[0];
            sq += o[1];
        }
        pb = -log(sp);  // from here on the terms are p and q themselves
        qb = -log(sq);
    }
    auto shares = [&](int first, int step, bool rest, double (&v)[PER]) {  // of a lane's tokens in what is drawn from
        float a[PER], d[PER];
        logits(pt, first, step, a);
        if (rest && pd) logits(pd, first, step, d);
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            v[e] = ep(a[e]);
            if (rest && pd) {
                v[e] -= eq(d[e]);
                if (__double2hiint(v[e]) < 0) v[e] = 0.0;  // (by its sign bit: no 64-bit comparison)
            }
            if (rest && first + e * step == gone) v[e] = 0.0;
        }
    };
    double whole = 0.0, before = 0.0, totals[VD_CLUSTER];
    bool rest = left;
    for (int turn = 0; turn < 2; ++turn) {  // again from p alone where nothing is left of p - q; p's largest has a share, so that `whole` is then above 0
        for (int t = t0 + warp; t < t1; t += VD_PICK_WARPS) {
            double x[PER], v = 0.0;
            shares(t * VD_TILE + lane, 32, rest, x);
#pragma unroll
            for (int e = 0; e < PER; ++e) v += x[e];
            v = warp_sum_d(v);
            if (lane == 0) tiles[t - t0] = v;
        }
        __syncthreads();
        if (warp == 0) {
            double v = 0.0;
            for (int t = lane; t < t1 - t0; t += 32) v += tiles[t];
            v = warp_sum_d(v);
            if (lane == 0) sh.total[2] = v;
        }
        cluster.sync();
        whole = before = 0.0;
#pragma unroll
        for (int r = 0; r < VD_CLUSTER; ++r) totals[r] = *cluster.map_shared_rank(&sh.total[2], r);
#pragma unroll
        for (int r = 0; r < VD_CLUSTER; ++r) {
            if (r < rank) before += totals[r];
            whole += totals[r];
        }
        if (whole > 0.0 || !rest) break;
        cluster.sync();  // (rounding left nothing: once in a lifetime)
        rest = false;
    }
    // the first token whose running sum exceeds u * whole: the CTA, then the tile, then the token.  Sums of sums round, so where none
    // does the last one that has a share is it.
    const double goal = (double)p.draws[b] * whole;
    double run = 0.0;
    int owner = -1;
    bool open = true;
#pragma unroll
    for (int r = 0; r < VD_CLUSTER; ++r) {
        if (open && totals[r] > 0.0) owner = r;
        run += totals[r];
        open = open && !(run > goal);
    }
    // others may still read this CTA's totals: it stays until all have them, but does not wait for that with its own work
    auto arrived = cluster.barrier_arrive();
    if (owner != rank || warp != 0) {
        cluster.barrier_wait(std::move(arrived));
        return;
    }
    // exclusive sums over the lanes' values in order; the first of them whose end exceeds the goal, or the last one with a share
    auto pick = [&](double v, double& before_it, double& all_) {
        double incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        const uint32_t over = __ballot_sync(0xffffffffu, v > 0.0 && run + incl > goal), some = __ballot_sync(0xffffffffu, v > 0.0);
        const int at = over ? __ffs(over) - 1 : some ? 31 - __clz(some) : -1;
        before_it = __shfl_sync(0xffffffffu, run + (incl - v), max(at, 0));
        all_ = __shfl_sync(0xffffffffu, incl, 31);
        return over ? at : at < 0 ? -64 : at - 32;  // below 0: none exceeds it
    };
    run = before;
    int tile = 0;
    double tile_run = before;
    for (int t = 0; t < t1 - t0; t += 32) {
        double from, all_;
        const int at = pick(t + lane < t1 - t0 ? tiles[t + lane] : 0.0, from, all_);
        if (at != -64) {
            tile = t + (at < 0 ? at + 32 : at);
            tile_run = from;
        }
        if (at >= 0) break;
        run += all_;
    }
    run = tile_run;
    const int first = (t0 + tile) * VD_TILE + lane * PER;  // eight tokens a lane, in order
    double v[PER], sum = 0.0, from, all_;
    shares(first, 1, rest, v);
#pragma unroll
    for (int e = 0; e < PER; ++e) sum += v[e];
    const int at = pick(sum, from, all_), holder = at < 0 ? at + 32 : at;
    if (lane == max(holder, 0)) {
        int found = -1;
        double acc = from;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const bool before_goal = !(acc > goal);
            acc += v[e];
            if (v[e] > 0.0 && (found < 0 || before_goal)) found = first + e;
        }
        p.out[row] = found;
    }
    __syncwarp();
    cluster.barrier_wait(std::move(arrived));
}

template <typename T, bool GREEDY> cudaError_t launch(const VerifyArgs& a, bool draft, cudaStream_t s) {
    verify_rows_kernel<T, GREEDY><<<(unsigned)(a.nrows * (draft ? 2 : 1)) * a.chunks, VD_THREADS, 0, s>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const int size = GREEDY ? 1 : VD_CLUSTER, tiles = (a.vocab + VD_TILE - 1) / VD_TILE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.nseq * size);
    cfg.blockDim = dim3(VD_PICK_THREADS);
    cfg.dynamicSmemBytes = GREEDY ? 0 : (size_t)((tiles + size - 1) / size) * 8;
    cfg.stream = s;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = size;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, verify_pick_kernel<T, GREEDY>, a);
}
template <typename T> cudaError_t launch_mode(const VerifyArgs& a, bool greedy, bool draft, cudaStream_t s) {
    return greedy ? launch<T, true>(a, false, s) : launch<T, false>(a, draft, s);
}
int check(int nrows, int nseq, int vocab) {
    if (nseq < 0 || nseq > 65535) return refuse(CD_ERR_INVALID, CALL, "nseq must be in 0..65535");
    if (nrows < 0 || nrows > 1 << 20) return refuse(CD_ERR_INVALID, CALL, "nrows must be in 0..1048576");
    if (vocab < 1) return refuse(CD_ERR_INVALID, CALL, "vocab must be positive");
    if (vocab > VD_VOCAB) return refuse(CD_ERR_UNSUPPORTED, CALL, "at most 4194304 tokens");
    return CD_OK;
}
size_t workspace_of(int nrows) { return (size_t)nrows * 2 * VD_CHUNKS * sizeof(Part) + 256; }
}  // namespace

extern "C" int cd_verify_drafts_workspace(int nrows, int nseq, int vocab, size_t* bytes) {
    if (!bytes) return refuse(CD_ERR_INVALID, CALL, "null argument");
    if (int rc = check(nrows, nseq, vocab)) return rc;
    *bytes = workspace_of(nrows);
    return CD_OK;
}

extern "C" int cd_verify_drafts(int device, int dtype, int nseq, int nrows, int max_rows, int vocab, const void* target, int64_t target_stride,
                                const void* draft, int64_t draft_stride, const int32_t* tokens, const int32_t* row_start, const float* uniforms,
                                const float* draws, double temperature, int32_t* accepted, int32_t* out_tokens, int32_t* status, void* workspace,
                                size_t workspace_bytes, void* stream) {
    if (int rc = check(nrows, nseq, vocab)) return rc;
    if (dtype < CD_DTYPE_F32 || dtype > CD_DTYPE_BF16) return refuse(CD_ERR_INVALID, CALL, "logits are f32, f16 or bf16");
    if (max_rows < 1) return refuse(CD_ERR_INVALID, CALL, "max_rows must be positive");
    if (!(temperature == 0.0 || (temperature >= 1e-6 && temperature <= 1e6))) return refuse(CD_ERR_INVALID, CALL, "temperature must be 0 or in 1e-6..1e6");
    if (nseq == 0) return CD_OK;
    if (!row_start || !accepted || !workspace) return refuse(CD_ERR_INVALID, CALL, "null argument");
    if (nrows > 0 && (!target || !tokens || !out_tokens)) return refuse(CD_ERR_INVALID, CALL, "null argument");
    const bool greedy = temperature == 0.0;
    if (nrows > 0 && !greedy && (!uniforms || !draws)) return refuse(CD_ERR_INVALID, CALL, "uniforms and draws are needed above temperature 0");
    if (target_stride == 0) target_stride = vocab;
    if (draft_stride == 0) draft_stride = vocab;
    if (target_stride < vocab || draft_stride < vocab) return refuse(CD_ERR_INVALID, CALL, "a row stride is shorter than a row");
    if (!aligned(target, dtype_size(dtype)) || !aligned(draft, dtype_size(dtype))) return refuse(CD_ERR_INVALID, CALL, "logits are not aligned to their type");
    if (!aligned(tokens, 4) || !aligned(row_start, 4) || !aligned(uniforms, 4) || !aligned(draws, 4) || !aligned(accepted, 4) || !aligned(out_tokens, 4) ||
        !aligned(status, 4) || !aligned(workspace, 256))
        return refuse(CD_ERR_INVALID, CALL, "int32 and fp32 arrays start on 4-byte boundaries, the workspace on a 256-byte one");
    if (workspace_bytes < workspace_of(nrows)) return refuse(CD_ERR_CAPACITY, CALL, "the workspace is smaller than cd_verify_drafts_workspace says");
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return cuda_status(guard.err, CALL);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (nrows == 0) return cuda_status(cudaMemsetAsync(accepted, 0, (size_t)nseq * 4, s), CALL);
    VerifyArgs a;
    a.target = target;
    a.draft = greedy ? nullptr : draft;
    a.target_stride = target_stride;
    a.draft_stride = draft_stride;
    a.tokens = tokens;
    a.row_start = row_start;
    a.uniforms = uniforms;
    a.draws = draws;
    a.accepted = accepted;
    a.out = out_tokens;
    a.status = status;
    a.parts = static_cast<Part*>(workspace);
    a.inv_t = greedy ? 1.0 : 1.0 / temperature;
    a.nseq = nseq;
    a.nrows = nrows;
    a.max_rows = max_rows;
    a.vocab = vocab;
    // chunks of a row: enough CTAs for the GPU (eight an SM), none below 2048 elements
    int sms = 0;
    if (cudaError_t e = sm_count(&sms); e != cudaSuccess) return cuda_status(e, CALL);
    const long long rows = (long long)nrows * (a.draft ? 2 : 1), want = std::max<long long>(1, (sms * 8 + rows - 1) / rows);
    a.chunks = (int)std::max<long long>(1, std::min<long long>({want, (vocab + 2047) / 2048, VD_CHUNKS}));
    a.chunk = ((vocab + a.chunks - 1) / a.chunks + 7) & ~7;
    // What a row's sum may be off by, in units of 2^-24 of it: the exponentials 4; their arguments' three roundings, 3 ln 2 for each of the at most 22 powers
    // of two that a term of 2^22 lies below the largest on average (weighted by the terms, an entropy); 32 terms summed at a time; a sum over
    // the loads and a rescaling by another exponential, 8 a load; three joints' exponentials.  p's and q's together twice that.
    a.near = (4 + 46 + 32 + 8.0 * (a.chunk / (VD_THREADS * 16) + 2) + 24) * 2.0 / (1 << 24);
    cudaError_t e;
    if (dtype == CD_DTYPE_F32) e = launch_mode<float>(a, greedy, a.draft != nullptr, s);
    else if (dtype == CD_DTYPE_F16) e = launch_mode<__half>(a, greedy, a.draft != nullptr, s);
    else e = launch_mode<__nv_bfloat16>(a, greedy, a.draft != nullptr, s);
    return cuda_status(e, CALL);
}
