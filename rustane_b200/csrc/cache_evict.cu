// cd_cache_evict: every sequence and kv head of a paged cache down to its `keep` heaviest entries.
//
// evict_select_kernel: a cluster of CTAs per (sequence, kv head) brings the entries' weights into shared memory as ordered 32-bit keys
// and finds the keep-th largest by up to three histograms (11, 11 and 10 bits; none more than needed), joined over the cluster through
// distributed shared memory, every CTA adding up its share of the bins; equal keys are counted off in order of place.  Survivors in
// places >= keep pair up with the holes below in order, so an entry moves at most once, only as many move as have to (one, for a cache
// that grows by one a step), sources and targets never overlap, and nothing but the two lists of places goes through memory.
// Bound by its chain of barriers and memory latencies: 36 us for 32 heads of 60001 entries in clusters of eight, 11 us for 128 heads
// of 2049.  (One loop of loads after the other, and histograms read word by word from every CTA of the cluster: 95 and 20 us.)
// evict_move_kernel: the pairs of all heads, spread over the GPU, 16 bytes a thread, four pairs under way.  Bound by rows of 256 bytes
// from all over the pool: 360000 pairs, 368 MB, 88 us, 4.2 TB/s (109 us with one pair at a time).
#include <cooperative_groups.h>

#include <algorithm>

#include "serve.cuh"

namespace cg = cooperative_groups;
using namespace cd;

namespace {
const char* CALL = "cd_cache_evict";
constexpr int EV_THREADS = 512, EV_WARPS = EV_THREADS / 32, EV_BINS = 2048, EV_CLUSTER = 8, EV_MOVE_THREADS = 256;
constexpr int EV_RESIDENT = 44000;  // keys a CTA holds; beyond them they are made again from the weights at every use

struct EvictArgs {
    PagedView c;
    int keep, sinks, recent, moves, row_bytes;  // moves: most pairs a head can have
    int* lens_out;
    float* weight_out;
    int* position_out;
    int *holes, *sources, *counts;  // [heads][moves] places, [heads]
};

// Larger weight, larger key; the two zeros are one; NaN below -inf
__device__ inline uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
    return u >> 31 ? ~u : u | 0x80000000u;
}

struct Shared {
    alignas(16) uint32_t hist[EV_BINS], total[EV_BINS];  // this CTA's; the cluster's, this CTA's share of the bins
    alignas(16) int warp_sums[EV_WARPS], warp_sums2[EV_WARPS];
    int newest, ties, holes, sources;  // this CTA's, read by the cluster
    uint32_t bin, above;               // of the pass: the bin that holds the keep-th largest, keys above it
    int red[32];
};

// exclusive sum over the block's warps of each warp's v (uniform in the warp), and the block's total; ends with a barrier
__device__ inline int warps_before(int v, int* sums, int& total) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) sums[warp] = v;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < EV_WARPS; i += 4) {
        const int4 x = *reinterpret_cast<const int4*>(sums + i);
        before += (i < warp ? x.x : 0) + (i + 1 < warp ? x.y : 0) + (i + 2 < warp ? x.z : 0) + (i + 3 < warp ? x.w : 0);
        total += x.x + x.y + x.z + x.w;
    }
    __syncthreads();
    return before;
}

// use(i, load(i)) for i = first, first + step .. below end, eight loads at a time: one after the other, each would wait for memory
template <typename L, typename U> __device__ inline void for_batches(int first, int end, int step, L&& load, U&& use, bool any) {
    if (!any) return;
    constexpr int DEEP = 8;
    for (int i = first; i < end; i += step * DEEP) {
        decltype(load(0)) v[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
            if (i + d * step < end) v[d] = load(i + d * step);
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
            if (i + d * step < end) use(i + d * step, v[d]);
    }
}

template <bool RESIDENT> __global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(const __grid_constant__ EvictArgs p) {
    extern __shared__ uint32_t keys[];
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int size = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int unit = blockIdx.x / size, b = unit / p.c.kv_heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* weight = p.c.weight + (size_t)unit * p.c.cap;
    const int* position = p.c.position + (size_t)unit * p.c.cap;
    float* weight_out = p.weight_out + (size_t)unit * p.c.cap;
    int* position_out = p.position_out + (size_t)unit * p.c.cap;
    const int given = p.c.lens[b], len = given < 0 || given > p.c.cap ? 0 : given, keep = p.keep;
    if (len != given) report(p.c.status, CD_STATUS_BATCH);
    if (unit % p.c.kv_heads == 0 && rank == 0 && tid == 0) p.lens_out[b] = len != given ? given : min(len, keep);
    const bool same_w = weight_out == weight, same_p = position_out == position;
    if (len <= keep || keep == 0) {
        for_batches(rank * EV_THREADS + tid, p.c.cap, size * EV_THREADS, [&](int i) { return make_int2(__float_as_int(weight[i]), position[i]); }, [&](int i, int2 v) {
            if (!same_w) weight_out[i] = __int_as_float(v.x);
            if (!same_p) position_out[i] = v.y;
        }, !same_w || !same_p);
        if (rank == 0 && tid == 0) p.counts[unit] = 0;
        return;
    }
    const int per = (len + size - 1) / size, s0 = min(len, rank * per), s1 = min(len, s0 + per), mine = s1 - s0;
    auto sync_all = [&]() {
        if (size == 1) __syncthreads();
        else cluster.sync();
    };
    auto of_rank = [&](auto* mine_, int r) { return r == rank ? mine_ : cluster.map_shared_rank(mine_, r); };

    // One pass over weights and positions: the keys as if nothing were protected, the newest position, and a copy of the
    // bookkeeping (what a hole keeps of it the moves write over).
    int newest = INT_MIN;
    bool low = false;  // an entry of this CTA at a position below `sinks` (with no sinks a negative one)
    for_batches(tid, mine, EV_THREADS, [&](int i) { return make_int2(__float_as_int(weight[s0 + i]), position[s0 + i]); }, [&](int i, int2 v) {
        if (RESIDENT) keys[i] = weight_key(__int_as_float(v.x));
        if (!same_w) weight_out[s0 + i] = __int_as_float(v.x);
        if (!same_p) position_out[s0 + i] = v.y;
        newest = max(newest, v.y);
        low |= v.y < p.sinks;
    }, true);
    for_batches(len + rank * EV_THREADS + tid, p.c.cap, size * EV_THREADS, [&](int i) { return make_int2(__float_as_int(weight[i]), position[i]); }, [&](int i, int2 v) {
        if (!same_w) weight_out[i] = __int_as_float(v.x);
        if (!same_p) position_out[i] = v.y;
    }, !same_w || !same_p);
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) sh.red[warp] = newest;
    low = __syncthreads_or(low);
    if (warp == 0) {
        newest = __reduce_max_sync(0xffffffffu, lane < EV_WARPS ? sh.red[lane] : INT_MIN);
        if (lane == 0) sh.newest = newest;
    }
    sync_all();
    newest = INT_MIN;
#pragma unroll
    for (int r = 0; r < EV_CLUSTER; ++r)
        if (r < size) newest = max(newest, *of_rank(&sh.newest, r));
    const long long recent_from = (long long)newest - p.recent;
    auto protects = [&](int pos) { return pos < p.sinks || pos > recent_from; };
    auto key = [&](int i) { return RESIDENT ? keys[i] : protects(position[s0 + i]) ? 0xffffffffu : weight_key(weight[s0 + i]); };
    if (RESIDENT && (low || p.recent > 0))
        for_batches(tid, mine, EV_THREADS, [&](int i) { return position[s0 + i]; }, [&](int i, int pos) {
            if (protects(pos)) keys[i] = 0xffffffffu;
        }, true);

    // the keep-th largest key, digit by digit, until all keys with its digits so far stay; `rest`: how many of those do
    uint32_t prefix = 0;
    int rest = keep, bits = 32, equal = 0;
    for (int pass = 0; pass < 3; ++pass) {
        const int width = pass < 2 ? 11 : 10, bins = 1 << width, shift = bits - width;
        reinterpret_cast<uint4*>(sh.hist)[tid] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (int i = tid; i < mine; i += EV_THREADS) {
            const uint32_t k = key(i);
            if (pass == 0 || k >> bits == prefix) atomicAdd(&sh.hist[k >> shift & (bins - 1)], 1u);
        }
        sync_all();
        // every CTA adds up its share of the bins; then from the top: thread t has the four bins below bins - 4 t
        if (tid * 4 < bins / size) {
            const int at = rank * (bins / size) + tid * 4;
            uint4 all4 = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < EV_CLUSTER; ++r)
                if (r < size) {
                    const uint4 h = *reinterpret_cast<const uint4*>(of_rank(sh.hist, r) + at);
                    all4.x += h.x; all4.y += h.y; all4.z += h.z; all4.w += h.w;
                }
            *reinterpret_cast<uint4*>(sh.total + tid * 4) = all4;
        }
        sync_all();
        const int low = bins - 4 - 4 * tid;
        uint4 sum4 = make_uint4(0, 0, 0, 0);
        if (low >= 0) sum4 = *reinterpret_cast<const uint4*>(of_rank(sh.total, low / (bins / size)) + low % (bins / size));
        const uint32_t count[4] = {sum4.w, sum4.z, sum4.y, sum4.x}, sum = sum4.x + sum4.y + sum4.z + sum4.w;
        uint32_t before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        int total;
        const uint32_t warps = (uint32_t)warps_before((int)__shfl_sync(0xffffffffu, before, 31), sh.warp_sums, total);
        before += warps - sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (before < (uint32_t)rest && before + count[j] >= (uint32_t)rest) {
                sh.bin = low + 3 - j;
                sh.above = before;
                sh.red[0] = (int)count[j];
            }
            before += count[j];
        }
        __syncthreads();
        prefix = prefix << width | sh.bin;
        rest -= (int)sh.above;
        equal = sh.red[0];
        bits = shift;
        if (rest == equal) break;
    }
    // `equal` keys begin with the threshold's digits, the first `rest` of them stay (fewer than all only with all digits known)
    const int chunk = (mine + EV_WARPS - 1) / EV_WARPS, w0 = min(mine, warp * chunk), w1 = min(mine, w0 + chunk);  // a warp's run of places
    const bool ties = rest < equal;
    int tie_at = 0;
    if (ties) {  // (the same in every CTA of the cluster)
        int n = 0, total;
        for (int i = w0; i < w1; i += 32) n += __popc(__ballot_sync(0xffffffffu, i + lane < w1 && key(min(i + lane, w1 - 1)) == prefix));
        tie_at = warps_before(n, sh.warp_sums, total);
        if (tid == 0) sh.ties = total;
        sync_all();
#pragma unroll
        for (int r = 0; r < EV_CLUSTER; ++r)
            if (r < rank) tie_at += *of_rank(&sh.ties, r);
    }
    const uint32_t below = lane == 0 ? 0u : 0xffffffffu >> (32 - lane);
    // which stay, in order: f(place, in, stays) for 32 places at a time (without ties tie_at is 0 and `rest` all equal keys: all stay)
    auto walk = [&](auto&& f) {
        int tie = tie_at;
        for (int i = w0; i < w1; i += 32) {
            const bool in = i + lane < w1;
            const uint32_t k = in ? key(i + lane) >> bits : 0u;
            const uint32_t same = __ballot_sync(0xffffffffu, in && k == prefix);
            const bool stays = in && (k > prefix || (k == prefix && tie + __popc(same & below) < rest));
            tie += __popc(same);
            f(s0 + i + lane, in, stays);
        }
    };
    int holes = 0, sources = 0;
    walk([&](int place, bool in, bool stays) {
        holes += __popc(__ballot_sync(0xffffffffu, in && place < keep && !stays));
        sources += __popc(__ballot_sync(0xffffffffu, in && place >= keep && stays));
    });
    int total_h, total_s;
    int hole_at = warps_before(holes, sh.warp_sums, total_h), source_at = warps_before(sources, sh.warp_sums2, total_s);
    if (tid == 0) {
        sh.holes = total_h;
        sh.sources = total_s;
    }
    sync_all();
    int all = 0;
#pragma unroll
    for (int r = 0; r < EV_CLUSTER; ++r)
        if (r < size) {
            const int h = *of_rank(&sh.holes, r), n = *of_rank(&sh.sources, r);
            if (r < rank) {
                hole_at += h;
                source_at += n;
            }
            all += h;
        }
    if (rank == 0 && tid == 0) p.counts[unit] = all;
    int *hole_list = p.holes + (size_t)unit * p.moves, *source_list = p.sources + (size_t)unit * p.moves;
    walk([&](int place, bool in, bool stays) {
        const bool hole = in && place < keep && !stays, source = in && place >= keep && stays;
        const uint32_t hs = __ballot_sync(0xffffffffu, hole), ss = __ballot_sync(0xffffffffu, source);
        if (hole) hole_list[hole_at + __popc(hs & below)] = place;
        if (source) source_list[source_at + __popc(ss & below)] = place;
        hole_at += __popc(hs);
        source_at += __popc(ss);
    });
    sync_all();  // nobody reads this CTA's shared memory any more
}

// One pair a group of LANES lanes: K and V rows of LANES * 16 bytes, weight and position.
template <int LANES> __global__ void __launch_bounds__(EV_MOVE_THREADS) evict_move_kernel(const __grid_constant__ EvictArgs p) {
    const int unit = blockIdx.y, b = unit / p.c.kv_heads, head = unit % p.c.kv_heads;
    const int sub = threadIdx.x % LANES, group = blockIdx.x * (EV_MOVE_THREADS / LANES) + threadIdx.x / LANES, groups = gridDim.x * (EV_MOVE_THREADS / LANES);
    pdl_wait();
    const int n = __ldcg(p.counts + unit);
    const int *holes = p.holes + (size_t)unit * p.moves, *sources = p.sources + (size_t)unit * p.moves;
    const size_t at = (size_t)unit * p.c.cap;
    char* pool = static_cast<char*>(p.c.pool);
    constexpr int DEEP = 4;  // pairs under way: places, then pages, then rows
    for (int i0 = group; i0 < n; i0 += groups * DEEP) {
        int to[DEEP], from[DEEP];
        uint4 k[DEEP], v[DEEP];
        float w[DEEP];
        int pos[DEEP], page_to[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const int i = i0 + d * groups;
            to[d] = i < n ? __ldcg(holes + i) : -1;
            from[d] = i < n ? __ldcg(sources + i) : 0;
        }
        int word_to[DEEP], word_from[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
            if (to[d] >= 0) {
                word_to[d] = page_word(p.c, b, to[d]);
                word_from[d] = page_word(p.c, b, from[d]);
            }
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
            if (to[d] >= 0) {
                page_to[d] = checked_page(p.c, word_to[d]);
                const int page_from = checked_page(p.c, word_from[d]);
                if (page_from < 0) page_to[d] = -1;
                if (page_to[d] >= 0) {
                    k[d] = *(reinterpret_cast<const uint4*>(pool + row_at(p.c, page_from, 0, head, from[d], LANES * 16)) + sub);
                    v[d] = *(reinterpret_cast<const uint4*>(pool + row_at(p.c, page_from, 1, head, from[d], LANES * 16)) + sub);
                }
                const int kept = page_to[d] >= 0 ? from[d] : to[d];
                if (sub == 0) w[d] = p.c.weight[at + kept];
                if (sub == 1) pos[d] = p.c.position[at + kept];
            }
#pragma unroll
        for (int d = 0; d < DEEP; ++d)
            if (to[d] >= 0) {
                if (page_to[d] >= 0) {
                    *(reinterpret_cast<uint4*>(pool + row_at(p.c, page_to[d], 0, head, to[d], LANES * 16)) + sub) = k[d];
                    *(reinterpret_cast<uint4*>(pool + row_at(p.c, page_to[d], 1, head, to[d], LANES * 16)) + sub) = v[d];
                }
                if (sub == 0) p.weight_out[at + to[d]] = w[d];
                if (sub == 1) p.position_out[at + to[d]] = pos[d];
            }
    }
}

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }
struct Plan {
    size_t units, list, bytes;
    int moves;
};
Plan plan_of(const cd_paged_cache* c, int keep) {
    Plan p;
    const long long cap = (long long)c->max_pages * c->page_tokens;
    p.units = (size_t)c->nseq * c->kv_heads;
    p.moves = (int)std::max<long long>(0, std::min<long long>(keep, cap - keep));
    p.list = up(p.units * p.moves * 4);
    p.bytes = 2 * p.list + up(p.units * 4) + 256;
    return p;
}
int check(const cd_paged_cache* c, int keep) {
    if (int rc = check_cache(c, CALL)) return rc;
    if (!c->weight) return refuse(CD_ERR_INVALID, CALL, "the cache needs its bookkeeping (weight and position)");
    if (keep < 0) return refuse(CD_ERR_INVALID, CALL, "keep must not be negative");
    if ((long long)c->max_pages * c->page_tokens > 1 << 30) return refuse(CD_ERR_UNSUPPORTED, CALL, "max_pages * page_tokens must not exceed 2^30");
    return CD_OK;
}

template <int LANES> cudaError_t move(const EvictArgs& a, unsigned units, int sms, cudaStream_t s) {
    const int per = EV_MOVE_THREADS / LANES;
    const unsigned most = (unsigned)((a.moves + per - 1) / per), share = (unsigned)((8 * sms + units - 1) / units);
    return launch_dependent(evict_move_kernel<LANES>, dim3(std::max(1u, std::min(most, share)), units), dim3(EV_MOVE_THREADS), 0, s, a);
}
}  // namespace

extern "C" int cd_cache_evict_workspace(const cd_paged_cache* c, int keep, size_t* bytes) {
    if (!bytes) return refuse(CD_ERR_INVALID, CALL, "null argument");
    if (int rc = check(c, keep)) return rc;
    *bytes = plan_of(c, keep).bytes;
    return CD_OK;
}

extern "C" int cd_cache_evict(const cd_paged_cache* c, int keep, int sinks, int recent, int32_t* lens_out, float* weight_out, int32_t* position_out,
                              void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check(c, keep)) return rc;
    if (sinks < 0 || recent < 0 || (long long)sinks + recent > keep) return refuse(CD_ERR_INVALID, CALL, "sinks and recent must not be negative, nor more than keep together");
    if (c->nseq == 0) return CD_OK;
    if (!lens_out || !weight_out || !position_out || !workspace) return refuse(CD_ERR_INVALID, CALL, "null argument");
    if (lens_out == c->lens) return refuse(CD_ERR_INVALID, CALL, "lens_out must not be the cache's lens");
    if (!aligned(lens_out, 4) || !aligned(weight_out, 4) || !aligned(position_out, 4) || !aligned(workspace, 256))
        return refuse(CD_ERR_INVALID, CALL, "lens_out, weight_out and position_out start on 4-byte boundaries, the workspace on a 256-byte one");
    const Plan plan = plan_of(c, keep);
    if (plan.units > 65535) return refuse(CD_ERR_UNSUPPORTED, CALL, "at most 65535 sequences times kv heads");
    if (workspace_bytes < plan.bytes) return refuse(CD_ERR_CAPACITY, CALL, "the workspace is smaller than cd_cache_evict_workspace says");
    char* ws = static_cast<char*>(workspace);
    EvictArgs a;
    a.c = view_of(c);
    a.keep = keep;
    a.sinks = sinks;
    a.recent = recent;
    a.moves = plan.moves;
    a.row_bytes = c->hd * (int)dtype_size(c->dtype);
    a.lens_out = lens_out;
    a.weight_out = weight_out;
    a.position_out = position_out;
    a.holes = reinterpret_cast<int*>(ws);
    a.sources = reinterpret_cast<int*>(ws + plan.list);
    a.counts = reinterpret_cast<int*>(ws + 2 * plan.list);
    DeviceGuard guard(c->device);
    if (guard.err != cudaSuccess) return cuda_status(guard.err, CALL);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int sms = 0;
    cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) return cuda_status(e, CALL);
    // CTAs a head: more of them while the GPU has room and each still has 8192 places, and as many as hold the keys.  (208 heads of 33000
    // entries, one to go: 118 us with eight each, which wait for one another more than they work.)
    int size = 1;
    while (size < EV_CLUSTER && ((long long)size * EV_RESIDENT < a.c.cap || ((long long)plan.units * size < 2 * sms && (long long)size * 8192 < a.c.cap))) size *= 2;
    const int per = (a.c.cap + size - 1) / size;
    const bool resident = per <= EV_RESIDENT;
    const size_t shared = resident ? (size_t)per * 4 : 0;
    void (*kernel)(EvictArgs) = resident ? evict_select_kernel<true> : evict_select_kernel<false>;
    if (resident && (e = allow_shared_memory((const void*)kernel)) != cudaSuccess) return cuda_status(e, CALL);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)plan.units * size);
    cfg.blockDim = dim3(EV_THREADS);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = s;
    cudaLaunchAttribute at = {};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = size;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if ((e = cudaLaunchKernelEx(&cfg, kernel, a)) != cudaSuccess) return cuda_status(e, CALL);
    switch (a.row_bytes / 16) {
        case 8: e = move<8>(a, (unsigned)plan.units, sms, s); break;
        case 16: e = move<16>(a, (unsigned)plan.units, sms, s); break;
        default: e = move<32>(a, (unsigned)plan.units, sms, s); break;
    }
    return cuda_status(e, CALL);
}
