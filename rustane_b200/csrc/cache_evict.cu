// cd_cache_evict: every sequence and kv head of a paged cache down to its `keep` heaviest entries.
//
// evict_select_kernel: a cluster of CTAs per (sequence, kv head) brings the entries' weights into shared memory as ordered 32-bit keys
// and finds the keep-th largest by three histograms (11, 11 and 10 bits), joined over the cluster through distributed shared memory; equal keys
// are counted off in order of place.  Survivors in places >= keep pair up with the holes below in order, so an entry moves
// at most once, only as many move as have to (one, for a cache that grows by one a step), sources and targets never
// overlap, and nothing but the two lists of places goes through memory.
// evict_move_kernel: the pairs of all heads, spread over the GPU, 16 bytes a thread at a time.
#include <cooperative_groups.h>

#include <algorithm>

#include "serve.cuh"

namespace cg = cooperative_groups;
using namespace cd;

namespace {
const char* CALL = "cd_cache_evict";
constexpr int EV_THREADS = 512, EV_WARPS = EV_THREADS / 32, EV_BINS = 2048, EV_CLUSTER = 8, EV_MOVE_THREADS = 256;
constexpr int EV_RESIDENT = 45000;  // keys a CTA holds; beyond them they are made again from the weights at every use

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
    uint32_t hist[EV_BINS];
    int warp_sums[EV_WARPS], warp_sums2[EV_WARPS];
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
    for (int i = 0; i < EV_WARPS; ++i) {
        if (i < warp) before += sums[i];
        total += sums[i];
    }
    __syncthreads();
    return before;
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
    if (weight_out != weight)
        for (int i = rank * EV_THREADS + tid; i < p.c.cap; i += size * EV_THREADS)
            if (len <= keep || i >= keep) weight_out[i] = weight[i];  // places below: at the end, where they are not holes
    if (position_out != position)
        for (int i = rank * EV_THREADS + tid; i < p.c.cap; i += size * EV_THREADS)
            if (len <= keep || i >= keep) position_out[i] = position[i];
    if (unit % p.c.kv_heads == 0 && rank == 0 && tid == 0) p.lens_out[b] = len != given ? given : min(len, keep);
    if (len <= keep || keep == 0) {
        if (rank == 0 && tid == 0) p.counts[unit] = 0;
        return;
    }
    const int per = (len + size - 1) / size, s0 = min(len, rank * per), s1 = min(len, s0 + per), mine = s1 - s0;

    // the newest position
    int newest = INT_MIN;
    for (int i = s0 + tid; i < s1; i += EV_THREADS) newest = max(newest, position[i]);
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) sh.red[warp] = newest;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < EV_WARPS; ++i) newest = max(newest, sh.red[i]);
        sh.newest = newest;
    }
    cluster.sync();
    newest = INT_MIN;
    for (int r = 0; r < size; ++r) newest = max(newest, *cluster.map_shared_rank(&sh.newest, r));
    const long long recent_from = (long long)newest - p.recent;
    auto make_key = [&](int i) {
        const int pos = position[i];
        return pos < p.sinks || pos > recent_from ? 0xffffffffu : weight_key(weight[i]);
    };
    auto key = [&](int i) { return RESIDENT ? keys[i] : make_key(s0 + i); };
    if (RESIDENT)
        for (int i = tid; i < mine; i += EV_THREADS) keys[i] = make_key(s0 + i);

    // the keep-th largest key, digit by digit; `rest`: how many of the keys with this prefix stay
    uint32_t prefix = 0;
    int rest = keep, bits = 32, equal = 0;
    for (int pass = 0; pass < 3; ++pass) {
        const int width = pass < 2 ? 11 : 10, bins = 1 << width, shift = bits - width;
        for (int i = tid; i < bins; i += EV_THREADS) sh.hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < mine; i += EV_THREADS) {
            const uint32_t k = key(i);
            if (pass == 0 || k >> bits == prefix) atomicAdd(&sh.hist[k >> shift & (bins - 1)], 1u);
        }
        cluster.sync();
        // from the top: thread t has the bins below bins - 4 t (bins - 2 t in the last pass)
        const int each = bins / EV_THREADS;
        uint32_t count[4], sum = 0;
        for (int j = 0; j < each; ++j) {
            const int bin = bins - 1 - (tid * each + j);
            uint32_t n = 0;
            for (int r = 0; r < size; ++r) n += cluster.map_shared_rank(sh.hist, r)[bin];
            count[j] = n;
            sum += n;
        }
        uint32_t before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        int total;
        const uint32_t warps = (uint32_t)warps_before((int)__shfl_sync(0xffffffffu, before, 31), sh.warp_sums, total);
        before += warps - sum;
        for (int j = 0; j < each; ++j) {
            if (before < (uint32_t)rest && before + count[j] >= (uint32_t)rest) {
                sh.bin = bins - 1 - (tid * each + j);
                sh.above = before;
                sh.red[0] = (int)count[j];
            }
            before += count[j];
        }
        cluster.sync();  // every CTA has read the histograms, too
        prefix = prefix << width | sh.bin;
        rest -= (int)sh.above;
        equal = sh.red[0];
        bits = shift;
    }
    // `equal` keys are the threshold itself, the first `rest` of them stay
    const int chunk = (mine + EV_WARPS - 1) / EV_WARPS, w0 = min(mine, warp * chunk), w1 = min(mine, w0 + chunk);  // a warp's run of places
    const bool ties = rest < equal;
    int tie_at = 0;
    if (ties) {  // (the same in every CTA of the cluster)
        int n = 0, total;
        for (int i = w0; i < w1; i += 32) n += __popc(__ballot_sync(0xffffffffu, i + lane < w1 && key(min(i + lane, w1 - 1)) == prefix));
        tie_at = warps_before(n, sh.warp_sums, total);
        if (tid == 0) sh.ties = total;
        cluster.sync();
        for (int r = 0; r < rank; ++r) tie_at += *cluster.map_shared_rank(&sh.ties, r);
    }
    const uint32_t below = lane == 0 ? 0u : 0xffffffffu >> (32 - lane);
    // which stay, in order: f(place, in, stays) for 32 places at a time (without ties tie_at is 0 and `rest` all equal keys: all stay)
    auto walk = [&](auto&& f) {
        int tie = tie_at;
        for (int i = w0; i < w1; i += 32) {
            const bool in = i + lane < w1;
            const uint32_t k = in ? key(i + lane) : 0u;
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
    cluster.sync();
    int all = 0;
    for (int r = 0; r < size; ++r) {
        const int h = *cluster.map_shared_rank(&sh.holes, r), s = *cluster.map_shared_rank(&sh.sources, r);
        if (r < rank) {
            hole_at += h;
            source_at += s;
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
        if (in && place < keep && stays) {
            if (weight_out != weight) weight_out[place] = weight[place];
            if (position_out != position) position_out[place] = position[place];
        }
    });
    cluster.sync();  // nobody reads this CTA's shared memory any more
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
#pragma unroll 4
    for (int i = group; i < n; i += groups) {
        const int to = __ldcg(holes + i), from = __ldcg(sources + i);
        const int page_to = page_at(p.c, b, to), page_from = page_at(p.c, b, from);
        if (page_to >= 0 && page_from >= 0) {
            const uint4 k = *(reinterpret_cast<const uint4*>(pool + row_at(p.c, page_from, 0, head, from, LANES * 16)) + sub);
            const uint4 v = *(reinterpret_cast<const uint4*>(pool + row_at(p.c, page_from, 1, head, from, LANES * 16)) + sub);
            *(reinterpret_cast<uint4*>(pool + row_at(p.c, page_to, 0, head, to, LANES * 16)) + sub) = k;
            *(reinterpret_cast<uint4*>(pool + row_at(p.c, page_to, 1, head, to, LANES * 16)) + sub) = v;
        }
        const int kept = page_to >= 0 && page_from >= 0 ? from : to;
        if (sub == 0) p.weight_out[at + to] = p.c.weight[at + kept];
        if (sub == 1) p.position_out[at + to] = p.c.position[at + kept];
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
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return cuda_status(e, CALL);
    int size = 1;  // one CTA for every 8192 places, so that a pass over the keys stays short
    while (size < EV_CLUSTER && (long long)size * 8192 < a.c.cap) size *= 2;
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
