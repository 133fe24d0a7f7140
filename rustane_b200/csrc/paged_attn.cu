// cd_paged_attention: the choice of kernel, the workspace and the launches.
#include <algorithm>
#include <cmath>

#include "paged_mma.cuh"

using namespace cd;

namespace {
const char* CALL = "cd_paged_attention";

struct Plan {
    int group, ru, row_warps, blocks;
    size_t units, part_o, part_ml, unit_info, lse2, scores, bytes;  // offsets in the workspace
    long long score_stride;
};
// What a tile costs by its unit's rows: up to 16, 32, more (tensor-core form).  A CTA's four warps work on four places at once, on two, on
// one; HBM evens out part of it.  24 sequences of one to six drafted rows, eight heads a kv head, with these costs, with 1, 2, 4 and with 1, 1, 2: fp16,
// heads of 64, 96, 98 and 100 us; bf16, heads of 128, 126, 121 and 134; fp32 rows over bf16, heads of 64, 132, 139 and 132; over fp16, heads
// of 128, 111, 108 and 114.  Four heads and one to eight rows, bf16, 128: 55, 55 and 63; sixteen heads and one to four rows 142, 142 and 148.
constexpr int PA_WEIGHTS[3] = {2, 4, 7};
size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

// A warp has 4 rows of a unit with an fp32 pool (FMAs), 16 with a 16-bit one (tensor cores); a unit as many of its warps as its rows need.
Plan plan_of(const cd_paged_cache* c, int heads, int nrows, int max_rows, int collect) {
    Plan p;
    p.group = heads / c->kv_heads;
    const int per_warp = c->dtype == CD_DTYPE_F32 ? 4 : 16;
    const long long rows = (long long)max_rows * p.group;
    p.row_warps = rows <= per_warp ? 1 : rows <= 2 * per_warp ? 2 : 4;
    p.ru = per_warp * p.row_warps;
    p.blocks = (int)((rows + p.ru - 1) / p.ru);
    p.units = (size_t)c->nseq * c->kv_heads * p.blocks;
    const size_t slots = PA_MAX_CTAS + p.units;
    p.part_o = 0;
    p.part_ml = up(slots * p.ru * c->hd * 4);
    p.unit_info = p.part_ml + up(slots * p.ru * 8);
    p.lse2 = p.unit_info + up(p.units * 8);
    p.score_stride = ((long long)c->max_pages * c->page_tokens + 3) & ~3ll;
    p.scores = p.lse2 + (collect ? up((size_t)nrows * heads * 4) : 0);
    p.bytes = p.scores + (collect ? up((size_t)nrows * heads * p.score_stride * 4) : 0);
    return p;
}
int check_shape(const cd_paged_cache* c, int heads, int nrows, int max_rows, int collect) {
    if (int rc = check_cache(c, CALL)) return rc;
    if (heads <= 0 || heads % c->kv_heads) return refuse(CD_ERR_INVALID, CALL, "heads must be a positive multiple of kv_heads");
    if (heads > 65536) return refuse(CD_ERR_UNSUPPORTED, CALL, "at most 65536 heads");
    if (nrows < 0 || nrows > 1 << 22) return refuse(CD_ERR_INVALID, CALL, "nrows must be in 0..4194304");
    if (max_rows < 1 || max_rows > 65536) return refuse(CD_ERR_INVALID, CALL, "max_rows must be in 1..65536");
    if (collect && !c->weight) return refuse(CD_ERR_INVALID, CALL, "collect needs the cache's weight");
    const Plan p = plan_of(c, heads, nrows, max_rows, collect);
    // (2^31, and a tile's cost is at most PA_WEIGHTS[2])
    const long long tiles = ((long long)c->max_pages * c->page_tokens + PA_TILE - 1) / PA_TILE;
    if (p.units > 0x7fffffffull || (long long)p.units * tiles * PA_WEIGHTS[2] >= 0x7fffffffll - PA_MAX_CTAS) return refuse(CD_ERR_UNSUPPORTED, CALL, "sequences x kv heads x row blocks x (max_pages x page_tokens / 64) must stay below 2^28");
    return CD_OK;
}

template <typename KT, typename QT, int HD> cudaError_t launch(const AttnArgs& a, const Plan& plan, int collect, cudaStream_t s) {
    int sms = 0;
    cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) return e;
    if constexpr (std::is_same<KT, float>::value) {
        attn_fma_kernel<QT, HD><<<std::min(2 * sms, PA_MAX_CTAS), PA_THREADS, (size_t)(a.c.nseq + 1) * 4, s>>>(a);
    } else {
        using Size = MmaSize<QT, HD>;
        const bool few = Size::slots(a.row_warps) == 8;
        void (*kernel)(AttnArgs) = attn_mma_kernel<KT, QT, HD, 12, 224>;
        if constexpr (Size::WIDE) {
            if (few) kernel = attn_mma_kernel<KT, QT, HD, 8, 224>;
        } else if constexpr (HD == 64) {
            if (few) kernel = attn_mma_kernel<KT, QT, HD, 8, 160>;
        }
        if ((e = allow_shared_memory((const void*)kernel)) != cudaSuccess) return e;
        const size_t shared = mma_shared<KT, QT, HD>(a.c.nseq, a.row_warps);
        const int fit = (int)(226 * 1024 / (shared + 2560));  // (and what the kernel has of its own and the system takes a CTA)
        kernel<<<std::min(std::max(1, std::min(fit, Size::three(a.row_warps) ? 3 : 2)) * sms, PA_MAX_CTAS), PA_THREADS, shared, s>>>(a);
    }
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    const dim3 grid((unsigned)plan.units, (unsigned)std::min<long long>(a.ru, (long long)a.max_rows * a.group));
    // about 2 sms / units parts a unit: 32 units over 296 CTAs join in 5.3 us with 256 threads a row, 48 units of 48 rows in 8 us with 64 (13 with 256)
    e = plan.units >= 24 ? launch_dependent(attn_join_kernel<QT, HD, 64>, grid, dim3(64), 0, s, a) : launch_dependent(attn_join_kernel<QT, HD, 256>, grid, dim3(256), 0, s, a);
    if (e != cudaSuccess) return e;
    if (collect)
        e = launch_dependent(attn_collect_kernel, dim3((a.c.cap + PA_COLLECT - 1) / PA_COLLECT, a.c.kv_heads, a.c.nseq), dim3(PA_THREADS), 0, s, a);
    return e;
}
template <typename KT, typename QT> cudaError_t launch_hd(int hd, const AttnArgs& a, const Plan& plan, int collect, cudaStream_t s) {
    return hd == 128 ? launch<KT, QT, 128>(a, plan, collect, s) : launch<KT, QT, 64>(a, plan, collect, s);
}
}  // namespace

extern "C" int cd_paged_attention_workspace(const cd_paged_cache* c, int heads, int nrows, int max_rows, int collect, size_t* bytes) {
    if (!bytes) return refuse(CD_ERR_INVALID, CALL, "null argument");
    if (int rc = check_shape(c, heads, nrows, max_rows, collect)) return rc;
    *bytes = plan_of(c, heads, nrows, max_rows, collect).bytes;
    return CD_OK;
}

extern "C" int cd_paged_attention(const cd_paged_cache* c, int dtype, int heads, int nrows, int max_rows, const void* q, int64_t q_stride,
                                  const int32_t* row_start, float scale, int window, int collect, void* out, float* lse, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    if (int rc = check_shape(c, heads, nrows, max_rows, collect)) return rc;
    if (dtype != CD_DTYPE_F32 && dtype != c->dtype) return refuse(CD_ERR_INVALID, CALL, "q is f32 or of the pool's type");
    if (window < 0) return refuse(CD_ERR_INVALID, CALL, "window must not be negative");
    if (!(scale <= 1e30f)) return refuse(CD_ERR_INVALID, CALL, "scale must be finite");
    if (nrows == 0 || c->nseq == 0) return CD_OK;
    const int64_t packed = (int64_t)heads * c->hd;
    if (q_stride == 0) q_stride = packed;
    if (int rc = check_rows(q, q_stride, packed, dtype, CALL)) return rc;
    if (int rc = check_rows(out, packed, packed, dtype, CALL)) return rc;
    if (!row_start || !workspace) return refuse(CD_ERR_INVALID, CALL, "null argument");
    if (!aligned(row_start, 4) || !aligned(lse, 4) || !aligned(workspace, 256))
        return refuse(CD_ERR_INVALID, CALL, "row_start and lse start on 4-byte boundaries, the workspace on a 256-byte one");
    const Plan plan = plan_of(c, heads, nrows, max_rows, collect);
    if (workspace_bytes < plan.bytes) return refuse(CD_ERR_CAPACITY, CALL, "the workspace is smaller than cd_paged_attention_workspace says");
    char* ws = static_cast<char*>(workspace);
    AttnArgs a;
    a.c = view_of(c);
    a.row_start = row_start;
    a.q = q;
    a.out = out;
    a.lse = lse;
    a.part_o = reinterpret_cast<float*>(ws + plan.part_o);
    a.part_ml = reinterpret_cast<float2*>(ws + plan.part_ml);
    a.unit_info = reinterpret_cast<int2*>(ws + plan.unit_info);
    a.lse2 = reinterpret_cast<float*>(ws + plan.lse2);
    a.scores = collect ? reinterpret_cast<float*>(ws + plan.scores) : nullptr;
    a.q_stride = q_stride;
    a.score_stride = plan.score_stride;
    for (int i = 0; i < 3; ++i) a.weights[i] = c->dtype == CD_DTYPE_F32 ? 1 : PA_WEIGHTS[i];
    a.scale_log2 = (scale > 0.f ? scale : 1.0f / std::sqrt((float)c->hd)) * 1.44269504088896340736f;
    a.heads = heads;
    a.group = plan.group;
    a.nrows = nrows;
    a.max_rows = max_rows;
    a.window = window;
    a.ru = plan.ru;
    a.row_warps = plan.row_warps;
    a.blocks = plan.blocks;
    DeviceGuard guard(c->device);
    if (guard.err != cudaSuccess) return cuda_status(guard.err, CALL);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (c->dtype == CD_DTYPE_F32) e = launch_hd<float, float>(c->hd, a, plan, collect, s);
    else if (c->dtype == CD_DTYPE_F16) e = dtype == CD_DTYPE_F32 ? launch_hd<__half, float>(c->hd, a, plan, collect, s) : launch_hd<__half, __half>(c->hd, a, plan, collect, s);
    else e = dtype == CD_DTYPE_F32 ? launch_hd<__nv_bfloat16, float>(c->hd, a, plan, collect, s) : launch_hd<__nv_bfloat16, __nv_bfloat16>(c->hd, a, plan, collect, s);
    return cuda_status(e, CALL);
}
