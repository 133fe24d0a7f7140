// What the operators of a serving step share: the batch and its paged cache as kernels see them, and the checks of both.
//
// Lengths, rows and page ids live on the device and a call never waits for them, so every kernel checks what it is about to use
// as an address: batch_seq() leaves a sequence out whose rows or length do not fit, page_at() refuses a page outside the pool.
#pragma once
#include <atomic>
#include <string>

#include "model.h"

namespace cd {

struct PagedView {
    int kv_heads, page_tokens, page_shift, npages, nseq, max_pages, cap;  // page_shift: log2(page_tokens), or -1; cap: entries a sequence may have
    long long table_stride;
    void* pool;
    const int *page_table, *lens;
    float* weight;
    int *position, *status;
};

__device__ inline void report(int* status, int bit) {
    if (status) atomicOr(status, bit);
}

struct BatchSeq {
    int r0, n, len;  // first row, rows, cache entries; n = 0 and len = 0: left out
};
__device__ inline BatchSeq batch_seq(const PagedView& c, const int* row_start, int b, int nrows, int max_rows) {
    BatchSeq s;
    const int r1 = row_start[b + 1];
    s.r0 = row_start[b];
    s.len = c.lens[b];
    const bool bad = s.r0 < 0 || r1 < s.r0 || r1 > nrows || r1 - s.r0 > max_rows || s.len < 0 || s.len > c.cap;
    s.n = r1 - s.r0;
    if (bad) {
        report(c.status, CD_STATUS_BATCH);
        s.r0 = s.n = s.len = 0;
    }
    return s;
}
__device__ inline int page_of(const PagedView& c, int entry) { return c.page_shift >= 0 ? entry >> c.page_shift : entry / c.page_tokens; }
// The table's word for the page that holds `entry` (0 <= entry < cap) of sequence b, and what it names: a page of the pool, or -1.
// (Apart, so that a word can be asked for long before it is looked at.)
__device__ inline int page_word(const PagedView& c, int b, int entry) {
    int w;  // (volatile: the compiler leaves the load where it is written)
    asm volatile("ld.global.nc.s32 %0, [%1];" : "=r"(w) : "l"(c.page_table + b * c.table_stride + page_of(c, entry)));
    return w;
}
__device__ inline int checked_page(const PagedView& c, int page) {
    if ((unsigned)page < (unsigned)c.npages) return page;
    report(c.status, CD_STATUS_PAGE);
    return -1;
}
__device__ inline int page_at(const PagedView& c, int b, int entry) { return checked_page(c, page_word(c, b, entry)); }
// Element offset of entry's row in the pool; which: 0 K, 1 V.  64 bits: a pool passes 2^31 elements.
__device__ inline size_t row_at(const PagedView& c, int page, int which, int head, int entry, int hd) {
    const int off = entry - page_of(c, entry) * c.page_tokens;
    return ((((size_t)page * 2 + which) * c.kv_heads + head) * c.page_tokens + off) * hd;
}

template <typename T> __device__ inline T from_float(float v);
template <> __device__ inline float from_float<float>(float v) { return v; }
template <> __device__ inline __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ inline __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <typename T> __device__ inline float as_float(T v);
template <> __device__ inline float as_float<float>(float v) { return v; }
template <> __device__ inline float as_float<__half>(__half v) { return __half2float(v); }
template <> __device__ inline float as_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
// 2^x to 2^-22 of itself; 0 for -inf
__device__ inline float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------------------------------------------------------ host side
// The caller's device for the length of a call.
struct DeviceGuard {
    int before = -1;
    cudaError_t err = cudaSuccess;
    explicit DeviceGuard(int device) {
        if (device < 0) return;
        int now = -1;
        err = cudaGetDevice(&now);
        if (err != cudaSuccess || now == device) return;
        err = cudaSetDevice(device);
        if (err == cudaSuccess) before = now;
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
};
// SMs of the current device (asked for once a device)
inline cudaError_t sm_count(int* sms) {
    static std::atomic<int> known[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && (*sms = known[dev].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
    e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess && dev < 64) known[dev].store(*sms, std::memory_order_relaxed);
    return e;
}
inline size_t dtype_size(int dtype) { return dtype == CD_DTYPE_F32 ? 4 : 2; }
inline bool aligned(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
inline int refuse(int code, const char* call, const char* what) { return fail(nullptr, code, std::string(call) + ": " + what); }
inline int cuda_status(cudaError_t e, const char* call) {
    return e == cudaSuccess ? CD_OK : fail(nullptr, CD_ERR_CUDA, std::string(call) + ": " + cudaGetErrorString(e));
}

inline int check_cache(const cd_paged_cache* c, const char* call) {
    if (!c) return refuse(CD_ERR_INVALID, call, "null cache");
    if (c->dtype < CD_DTYPE_F32 || c->dtype > CD_DTYPE_BF16) return refuse(CD_ERR_INVALID, call, "the pool is f32, f16 or bf16");
    if (c->kv_heads <= 0 || c->kv_heads > 4096) return refuse(CD_ERR_INVALID, call, "kv_heads must be in 1..4096");
    if (c->hd != 64 && c->hd != 128) return refuse(CD_ERR_UNSUPPORTED, call, "head dimension must be 64 or 128");
    if (c->page_tokens <= 0 || c->page_tokens > 65536) return refuse(CD_ERR_INVALID, call, "page_tokens must be in 1..65536");
    if (c->npages <= 0 || c->max_pages <= 0) return refuse(CD_ERR_INVALID, call, "the pool and the page table hold at least one page");
    if (c->nseq < 0 || c->nseq > 4096) return refuse(CD_ERR_UNSUPPORTED, call, "at most 4096 sequences");
    if ((long long)c->max_pages * c->page_tokens > 0x7ffffc00ll) return refuse(CD_ERR_UNSUPPORTED, call, "max_pages * page_tokens must stay below 2^31 - 1024");
    if (c->table_stride < c->max_pages && c->nseq > 1) return refuse(CD_ERR_INVALID, call, "table_stride is shorter than a page_table row");
    if (!c->pool || !c->page_table || !c->lens) return refuse(CD_ERR_INVALID, call, "null pool, page_table or lens");
    if (!c->weight != !c->position) return refuse(CD_ERR_INVALID, call, "weight and position come together");
    if (!aligned(c->pool, 16)) return refuse(CD_ERR_INVALID, call, "the pool must start on a 16-byte boundary");
    if (!aligned(c->page_table, 4) || !aligned(c->lens, 4) || !aligned(c->weight, 4) || !aligned(c->position, 4) || !aligned(c->status, 4))
        return refuse(CD_ERR_INVALID, call, "page_table, lens, weight, position and status must start on a 4-byte boundary");
    return CD_OK;
}
inline PagedView view_of(const cd_paged_cache* c) {
    PagedView v;
    v.kv_heads = c->kv_heads;
    v.page_tokens = c->page_tokens;
    v.page_shift = (c->page_tokens & (c->page_tokens - 1)) == 0 ? __builtin_ctz(c->page_tokens) : -1;
    v.npages = c->npages;
    v.nseq = c->nseq;
    v.max_pages = c->max_pages;
    v.cap = c->max_pages * c->page_tokens;
    v.table_stride = c->table_stride;
    v.pool = c->pool;
    v.page_table = c->page_table;
    v.lens = c->lens;
    v.weight = c->weight;
    v.position = c->position;
    v.status = c->status;
    return v;
}
// q, k, v of a batch: `dtype`, their row strides and the alignment the 16-byte loads need.
inline int check_rows(const void* p, int64_t stride, int64_t packed, int dtype, const char* call) {
    if (!p) return refuse(CD_ERR_INVALID, call, "null argument");
    if (stride < packed) return refuse(CD_ERR_INVALID, call, "a row stride is shorter than a row");
    if (!aligned(p, 16) || (stride * (int64_t)dtype_size(dtype)) % 16)
        return refuse(CD_ERR_INVALID, call, "rows of q, k, v and out must start on 16-byte boundaries");
    return CD_OK;
}
// Launch as a programmatic dependent of the kernel ahead in the stream (it may start before that one has ended; pdl_wait() orders it).
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cudaLaunchAttribute at = {};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

}  // namespace cd
