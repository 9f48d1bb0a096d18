// kv_paged.cu - the paged key-value cache of include/kv_paged.h: block
// tables and slot maps (map_kernel), append with rotary positions
// (append_kernel) and attention of single new tokens (attend_kernel).
#include <cuda_runtime.h>
#include <math.h>
#include <new>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "kv_paged.h"
#include "pk_quant.cuh"

namespace pk {
namespace kvp {

// x / d for 0 <= x < 2^31 by one multiplication: with 2^s >= d and
// m = ceil(2^(31+s) / d) < 2^32 + 1, x m / 2^(31+s) exceeds x / d by less
// than x 2^s / (d 2^(31+s)) < 1 / d.
struct Div {
    uint64_t m;
    uint32_t d;
    int s;
};
__host__ inline Div make_div(uint32_t d)
{
    Div v;
    v.d = d;
    v.s = 0;
    while (((uint64_t)1 << v.s) < d) v.s++;
    v.m = (((uint64_t)1 << (31 + v.s)) + d - 1) / d;
    v.s += 31;
    return v;
}
__host__ __device__ __forceinline__ int div_by(const Div &v, int x)
{
    return (int)(((uint64_t)(uint32_t)x * v.m) >> v.s);
}

// What the kernels know of a handle's cache.
struct Cache {
    Div page;  // page_tokens
    int n_pages, max_blocks;
    uint64_t page_stride, token_stride, head_stride;
};

// ------------------------------------------------------------------ //
// map                                                                //
// ------------------------------------------------------------------ //

constexpr int MAP_THREADS = 256;

struct MapArgs {
    const int *len, *start, *end;
    int n;
    int *table, *free_pages;
    const int *n_free;
    int *n_free_out;
    int max_rows;
    int *row_request, *row_pos, *row_slot, *row0;
    Cache c;
    unsigned *arrived;  // CTAs that have read *n_free; wraps to 0 by itself
    int *err;
};

// The largest i with p[i] <= x, for p ascending, p[0] = 0, 0 <= x < p[n]
// (the request of row, push or pop x in an exclusive prefix sum).
__host__ __device__ __forceinline__ int find_request(const int *p, int n, int x)
{
    int lo = 0, hi = n;  // p[lo] <= x < p[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p[mid] <= x) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    return lo;
}

// Pages that hold x tokens.
__host__ __device__ __forceinline__ int pages_of(const Div &page, int x)
{
    return x > 0 ? div_by(page, x - 1) + 1 : 0;
}

// Every CTA makes the three exclusive prefix sums over the requests (rows,
// pages pushed, pages popped) for itself in shared memory and then takes its
// share of the pushes, pops and rows, so nothing waits for another CTA. A
// popped page that this same call pushes is read from where its pusher reads
// it, the old table entry; a new block's page that a row needs is looked up
// like the pop that writes it. *n_free is replaced by the last CTA to have
// read it.
__global__ void __launch_bounds__(MAP_THREADS) map_kernel(const MapArgs a)
{
    extern __shared__ int sums[];  // [3][n + 1]
    __shared__ long long wsum[3][MAP_THREADS / 32];
    __shared__ int any_bad, had_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n;
    int *rows = sums, *push = sums + (n + 1), *pop = sums + 2 * (n + 1);
    if (tid == 0) {
        any_bad = 0;
        had_s = *a.n_free;
    }
    __syncthreads();
    const long long most = (long long)a.c.max_blocks * a.c.page.d;
    const int per = (n + MAP_THREADS - 1) / MAP_THREADS, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    long long s[3] = {0, 0, 0};
    bool bad = false;
    for (int i = i0; i < i1; i++) {
        const int len = a.len[i], st = a.start[i], en = a.end[i];
        if (st < 0 || st > len || en < st || en > most || len > most) {
            bad = true;
            continue;
        }
        const int d = pages_of(a.c.page, en) - pages_of(a.c.page, len);
        s[0] += en - st;
        s[1] += max(0, -d);
        s[2] += max(0, d);
    }
    if (bad) any_bad = 1;
    long long e[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {
        long long v = s[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xFFFFFFFFu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) wsum[k][warp] = v;
        e[k] = v - s[k];
    }
    __syncthreads();
    long long tot[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {
        long long t = 0;
        for (int w = 0; w < MAP_THREADS / 32; w++) {
            if (w == warp) e[k] += t;
            t += wsum[k][w];
        }
        tot[k] = t;
    }
    const int had = had_s;
    int code = 0;
    if (any_bad || had < 0 || had > a.c.n_pages) {
        code = KV_PAGED_BAD_LENGTH;
    } else {
        if (tot[0] > a.max_rows) code |= KV_PAGED_NO_ROWS;
        if (tot[2] > had + tot[1]) {
            code |= KV_PAGED_NO_PAGES;
        } else if (had + tot[1] - tot[2] > a.c.n_pages) {
            code |= KV_PAGED_BAD_LENGTH;  // more pages given back than the pool has
        }
    }
    const int n_rows = code ? 0 : (int)tot[0], n_push = code ? 0 : (int)tot[1], n_pop = code ? 0 : (int)tot[2];
    const int top = had + n_push;  // the stack's height between the pushes and the pops
    if (!code) {
        for (int i = i0; i < i1; i++) {
            const int st = a.start[i], en = a.end[i];
            const int d = pages_of(a.c.page, en) - pages_of(a.c.page, a.len[i]);
            rows[i] = (int)e[0];
            push[i] = (int)e[1];
            pop[i] = (int)e[2];
            e[0] += en - st;
            e[1] += max(0, -d);
            e[2] += max(0, d);
        }
        if (tid == 0) {
            rows[n] = n_rows;
            push[n] = n_push;
            pop[n] = n_pop;
        }
    }
    __syncthreads();
    // the page of push `x`, where its request still holds it
    auto pushed = [&](int x) {
        const int i = find_request(push, n, x);
        return a.table[(size_t)i * a.c.max_blocks + pages_of(a.c.page, a.end[i]) + (x - push[i])];
    };
    // the page that pop `x` takes
    auto popped = [&](int x) {
        const int p = top - 1 - x;
        return p >= had ? pushed(p - had) : a.free_pages[p];
    };
    const int gid = blockIdx.x * MAP_THREADS + tid, gsz = gridDim.x * MAP_THREADS;
    int found = code;
    if (blockIdx.x == 0) {
        for (int i = tid; i <= n; i += MAP_THREADS) a.row0[i] = code ? 0 : rows[i];
    }
    for (int x = gid; x < top - n_pop - had; x += gsz) {
        const int p = pushed(x);
        if (p < 0 || p >= a.c.n_pages) found |= KV_PAGED_BAD_PAGE;
        a.free_pages[had + x] = p;
    }
    for (int x = gid; x < n_pop; x += gsz) {
        const int i = find_request(pop, n, x), p = popped(x);
        if (p < 0 || p >= a.c.n_pages) found |= KV_PAGED_BAD_PAGE;
        a.table[(size_t)i * a.c.max_blocks + pages_of(a.c.page, a.len[i]) + (x - pop[i])] = p;
    }
    for (int r = gid; r < a.max_rows; r += gsz) {
        int req = -1, pos = -1, slot = -1;
        if (r < n_rows) {
            req = find_request(rows, n, r);
            pos = a.start[req] + (r - rows[req]);
            const int blk = div_by(a.c.page, pos), held = pages_of(a.c.page, a.len[req]);
            const int p = blk < held ? a.table[(size_t)req * a.c.max_blocks + blk] : popped(pop[req] + blk - held);
            if (p < 0 || p >= a.c.n_pages) {
                found |= KV_PAGED_BAD_PAGE;
            } else {
                slot = p * (int)a.c.page.d + (pos - blk * (int)a.c.page.d);
            }
        }
        a.row_request[r] = req;
        a.row_pos[r] = pos;
        a.row_slot[r] = slot;
    }
    if (found) atomicOr(a.err, found);
    if (tid == 0) {
        bool last = true;
        if (gridDim.x > 1) {
            __threadfence();  // the read of *n_free above comes before this arrival
            last = atomicInc(a.arrived, gridDim.x - 1) == gridDim.x - 1;
        }
        if (last) *a.n_free_out = top - n_pop;
    }
}

// ------------------------------------------------------------------ //
// append                                                             //
// ------------------------------------------------------------------ //

struct AppendArgs {
    const float *q, *k, *v;
    const int *row_pos, *row_slot;
    float *q_out;
    void *k_pool, *v_pool;
    const float *rope_cs;
    int rope_dim, rope_len, heads, kv_heads, hs;
    uint64_t q_stride, kv_stride, q_out_stride;
    Cache c;
    int *err;
};

template <typename KV>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a)
{
    const int r = blockIdx.x, slot = a.row_slot[r], pos = a.row_pos[r];
    if (slot < 0) return;
    if (slot >= a.c.n_pages * (int)a.c.page.d || (a.rope_dim > 0 && (pos < 0 || pos >= a.rope_len))) {
        if (threadIdx.x == 0) atomicOr(a.err, KV_PAGED_BAD_ROW);
        return;
    }
    const int page = div_by(a.c.page, slot), place = slot - page * (int)a.c.page.d;
    const float *rope = a.rope_cs + (size_t)pos * a.rope_dim;
    KV *kp = static_cast<KV *>(a.k_pool) + page * a.c.page_stride + place * a.c.token_stride;
    KV *vp = static_cast<KV *>(a.v_pool) + page * a.c.page_stride + place * a.c.token_stride;
    auto turn = [&](const float *x, int d, float &x0, float &x1) {
        x0 = x[0];
        x1 = x[1];
        if (d < a.rope_dim) {
            const float c = rope[d], sn = rope[d + 1];
            const float t = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, sn));
            x1 = __fadd_rn(__fmul_rn(x0, sn), __fmul_rn(x1, c));
            x0 = t;
        }
    };
    if (a.q != nullptr) {
        for (int p = threadIdx.x; p < a.heads * a.hs / 2; p += blockDim.x) {
            float x0, x1;
            turn(a.q + r * a.q_stride + 2 * p, 2 * p % a.hs, x0, x1);
            float *o = a.q_out + r * a.q_out_stride + 2 * p;
            o[0] = x0;
            o[1] = x1;
        }
    }
    for (int p = threadIdx.x; p < a.kv_heads * a.hs / 2; p += blockDim.x) {
        const int h = 2 * p / a.hs, d = 2 * p - h * a.hs;
        float x0, x1;
        turn(a.k + r * a.kv_stride + 2 * p, d, x0, x1);
        kv_store(kp, h * a.c.head_stride + d, x0);
        kv_store(kp, h * a.c.head_stride + d + 1, x1);
        const float *v = a.v + r * a.kv_stride + 2 * p;
        kv_store(vp, h * a.c.head_stride + d, v[0]);
        kv_store(vp, h * a.c.head_stride + d + 1, v[1]);
    }
}

// ------------------------------------------------------------------ //
// attend                                                             //
// ------------------------------------------------------------------ //

constexpr int ATT_WARPS = 4;

struct AttendArgs {
    const float *q;
    const void *k_pool, *v_pool;
    const int *table, *row_request, *row_pos;
    int n, n_requests, heads, kv_heads, hs;
    float scale;
    float *out;
    uint64_t q_stride;
    Cache c;
    int *err;
};

__device__ __forceinline__ float kv_get(const float *p)
{
    return *p;
}
__device__ __forceinline__ float kv_get(const __half *p)
{
    return __half2float(*p);
}

// One CTA per (row, query head). Warp w takes tokens w, w + ATT_WARPS, ...:
// its lanes share the channels of a token's key, and keep a running maximum
// m, sum l and weighted values o; the warps' are joined at the end.
template <typename KV>
__global__ void __launch_bounds__(32 * ATT_WARPS) attend_kernel(const AttendArgs a)
{
    __shared__ float part[ATT_WARPS][256 + 2];
    const int r = blockIdx.y, h = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int req = a.row_request[r];
    if (req < 0) return;
    int last = a.row_pos[r];
    const int cap = min((long long)a.c.max_blocks * a.c.page.d, 0x7FFFFFFFll);
    if (req >= a.n_requests) {
        if (threadIdx.x == 0) atomicOr(a.err, KV_PAGED_BAD_ROW);
        return;
    }
    if (last < -1 || last >= cap) {
        if (threadIdx.x == 0) atomicOr(a.err, KV_PAGED_BAD_ROW);
        last = last < 0 ? -1 : cap - 1;
    }
    const float *q = a.q + r * a.q_stride + (size_t)h * a.hs;
    const size_t head = (size_t)(h / (a.heads / a.kv_heads)) * a.c.head_stride;
    float qv[8], o[8], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        qv[j] = lane + 32 * j < a.hs ? q[lane + 32 * j] : 0.0f;
        o[j] = 0.0f;
    }
    for (int t = warp; t <= last; t += ATT_WARPS) {
        const int blk = div_by(a.c.page, t), p = a.table[(size_t)req * a.c.max_blocks + blk];
        if (p < 0 || p >= a.c.n_pages) {
            if (lane == 0) atomicOr(a.err, KV_PAGED_BAD_PAGE);
            continue;
        }
        const size_t at = p * a.c.page_stride + (t - blk * (int)a.c.page.d) * a.c.token_stride + head;
        const KV *k = static_cast<const KV *>(a.k_pool) + at, *v = static_cast<const KV *>(a.v_pool) + at;
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (lane + 32 * j < a.hs) s = fmaf(qv[j], kv_get(k + lane + 32 * j), s);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
        s *= a.scale;
        const float mn = fmaxf(m, s), f = expf(m - mn), e = expf(s - mn);
        l = l * f + e;
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] = o[j] * f + (lane + 32 * j < a.hs ? e * kv_get(v + lane + 32 * j) : 0.0f);
        m = mn;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) part[warp][lane + 32 * j] = o[j];
    if (lane == 0) {
        part[warp][256] = m;
        part[warp][257] = l;
    }
    __syncthreads();
    float mt = -INFINITY, lt = 0.0f;
    for (int w = 0; w < ATT_WARPS; w++) mt = fmaxf(mt, part[w][256]);
    for (int w = 0; w < ATT_WARPS; w++)
        if (part[w][257] > 0.0f) lt += part[w][257] * expf(part[w][256] - mt);
    for (int d = threadIdx.x; d < a.hs; d += blockDim.x) {
        float s = 0.0f;
        for (int w = 0; w < ATT_WARPS; w++)
            if (part[w][257] > 0.0f) s += part[w][d] * expf(part[w][256] - mt);
        a.out[((size_t)r * a.heads + h) * a.hs + d] = lt > 0.0f ? s / lt : 0.0f;
    }
}

}  // namespace kvp
}  // namespace pk

using namespace pk;

struct KvPaged {
    KvPagedShape s;
    kvp::Cache c;
    int device, sms;
    unsigned *arrived;  // device: map's arrivals
    int *err;           // device: error bits
    char msg[256];
};

static const char *shape_fault(KvPagedShape &s)
{
    if (s.type != 0 && s.type != 1) return "The cache's type must be 0 (F32) or 1 (F16).";
    if (s.n_heads < 1 || s.n_kv_heads < 1 || s.n_heads % s.n_kv_heads || s.n_heads > 65535)
        return "The query heads must be a multiple of the key-value heads, at most 65535.";
    if (s.head_size < 8 || s.head_size > 256 || s.head_size % 8) return "The head size must be a multiple of 8, 8 to 256.";
    if (s.page_tokens < 1 || s.n_pages < 1 || (long long)s.page_tokens * s.n_pages > 0x7FFFFFFFll)
        return "Pages and page size must be positive, with less than 2^31 tokens in all.";
    if (s.max_requests < 1 || s.max_requests > KV_PAGED_MAX_REQUESTS)
        return "The block table takes 1 to 4096 requests.";
    if (s.max_blocks < 1 || (long long)s.max_blocks * s.page_tokens > 0x7FFFFFFFll)
        return "A request's blocks must be positive, with less than 2^31 tokens in all.";
    const uint64_t hs = (uint64_t)s.head_size, unit = s.type == 1 ? 8 : 4, big = (uint64_t)1 << 40;
    if (s.page_stride == 0 && s.token_stride == 0 && s.head_stride == 0) {
        s.head_stride = hs;
        s.token_stride = hs * s.n_kv_heads;
        s.page_stride = s.token_stride * s.page_tokens;
    }
    if (s.page_stride % unit || s.token_stride % unit || s.head_stride % unit)
        return "Page, token and head strides must be multiples of 16 bytes.";
    // pages, tokens and heads must not overlap: each axis, from the shortest
    // stride up, steps over all of the ones below it
    uint64_t st[3] = {s.page_stride, s.token_stride, s.head_stride};
    uint64_t cnt[3] = {(uint64_t)s.n_pages, (uint64_t)s.page_tokens, (uint64_t)s.n_kv_heads};
    for (int i = 0; i < 3; i++)
        for (int j = i + 1; j < 3; j++)
            if (st[j] < st[i] || (st[j] == st[i] && cnt[j] < cnt[i])) {
                const uint64_t a = st[i], b = cnt[i];
                st[i] = st[j], cnt[i] = cnt[j], st[j] = a, cnt[j] = b;
            }
    uint64_t below = hs;
    for (int i = 0; i < 3; i++) {
        if (cnt[i] == 1) continue;
        if (st[i] < below) return "Page, token and head strides overlap.";
        if (st[i] > big) return "Page, token or head stride too large.";
        below += st[i] * (cnt[i] - 1);
    }
    return nullptr;
}

// Makes the handle's device current for a call, and the old one again after it.
struct OnDevice {
    int was;
    bool moved, ok;
    explicit OnDevice(int device) : was(0), moved(false), ok(true)
    {
        ok = cudaGetDevice(&was) == cudaSuccess;
        if (ok && was != device) {
            ok = cudaSetDevice(device) == cudaSuccess;
            moved = ok;
        }
    }
    ~OnDevice()
    {
        if (moved) cudaSetDevice(was);
    }
};

static int refuse(KvPaged *kv, const char *why)
{
    snprintf(kv->msg, sizeof(kv->msg), "%s", why);
    return 0;
}

static int launched(KvPaged *kv, const char *what)
{
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return 1;
    snprintf(kv->msg, sizeof(kv->msg), "CUDA %s failed: %s", what, cudaGetErrorString(e));
    return 0;
}

static bool off16(const void *p)
{
    return ((uintptr_t)p & 15) != 0;
}

extern "C" KvPaged *kv_paged_open(const KvPagedShape *shape, int device, char *error, size_t cap)
{
    auto fail = [&](const char *why) -> KvPaged * {
        if (error && cap) snprintf(error, cap, "%s", why);
        return nullptr;
    };
    if (error && cap) error[0] = '\0';
    if (shape == nullptr) return fail("No cache shape given.");
    KvPagedShape s = *shape;
    if (const char *why = shape_fault(s)) return fail(why);
    if (device < -1) return fail("Invalid device.");
    KvPaged *kv = new (std::nothrow) KvPaged();
    if (kv == nullptr) return fail("Out of memory.");
    kv->s = s;
    kv->device = device;
    kv->c.page = kvp::make_div((uint32_t)s.page_tokens);
    kv->c.n_pages = s.n_pages;
    kv->c.max_blocks = s.max_blocks;
    kv->c.page_stride = s.page_stride;
    kv->c.token_stride = s.token_stride;
    kv->c.head_stride = s.head_stride;
    if (device < 0) return kv;
    int count = 0;
    cudaError_t e = cudaGetDeviceCount(&count);
    if (e == cudaSuccess && device >= count) e = cudaErrorInvalidDevice;
    if (e == cudaSuccess) {
        OnDevice on(device);
        e = on.ok ? cudaDeviceGetAttribute(&kv->sms, cudaDevAttrMultiProcessorCount, device) : cudaErrorInvalidDevice;
        if (e == cudaSuccess) e = cudaMalloc(&kv->arrived, 256);
        if (e == cudaSuccess) e = cudaMemset(kv->arrived, 0, 256);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kvp::map_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     3 * (KV_PAGED_MAX_REQUESTS + 1) * 4);
        if (e == cudaSuccess) e = cudaDeviceSynchronize();
    }
    if (e != cudaSuccess) {
        if (error && cap) snprintf(error, cap, "CUDA setup of the paged cache failed: %s", cudaGetErrorString(e));
        cudaGetLastError();
        kv_paged_close(kv);
        return nullptr;
    }
    kv->err = (int *)(kv->arrived + 32);
    return kv;
}

extern "C" void kv_paged_close(KvPaged *kv)
{
    if (kv == nullptr) return;
    if (kv->arrived) {
        OnDevice on(kv->device);
        cudaFree(kv->arrived);
    }
    delete kv;
}

extern "C" const char *kv_paged_last_error(const KvPaged *kv)
{
    return kv ? kv->msg : "";
}

extern "C" int kv_paged_error(KvPaged *kv)
{
    if (kv == nullptr || kv->device < 0) return -1;
    OnDevice on(kv->device);
    int v = 0;
    if (!on.ok || cudaDeviceSynchronize() != cudaSuccess ||
        cudaMemcpy(&v, kv->err, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess ||
        (v != 0 && cudaMemset(kv->err, 0, sizeof(int)) != cudaSuccess)) {
        cudaGetLastError();
        return -1;
    }
    return v;
}

extern "C" int kv_paged_map(KvPaged *kv, const int *len, const int *start, const int *end, int n, int *table,
                            int *free_pages, const int *n_free, int *n_free_out, int max_rows, int *row_request,
                            int *row_pos, int *row_slot, int *row0, void *stream)
{
    if (kv == nullptr) return 0;
    if (!len || !start || !end || !table || !free_pages || !n_free || !n_free_out || !row0)
        return refuse(kv, "map: a pointer is NULL.");
    if (n < 1 || n > kv->s.max_requests) return refuse(kv, "map: requests outside 1 .. max_requests.");
    if (max_rows < 0 || (max_rows > 0 && (!row_request || !row_pos || !row_slot)))
        return refuse(kv, "map: no room for the rows.");
    if (kv->device < 0) return refuse(kv, "The handle has no device.");
    OnDevice on(kv->device);
    if (!on.ok) return refuse(kv, "CUDA device cannot be used.");
    kvp::MapArgs a = {len, start, end, n, table, free_pages, n_free, n_free_out, max_rows, row_request, row_pos,
                      row_slot, row0, kv->c, kv->arrived, kv->err};
    int grid = (max_rows + 4 * kvp::MAP_THREADS - 1) / (4 * kvp::MAP_THREADS);
    if (grid > 2 * kv->sms) grid = 2 * kv->sms;
    if (grid < 1) grid = 1;
    cudaGetLastError();
    kvp::map_kernel<<<grid, kvp::MAP_THREADS, 3 * (n + 1) * 4, (cudaStream_t)stream>>>(a);
    return launched(kv, "map");
}

extern "C" int kv_paged_append(KvPaged *kv, const float *q, const float *k, const float *v, const int *row_pos,
                               const int *row_slot, int n, float *q_out, void *k_pool, void *v_pool,
                               const float *rope_cs, int rope_dim, int rope_len, uint64_t q_stride,
                               uint64_t kv_stride, void *stream)
{
    if (kv == nullptr) return 0;
    const KvPagedShape &s = kv->s;
    const uint64_t qd = (uint64_t)s.n_heads * s.head_size, kvd = (uint64_t)s.n_kv_heads * s.head_size;
    if (!k || !v || !row_pos || !row_slot || !k_pool || !v_pool || !q != !q_out)
        return refuse(kv, "append: a pointer is NULL.");
    if (n < 0) return refuse(kv, "append: negative row count.");
    if (rope_dim < 0 || rope_dim > s.head_size || rope_dim % 2 || (rope_dim > 0 && (!rope_cs || rope_len < 1)))
        return refuse(kv, "append: the rotary dimension must be even, at most the head size, with a table.");
    if (q_stride == 0) q_stride = qd;
    if (kv_stride == 0) kv_stride = kvd;
    if (q_stride < qd || kv_stride < kvd || q_stride % 4 || kv_stride % 4)
        return refuse(kv, "append: a row stride is too small or no multiple of 4.");
    if (off16(q) || off16(k) || off16(v) || off16(q_out) || off16(k_pool) || off16(v_pool) ||
        ((uintptr_t)rope_cs & 7))
        return refuse(kv, "append: a pointer is not on 16 bytes (the rotary table: 8).");
    if (kv->device < 0) return refuse(kv, "The handle has no device.");
    if (n == 0) return 1;
    OnDevice on(kv->device);
    if (!on.ok) return refuse(kv, "CUDA device cannot be used.");
    kvp::AppendArgs a = {q, k, v, row_pos, row_slot, q_out, k_pool, v_pool, rope_cs, rope_dim, rope_len, s.n_heads,
                         s.n_kv_heads, s.head_size, q_stride, kv_stride, q_out == q ? q_stride : qd, kv->c, kv->err};
    cudaGetLastError();
    if (s.type == 1) {
        kvp::append_kernel<__half><<<n, 256, 0, (cudaStream_t)stream>>>(a);
    } else {
        kvp::append_kernel<float><<<n, 256, 0, (cudaStream_t)stream>>>(a);
    }
    return launched(kv, "append");
}

extern "C" int kv_paged_attend(KvPaged *kv, const float *q, const void *k_pool, const void *v_pool, const int *table,
                               int n_requests, const int *row_request, const int *row_pos, int n, float scale,
                               float *out, uint64_t q_stride, void *stream)
{
    if (kv == nullptr) return 0;
    const KvPagedShape &s = kv->s;
    const uint64_t qd = (uint64_t)s.n_heads * s.head_size;
    if (!q || !k_pool || !v_pool || !table || !row_request || !row_pos || !out)
        return refuse(kv, "attend: a pointer is NULL.");
    if (n < 0 || n > 65535) return refuse(kv, "attend: rows outside 0 .. 65535.");
    if (n_requests < 1 || n_requests > s.max_requests)
        return refuse(kv, "attend: requests outside 1 .. max_requests.");
    if (!isfinite(scale)) return refuse(kv, "attend: the scale is not finite.");
    if (q_stride == 0) q_stride = qd;
    if (q_stride < qd || q_stride % 4) return refuse(kv, "attend: the row stride is too small or no multiple of 4.");
    if (off16(q) || off16(k_pool) || off16(v_pool) || off16(out))
        return refuse(kv, "attend: a pointer is not on 16 bytes.");
    const char *q0 = (const char *)q, *o0 = (const char *)out;
    if (n > 0 && q0 < o0 + (size_t)n * qd * 4 && o0 < q0 + ((size_t)(n - 1) * q_stride + qd) * 4)
        return refuse(kv, "attend: out overlaps q.");
    if (kv->device < 0) return refuse(kv, "The handle has no device.");
    if (n == 0) return 1;
    OnDevice on(kv->device);
    if (!on.ok) return refuse(kv, "CUDA device cannot be used.");
    kvp::AttendArgs a = {q, k_pool, v_pool, table, row_request, row_pos, n, n_requests, s.n_heads, s.n_kv_heads,
                         s.head_size, scale, out, q_stride, kv->c, kv->err};
    cudaGetLastError();
    const dim3 grid(s.n_heads, n);
    if (s.type == 1) {
        kvp::attend_kernel<__half><<<grid, 32 * kvp::ATT_WARPS, 0, (cudaStream_t)stream>>>(a);
    } else {
        kvp::attend_kernel<float><<<grid, 32 * kvp::ATT_WARPS, 0, (cudaStream_t)stream>>>(a);
    }
    return launched(kv, "attend");
}
