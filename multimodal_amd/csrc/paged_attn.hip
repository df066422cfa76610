// Attention of one token over a paged key-value cache, with its append, and the storing of runs (include/mmhip.h).
#include "paged.h"

struct PagedP {
    const void* q; const void* kn; const void* vn; void* kpool; void* vpool; void* o; float* w; const int* lengths; const int* positions;
    const float* cos_t; const float* sin_t; float* sc; PagedMap map;
    int B, H, Hkv, G, d, rot, n_pos; long ld_q, ld_k, ld_v; float scale;
};

__device__ __forceinline__ int paged_pos(const PagedP& p, int b) {
    const int n = p.lengths[b];
    const int pos = p.positions ? p.positions[b] : (p.kn ? n : n - 1);
    return min(max(pos, 0), p.n_pos - 1);
}
// element c of a head, rotated at table row `cs` / `sn`
template <typename T> __device__ __forceinline__ float rotated(const T* x, int c, int rot, const float* cs, const float* sn) {
    const int half = rot >> 1;
    const float a = to_f(x[c]);
    if (c >= rot) return a;
    const int i = c < half ? c : c - half;
    const float o = to_f(x[c < half ? c + half : c - half]);
    return c < half ? a * cs[i] - o * sn[i] : a * cs[i] + o * sn[i];
}

template <typename T> __global__ __launch_bounds__(64) void paged_append_k(const PagedP p) {
    const int b = blockIdx.x, h = blockIdx.y, n = p.lengths[b];
    if (n < 0) return;
    const long row = p.map.row(b, h, n);
    if (row < 0) return;
    const long t = (long)paged_pos(p, b) * (p.rot >> 1);
    const T* k = (const T*)p.kn + (long)b * p.ld_k + (long)h * p.d;
    const T* v = (const T*)p.vn + (long)b * p.ld_v + (long)h * p.d;
    for (int c = threadIdx.x; c < p.d; c += 64) {
        ((T*)p.kpool)[row * p.d + c] = from_f<T>(rotated(k, c, p.rot, p.cos_t + t, p.sin_t + t));
        ((T*)p.vpool)[row * p.d + c] = v[c];
    }
    if (p.w && threadIdx.x == 0) p.w[row] = 0.f;
}

__device__ __forceinline__ float block_max(float v, float* red) {
    for (int i = 1; i < 64; i <<= 1) v = fmaxf(v, __shfl_xor(v, i));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

template <typename T> __global__ __launch_bounds__(256) void paged_attn_k(const PagedP p, int stable) {
    __shared__ float qs[512], red[4];
    const int b = blockIdx.x, h = blockIdx.y, hk = h / p.G;
    const int n = min(p.lengths[b] < 0 ? 0 : p.lengths[b] + (p.kn ? 1 : 0), p.map.capacity());
    const long t = (long)paged_pos(p, b) * (p.rot >> 1);
    float* sc = p.sc + ((long)b * p.H + h) * p.map.capacity();
    for (int c = threadIdx.x; c < p.d; c += 256)
        qs[c] = rotated((const T*)p.q + (long)b * p.ld_q + (long)h * p.d, c, p.rot, p.cos_t + t, p.sin_t + t);
    __syncthreads();
    float m = -INFINITY;
    for (int s = threadIdx.x; s < n; s += 256) {
        const long row = p.map.row(b, hk, s);
        float x = 0.f;
        if (row >= 0) {
            for (int c = 0; c < p.d; c++) x = fmaf(qs[c], to_f(((const T*)p.kpool)[row * p.d + c]), x);
            x *= p.scale;
            m = fmaxf(m, x);
        }
        sc[s] = x;
    }
    m = block_max(m, red);
    if (m == -INFINITY) m = 0.f;
    float l = 0.f;
    for (int s = threadIdx.x; s < n; s += 256) {
        const bool there = p.map.row(b, hk, s) >= 0;
        const float x = sc[s];
        const float e = !there ? 0.f : stable ? (x < 0.f ? 1.f / (1.f - x + 1e-9f) : x + 1.f) : expf(x - m);
        sc[s] = e;
        l += e;
    }
    __syncthreads();
    l = block_sum<4>(l, red);
    const float inv = stable ? 1.f / fmaxf(l, 1e-9f) : l == 0.f ? 0.f : 1.f / l;
    __threadfence_block();
    __syncthreads();
    for (int c = threadIdx.x; c < p.d; c += 256) {
        float a = 0.f;
        for (int s = 0; s < n; s++) {
            const long row = p.map.row(b, hk, s);
            if (row >= 0) a = fmaf(sc[s], to_f(((const T*)p.vpool)[row * p.d + c]), a);
        }
        ((T*)p.o)[((long)b * p.H + h) * p.d + c] = from_f<T>(a * inv);
    }
    __syncthreads();
    for (int s = threadIdx.x; s < n; s += 256) sc[s] *= inv;
}
__global__ __launch_bounds__(256) void paged_weights_k(const PagedP p) {
    const int b = blockIdx.x, hk = blockIdx.y;
    const int n = min(p.lengths[b] < 0 ? 0 : p.lengths[b] + (p.kn ? 1 : 0), p.map.capacity());
    for (int s = threadIdx.x; s < n; s += 256) {
        const long row = p.map.row(b, hk, s);
        if (row < 0) continue;
        float a = 0.f;
        for (int g = 0; g < p.G; g++) a += p.sc[((long)b * p.H + hk * p.G + g) * p.map.capacity() + s];
        p.w[row] += a;
    }
}

extern "C" size_t mm_paged_decode_attn_workspace(const mm_paged_attn_args* a) {
    if (!a || a->B <= 0 || a->H <= 0 || a->width <= 0 || a->page <= 0) return 0;
    return (size_t)a->B * a->H * a->width * a->page * sizeof(float);
}

extern "C" int mm_paged_decode_attn(const mm_paged_attn_args* a, void* stream) {
    MM_CHECK(a, "paged_decode_attn: null arguments");
    int rc = paged_check("paged_decode_attn", a->kpool, a->vpool, a->page_table, a->B, a->Hkv, a->d, a->page, a->n_pages, a->width, a->ld_table, a->dtype);
    if (rc != MM_OK) return rc;
    if (a->B == 0) return MM_OK;
    MM_CHECK(a->q && a->o && a->lengths && (!a->k_new == !a->v_new), "paged_decode_attn: null pointer");
    MM_CHECK(a->H > 0 && a->H <= 65535 && a->H % a->Hkv == 0, "paged_decode_attn: %lld query heads over %lld KV heads", (long long)a->H, (long long)a->Hkv);
    MM_CHECK(a->rot >= 0 && a->rot <= a->d && a->rot % 2 == 0 && (a->rot == 0 || (a->cos_t && a->sin_t && a->n_pos > 0)), "paged_decode_attn: bad rot/tables");
    MM_CHECK(a->ld_q >= 0 && a->ld_k >= 0 && a->ld_v >= 0, "paged_decode_attn: negative row stride");
    MM_CHECK(a->mode == MM_ATTN_SOFTMAX || a->mode == MM_ATTN_STABLEMAX, "paged_decode_attn: bad mode %d", a->mode);
    MM_CHECK(a->workspace && a->workspace_bytes >= mm_paged_decode_attn_workspace(a), "paged_decode_attn: workspace too small");
    hipStream_t st = (hipStream_t)stream;
    PagedP p{};
    p.q = a->q; p.kn = a->k_new; p.vn = a->v_new; p.kpool = a->kpool; p.vpool = a->vpool; p.o = a->o; p.w = a->weights;
    p.lengths = a->lengths; p.positions = a->positions; p.cos_t = a->cos_t; p.sin_t = a->sin_t; p.sc = (float*)a->workspace;
    p.map = {a->page_table, (long)a->ld_table, (int)a->width, paged_shift(a->page), (int)a->n_pages, (int)a->Hkv};
    p.B = (int)a->B; p.H = (int)a->H; p.Hkv = (int)a->Hkv; p.G = (int)(a->H / a->Hkv); p.d = (int)a->d; p.rot = (int)a->rot;
    p.n_pos = a->rot ? (int)a->n_pos : 1; p.ld_q = a->ld_q; p.ld_k = a->ld_k; p.ld_v = a->ld_v; p.scale = (float)(1.0 / sqrt((double)a->d));
    const dim3 gk((unsigned)a->B, (unsigned)a->Hkv), gh((unsigned)a->B, (unsigned)a->H);
    const bool bf = a->dtype == MM_BF16;
    if (a->k_new) {
        if (bf) hipLaunchKernelGGL(paged_append_k<bf16>, gk, dim3(64), 0, st, p);
        else hipLaunchKernelGGL(paged_append_k<float>, gk, dim3(64), 0, st, p);
        MM_LAUNCH_CHECK();
    }
    if (bf) hipLaunchKernelGGL(paged_attn_k<bf16>, gh, dim3(256), 0, st, p, a->mode);
    else hipLaunchKernelGGL(paged_attn_k<float>, gh, dim3(256), 0, st, p, a->mode);
    MM_LAUNCH_CHECK();
    if (a->weights) {
        hipLaunchKernelGGL(paged_weights_k, gk, dim3(256), 0, st, p);
        MM_LAUNCH_CHECK();
    }
    return MM_OK;
}

// ------------------------------------------------------------------------------------------------ runs of keys and values
struct FillP {
    const void* k; const void* v; void* kpool; void* vpool; float* w; const int* start; const int* counts; const int* positions;
    const float* cos_t; const float* sin_t; PagedMap map; int S, Hkv, d, rot, n_pos; long ld_k, bs_k, ld_v, bs_v;
};
template <typename T> __global__ __launch_bounds__(256) void paged_fill_k(const FillP p) {
    const int b = blockIdx.y;
    const long idx = (long)blockIdx.x * 256 + threadIdx.x;              // over [S][Hkv][d]
    const int c = (int)(idx % p.d), h = (int)(idx / p.d % p.Hkv), s = (int)(idx / ((long)p.d * p.Hkv));
    const int st = p.start ? p.start[b] : 0, n = p.counts ? min(p.counts[b], p.S) : p.S;
    if (st < 0 || s >= n) return;
    const long row = p.map.row(b, h, st + s);
    if (row < 0) return;
    const long t = (long)min(max((p.positions ? p.positions[b] : st) + s, 0), p.n_pos - 1) * (p.rot >> 1);
    const T* k = (const T*)p.k + (long)b * p.bs_k + (long)s * p.ld_k + (long)h * p.d;
    ((T*)p.kpool)[row * p.d + c] = from_f<T>(rotated(k, c, p.rot, p.cos_t + t, p.sin_t + t));
    ((T*)p.vpool)[row * p.d + c] = ((const T*)p.v)[(long)b * p.bs_v + (long)s * p.ld_v + (long)h * p.d + c];
    if (p.w && c == 0) p.w[row] = 0.f;
}

extern "C" int mm_paged_cache_fill(const mm_paged_fill_args* a, void* stream) {
    MM_CHECK(a, "paged_cache_fill: null arguments");
    int rc = paged_check("paged_cache_fill", a->kpool, a->vpool, a->page_table, a->B, a->Hkv, a->d, a->page, a->n_pages, a->width, a->ld_table, a->dtype);
    if (rc != MM_OK) return rc;
    MM_CHECK(a->S >= 0 && a->S < (1LL << 30), "paged_cache_fill: S=%lld", (long long)a->S);
    if (a->B == 0 || a->S == 0) return MM_OK;
    MM_CHECK(a->k && a->v, "paged_cache_fill: null pointer");
    MM_CHECK(a->rot >= 0 && a->rot <= a->d && a->rot % 2 == 0 && (a->rot == 0 || (a->cos_t && a->sin_t && a->n_pos > 0)), "paged_cache_fill: bad rot/tables");
    MM_CHECK(a->ld_k >= 0 && a->ld_v >= 0 && a->bs_k >= 0 && a->bs_v >= 0, "paged_cache_fill: negative stride");
    FillP p{};
    p.k = a->k; p.v = a->v; p.kpool = a->kpool; p.vpool = a->vpool; p.w = a->weights; p.start = a->start; p.counts = a->counts; p.positions = a->positions;
    p.cos_t = a->cos_t; p.sin_t = a->sin_t; p.map = {a->page_table, (long)a->ld_table, (int)a->width, paged_shift(a->page), (int)a->n_pages, (int)a->Hkv};
    p.S = (int)a->S; p.Hkv = (int)a->Hkv; p.d = (int)a->d; p.rot = (int)a->rot; p.n_pos = a->rot ? (int)a->n_pos : 1;
    p.ld_k = a->ld_k; p.bs_k = a->bs_k; p.ld_v = a->ld_v; p.bs_v = a->bs_v;
    const int64_t per = a->S * a->Hkv * a->d;
    MM_CHECK(cdiv(per, 256) < (1LL << 31), "paged_cache_fill: too many tokens");
    const dim3 grid((unsigned)cdiv(per, 256), (unsigned)a->B);
    if (a->dtype == MM_BF16) hipLaunchKernelGGL(paged_fill_k<bf16>, grid, dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(paged_fill_k<float>, grid, dim3(256), 0, (hipStream_t)stream, p);
    MM_LAUNCH_CHECK();
    return MM_OK;
}
