// Eviction from a paged key-value cache by accumulated attention weight (include/mmhip.h).
#include "paged.h"

// Order of weights as unsigned integers: greater weight, greater key; NaN above everything, -0 = 0, a slot that does not exist lowest.
__device__ __forceinline__ unsigned weight_key(float x) {
    if (x != x) return 0xffffffffu;
    const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
struct EvictP {
    void* kpool; void* vpool; float* w; int* lengths; int* kept; PagedMap map; unsigned* keys; int d, es, budget, recent;
};
__device__ __forceinline__ void move_slot(const EvictP& p, long to, long from, int lane, int lanes) {
    if (to < 0 || from < 0) return;
    const int n4 = p.d * p.es / 4;                                     // d % 4 == 0: whole 4-byte words (8 in bf16)
    const unsigned* ks = (const unsigned*)p.kpool + from * n4; unsigned* kd = (unsigned*)p.kpool + to * n4;
    const unsigned* vs = (const unsigned*)p.vpool + from * n4; unsigned* vd = (unsigned*)p.vpool + to * n4;
    for (int i = lane; i < n4; i += lanes) { kd[i] = ks[i]; vd[i] = vs[i]; }
    if (lane == 0) p.w[to] = p.w[from];
}
// One workgroup per (row, KV head): rank every old slot by counting, list the moves, make them.
__global__ __launch_bounds__(256) void paged_evict_k(const EvictP p) {
    const int b = blockIdx.x, h = blockIdx.y, cap = p.map.capacity(), tid = threadIdx.x;
    const int n = min(p.lengths[b], cap);
    int* kept = p.kept + ((long)b * p.map.Hkv + h) * p.budget;
    if (n <= p.budget) {
        for (int j = tid; j < p.budget; j += 256) kept[j] = j < n ? j : -1;
        return;
    }
    const int A = p.budget - p.recent, old = n - p.recent;
    unsigned* key = p.keys + ((long)b * p.map.Hkv + h) * cap;
    for (int s = tid; s < old; s += 256) { const long r = p.map.row(b, h, s); key[s] = r < 0 ? 0u : weight_key(p.w[r]); }
    __syncthreads();
    for (int s = tid; s < A; s += 256) kept[s] = -2;
    __syncthreads();
    int* mark = (int*)key;                                             // becomes 1 for survivors behind the kept region (after all ranks)
    __shared__ int any;
    // ranks: survivors of the kept region say so in kept[]; those behind it are found again below by the same count
    for (int s = tid; s < old; s += 256) {
        int rank = 0;
        const unsigned mine = key[s];
        for (int o = 0; o < old; o++) rank += key[o] > mine || (key[o] == mine && o < s);
        if (s < A && rank < A) kept[s] = s;
    }
    __syncthreads();
    if (tid == 0) any = 0;
    __syncthreads();
    for (int s0 = A; s0 < old; s0 += 256) {                            // in order: the i-th survivor takes the i-th hole
        const int s = s0 + tid;
        int rank = old;
        if (s < old) {
            rank = 0;
            const unsigned mine = key[s];
            for (int o = 0; o < old; o++) rank += key[o] > mine || (key[o] == mine && o < s);
        }
        __shared__ int late[256];
        late[tid] = rank < A;
        __syncthreads();
        if (tid == 0)
            for (int i = 0; i < 256; i++)
                if (late[i]) {
                    while (kept[any] != -2) any++;
                    kept[any] = s0 + i;
                }
        __syncthreads();
    }
    (void)mark;
    const int wave = tid >> 6, lane = tid & 63;
    for (int j = wave; j < A; j += 4) if (kept[j] != j) move_slot(p, p.map.row(b, h, j), p.map.row(b, h, kept[j]), lane, 64);
    __threadfence_block();
    __syncthreads();
    for (int j = A; j < p.budget; j++) {                               // the newest slots: down by n - budget, in order
        move_slot(p, p.map.row(b, h, j), p.map.row(b, h, n - p.budget + j), tid, 256);
        if (tid == 0) kept[j] = n - p.budget + j;
        __threadfence_block();
        __syncthreads();
    }
}
__global__ void paged_lengths_k(int* lengths, int B, int budget, int cap) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < B && min(lengths[b], cap) > budget) lengths[b] = budget;
}

extern "C" size_t mm_paged_evict_workspace(int64_t B, int64_t Hkv, int64_t page, int64_t width, int64_t budget, int64_t recent) {
    (void)budget; (void)recent;
    return (B > 0 && Hkv > 0 && page > 0 && width > 0) ? (size_t)(B * Hkv * page * width) * sizeof(unsigned) : 0;
}
extern "C" int mm_paged_evict(void* kpool, void* vpool, float* weights, const int32_t* page_table, int32_t* lengths, int32_t* kept, int64_t B,
                              int64_t Hkv, int64_t d, int64_t page, int64_t n_pages, int64_t width, int64_t ld_table, int64_t budget,
                              int64_t recent, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = paged_check("paged_evict", kpool, vpool, page_table, B, Hkv, d, page, n_pages, width, ld_table, dtype);
    if (rc != MM_OK) return rc;
    MM_CHECK(budget > 0 && budget < (1LL << 30) && recent >= 0 && recent <= budget, "paged_evict: budget=%lld recent=%lld (0 <= recent <= budget, budget > 0)",
             (long long)budget, (long long)recent);
    if (B == 0) return MM_OK;
    MM_CHECK(weights && lengths && kept && workspace, "paged_evict: null pointer");
    MM_CHECK(workspace_bytes >= mm_paged_evict_workspace(B, Hkv, page, width, budget, recent), "paged_evict: workspace too small");
    EvictP p{};
    p.kpool = kpool; p.vpool = vpool; p.w = weights; p.lengths = lengths; p.kept = kept;
    p.map = {page_table, (long)ld_table, (int)width, paged_shift(page), (int)n_pages, (int)Hkv};
    p.keys = (unsigned*)workspace; p.d = (int)d; p.es = dtype == MM_BF16 ? 2 : 4; p.budget = (int)budget; p.recent = (int)recent;
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(paged_evict_k, dim3((unsigned)B, (unsigned)Hkv), dim3(256), 0, st, p);
    MM_LAUNCH_CHECK();
    hipLaunchKernelGGL(paged_lengths_k, dim3((unsigned)cdiv(B, 256)), dim3(256), 0, st, lengths, (int)B, (int)budget, (int)(width * page));
    MM_LAUNCH_CHECK();
    return MM_OK;
}
