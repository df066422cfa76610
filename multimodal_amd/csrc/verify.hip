// Drafted tokens against the target's probabilities (include/mmhip.h).
#include "common.h"

struct VerifyP {
    const int64_t* x; const float* p; const float* q; const float* u; const int* counts; int64_t* tokens; int* accepted;
    int K, V; long ld_x, bs_p, ld_p, bs_q, ld_q, ld_u;
};
// value of the final distribution at v: the residual of row a, or row a itself
__device__ __forceinline__ double rest(const VerifyP& p, const float* pr, const float* qr, int mode, int64_t x, int v) {
    double r = pr[v];
    if (mode == 1) r -= (double)qr[v];
    if (mode == 2 && v == x) r -= 1.0;
    return r > 0.0 ? r : 0.0;
}
__global__ __launch_bounds__(256) void verify_k(const VerifyP p) {
    __shared__ int acc;
    __shared__ double part[256];
    __shared__ int last[256];
    const int b = blockIdx.x, tid = threadIdx.x;
    const int n = p.counts ? min(max(p.counts[b], 0), p.K) : p.K;
    if (tid == 0) {
        int a = 0;
        for (; a < n; a++) {
            const int64_t x = p.x[b * p.ld_x + a];
            if (x < 0 || x >= p.V) break;
            const double q = p.q ? (double)p.q[b * p.bs_q + a * p.ld_q + x] : 1.0;
            if (!((double)p.u[b * p.ld_u + a] * q < (double)p.p[b * p.bs_p + a * p.ld_p + x])) break;
            p.tokens[(long)b * (p.K + 1) + a] = x;
        }
        acc = a;
        p.accepted[b] = a;
    }
    __syncthreads();
    const int a = acc, per = (p.V + 255) / 256, v0 = min(tid * per, p.V), v1 = min(v0 + per, p.V);
    const float* pr = p.p + b * p.bs_p + a * p.ld_p;
    const float* qr = p.q ? p.q + b * p.bs_q + a * p.ld_q : nullptr;
    const int64_t x = a < n ? p.x[b * p.ld_x + a] : -1;
    int mode = a < n ? (p.q ? 1 : 2) : 0;
    for (;;) {
        double s = 0.0;
        int l = -1;
        for (int v = v0; v < v1; v++) { const double r = rest(p, pr, qr, mode, x, v); s += r; if (r > 0.0) l = v; }
        part[tid] = s; last[tid] = l;
        __syncthreads();
        bool any = false;
        for (int i = 0; i < 256; i++) any |= last[i] >= 0;
        if (any || mode == 0) break;
        mode = 0;
        __syncthreads();
    }
    if (tid == 0) {
        double total = 0.0, before = 0.0;
        for (int i = 0; i < 256; i++) total += part[i];
        const double t = (double)p.u[b * p.ld_u + p.K] * total;
        int64_t token = -1;
        for (int i = 0; i < 256 && token < 0; i++) {
            if (before + part[i] > t) {
                double run = 0.0;
                for (int v = i * per; v < min((i + 1) * per, p.V); v++) { run += rest(p, pr, qr, mode, x, v); if (before + run > t) { token = v; break; } }
            }
            before += part[i];
        }
        if (token < 0) { token = 0; for (int i = 0; i < 256; i++) if (last[i] >= 0) token = last[i]; }
        p.tokens[(long)b * (p.K + 1) + a] = token;
        for (int j = a + 1; j <= p.K; j++) p.tokens[(long)b * (p.K + 1) + j] = -1;
    }
}

extern "C" size_t mm_verify_drafts_workspace(int64_t B, int64_t V) { (void)B; (void)V; return 0; }
extern "C" int mm_verify_drafts(const mm_verify_args* a, void* stream) {
    MM_CHECK(a, "verify_drafts: null arguments");
    MM_CHECK(a->B >= 0 && a->B < (1LL << 31) && a->K >= 0 && a->K < (1 << 20) && a->V > 0 && a->V < (1LL << 30), "verify_drafts: bad shape (B=%lld K=%lld V=%lld)",
             (long long)a->B, (long long)a->K, (long long)a->V);
    if (a->B == 0) return MM_OK;
    MM_CHECK(a->p && a->u && a->tokens && a->accepted && (a->K == 0 || a->drafts), "verify_drafts: null pointer");
    MM_CHECK(a->ld_drafts >= 0 && a->bs_p >= 0 && a->ld_p >= 0 && a->bs_q >= 0 && a->ld_q >= 0 && a->ld_u >= 0, "verify_drafts: negative stride");
    VerifyP p{a->drafts, a->p, a->K ? a->q : nullptr, a->u, a->counts, a->tokens, a->accepted, (int)a->K, (int)a->V,
              (long)a->ld_drafts, (long)a->bs_p, (long)a->ld_p, (long)a->bs_q, (long)a->ld_q, (long)a->ld_u};
    hipLaunchKernelGGL(verify_k, dim3((unsigned)a->B), dim3(256), 0, (hipStream_t)stream, p);
    MM_LAUNCH_CHECK();
    return MM_OK;
}
