// Drafted tokens against the target's probabilities (include/mmhip.h).
//
// Bound by reading one row of p (and of q): the drafts themselves touch two scattered values each, which the first lanes fetch at once.
// One pass: the vocabulary is cut into blocks, a wave sums a block of 256 by a scan over its lanes (four values a lane), and only the
// block totals are kept; the block that holds the drawn point is found among the totals, and that one block is read again.  Sums are 64-bit:
// the drawn token is where a cumulative sum passes a number, and float32 sums over a large vocabulary move that place.  Each level
// repeats the additions of the one below it in the same order, so that a block chosen by its total always holds the point.
#include "common.h"

struct VerifyP {
    const int64_t* x; const float* p; const float* q; const float* u; const int* counts; int64_t* tokens; int* accepted; double* ws;
    int K, V, nblocks, sub, parts; long ld_x, bs_p, ld_p, bs_q, ld_q, ld_u;       // a block: sub * 256 values
};
typedef float vf4_t __attribute__((ext_vector_type(4), aligned(4)));               // rows need no alignment beyond a float's

struct Draw {                                                                      // the distribution the last token is drawn from
    const float* p; const float* q; int64_t x; int V;                              // q row, or the copied draft's id, or neither
    __device__ __forceinline__ void four(int v, double (&r)[4]) const {
        float a[4] = {0.f, 0.f, 0.f, 0.f}, c[4] = {0.f, 0.f, 0.f, 0.f};
        if (v + 4 <= V) {
            const vf4_t t = *reinterpret_cast<const vf4_t*>(p + v);
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = t[i];
            if (q) {
                const vf4_t s = *reinterpret_cast<const vf4_t*>(q + v);
#pragma unroll
                for (int i = 0; i < 4; i++) c[i] = s[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) if (v + i < V) { a[i] = p[v + i]; if (q) c[i] = q[v + i]; }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double d = (double)a[i] - (x == v + i ? 1.0 : (double)c[i]);
            r[i] = d > 0.0 ? d : 0.0;
        }
    }
};
// inclusive scan over the wave, always the same additions
__device__ __forceinline__ double wave_scan(double s) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const double t = __shfl_up(s, o); if (lane >= o) s += t; }
    return s;
}
// lane i's value, i uniform
__device__ __forceinline__ double lane_value(double v, int i) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)u, i), hi = __builtin_amdgcn_readlane((unsigned)(u >> 32), i);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
// total of block k (wave-uniform)
__device__ __forceinline__ double block_total(const Draw& w, int k, int sub) {
    const int lane = threadIdx.x & 63;
    double total = 0.0;
    for (int j = 0; j < sub; j++) {
        double r[4];
        w.four((k * sub + j) * 256 + lane * 4, r);
        total += lane_value(wave_scan(((r[0] + r[1]) + r[2]) + r[3]), 63);
    }
    return total;
}
// drafts accepted by row b (every wave finds the same number)
__device__ __forceinline__ int accept(const VerifyP& p, int b, int& n) {
    const int lane = threadIdx.x & 63;
    n = p.counts ? min(max(p.counts[b], 0), p.K) : p.K;
    for (int i0 = 0; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        bool yes = false;
        if (i < n) {
            const int64_t x = p.x[b * p.ld_x + i];
            if (x >= 0 && x < p.V) {
                const double q = p.q ? (double)p.q[b * p.bs_q + i * p.ld_q + x] : 1.0;
                yes = (double)p.u[b * p.ld_u + i] * q < (double)p.p[b * p.bs_p + i * p.ld_p + x];
            }
        }
        const unsigned long long no = ~__ballot(yes);
        const int first = no ? __ffsll(no) - 1 : 64;
        if (first < 64 && i0 + first < n) return i0 + first;
    }
    return n;
}
__device__ __forceinline__ Draw residual(const VerifyP& p, int b, int a, int n) {
    return Draw{p.p + b * p.bs_p + a * p.ld_p, a < n && p.q ? p.q + b * p.bs_q + a * p.ld_q : nullptr,
                a < n && !p.q ? p.x[b * p.ld_x + a] : (int64_t)-1, p.V};
}
// totals of the blocks first, first + step, ..: four of them in flight a wave
__device__ __forceinline__ void all_totals(const Draw& w, double* totals, int first, int step, int nblocks, int sub) {
    const int lane = threadIdx.x & 63;
    int k = first;
    if (sub == 1)
        for (; k + 3 * step < nblocks; k += 4 * step) {
            double r[4][4];
#pragma unroll
            for (int j = 0; j < 4; j++) w.four((k + j * step) * 256 + lane * 4, r[j]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const double t = wave_scan(((r[j][0] + r[j][1]) + r[j][2]) + r[j][3]);
                if (lane == 63) totals[k + j * step] = t;
            }
        }
    for (; k < nblocks; k += step) { const double t = block_total(w, k, sub); if (lane == 0) totals[k] = t; }
}

// totals of a part of a row's blocks, for few rows of a large vocabulary
__global__ __launch_bounds__(256) void verify_totals_k(const VerifyP p) {
    const int b = blockIdx.y;
    int n;
    const int a = accept(p, b, n);
    const Draw w = residual(p, b, a, n);
    all_totals(w, p.ws + (long)b * p.nblocks, blockIdx.x * 4 + (threadIdx.x >> 6), gridDim.x * 4, p.nblocks, p.sub);
}

constexpr int VERIFY_BLOCKS = 4096;
template <int NW> __global__ __launch_bounds__(NW * 64) void verify_k(const VerifyP p) {
    __shared__ double totals[VERIFY_BLOCKS];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int n;
    const int a = accept(p, b, n);
    Draw w = residual(p, b, a, n);
    int64_t* out = p.tokens + (long)b * (p.K + 1);
    for (int j = tid; j < p.K + 1; j += NW * 64) if (j != a) out[j] = j < a ? p.x[b * p.ld_x + j] : -1;
    if (tid == 0) p.accepted[b] = a;
    const double u = (double)p.u[b * p.ld_u + p.K];
    bool have = p.parts > 1;
    for (;;) {
        if (have) for (int k = tid; k < p.nblocks; k += NW * 64) totals[k] = p.ws[(long)b * p.nblocks + k];
        else all_totals(w, totals, wave, NW, p.nblocks, p.sub);
        __syncthreads();
        // 64 segments of blocks, each summed in order by a lane; the segments in order
        const int per = (p.nblocks + 63) / 64, k0 = min(lane * per, p.nblocks), k1 = min(k0 + per, p.nblocks);
        double run = 0.0;
        for (int k = k0; k < k1; k++) run += totals[k];
        double sum = 0.0, base = 0.0;                                              // base: what lies before this lane's segment
#pragma unroll 4
        for (int i = 0; i < 64; i++) { if (i == lane) base = sum; sum += lane_value(run, i); }
        if (!(sum > 0.0) && (w.q || w.x >= 0)) {                                   // nothing is left of p: the row itself
            w.q = nullptr; w.x = -1; have = false;
            __syncthreads();
            continue;
        }
        if (wave) return;
        const double t = u * sum;
        const unsigned long long over = __ballot(base + run > t);
        int64_t token = 0;
        if (sum > 0.0 && over) {
            const int seg = __ffsll(over) - 1;
            const double sb = lane_value(base, seg);
            const int s0 = min(seg * per, p.nblocks), s1 = min(s0 + per, p.nblocks);
            double before = 0.0;                                                   // within the segment
            int k = s0;
            for (; k < s1 - 1; k++) { const double next = before + totals[k]; if (sb + next > t) break; before = next; }
            double blk = 0.0;                                                      // within the block
            for (int j = 0; j < p.sub; j++) {
                const int v = (k * p.sub + j) * 256 + lane * 4;
                double r[4];
                w.four(v, r);
                const double inc = wave_scan(((r[0] + r[1]) + r[2]) + r[3]), end = lane_value(inc, 63);
                const unsigned long long hit = __ballot(sb + (before + (blk + inc)) > t);
                if (!hit && j + 1 < p.sub) { blk += end; continue; }
                int who = hit ? __ffsll(hit) - 1 : 63;
                const double prev = __shfl_up(inc, 1), exc = lane ? prev : 0.0;
                int at = -1, lastp = -1;
                double c = 0.0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    c = i ? c + r[i] : r[0];
                    if (r[i] > 0.0) { lastp = v + i; if (at < 0 && sb + (before + (blk + (exc + c))) > t) at = v + i; }
                }
                // neighbouring lanes' sums were added up in different orders: the lane found may hold nothing, the one before it is meant then
                const unsigned long long mass = __ballot(lastp >= 0), upto = mass & ((2ull << who) - 1);
                who = upto ? 63 - __clzll(upto) : mass ? __ffsll(mass) - 1 : 0;
                token = max(__shfl(at >= 0 ? at : lastp, who), 0);
                break;
            }
        } else if (sum > 0.0) {                                                    // u outside [0, 1): the last value with any mass
            int last = 0;
            for (int v = lane * 4; v < p.V; v += 256) {
                double r[4];
                w.four(v, r);
#pragma unroll
                for (int i = 0; i < 4; i++) if (r[i] > 0.0) last = v + i;
            }
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) last = max(last, __shfl_xor(last, o));
            token = last;
        }
        if (lane == 0) out[a] = token;
        return;
    }
}

// Few rows cannot fill the card with a workgroup each: the totals of a row are then split over workgroups of a launch of their own.
static int verify_parts(int64_t B, int64_t V) {
    if (B >= 128 || V <= 16384) return 1;
    const int64_t w = cdiv(512, B), most = cdiv(V, 4096);
    return (int)(w < most ? w : most);
}
static int64_t verify_sub(int64_t V) { return cdiv(cdiv(V, 256), VERIFY_BLOCKS); }
extern "C" size_t mm_verify_drafts_workspace(int64_t B, int64_t V) {
    if (B <= 0 || V <= 0 || verify_parts(B, V) == 1) return 0;
    return (size_t)B * (size_t)cdiv(V, 256 * verify_sub(V)) * sizeof(double);
}
extern "C" int mm_verify_drafts(const mm_verify_args* a, void* stream) {
    MM_CHECK(a, "verify_drafts: null arguments");
    MM_CHECK(a->B >= 0 && a->B <= 65535 && a->K >= 0 && a->K < (1 << 20) && a->V > 0 && a->V < (1LL << 30), "verify_drafts: bad shape (B=%lld K=%lld V=%lld)",
             (long long)a->B, (long long)a->K, (long long)a->V);
    if (a->B == 0) return MM_OK;
    MM_CHECK(a->p && a->u && a->tokens && a->accepted && (a->K == 0 || a->drafts), "verify_drafts: null pointer");
    MM_CHECK(a->ld_drafts >= 0 && a->bs_p >= 0 && a->ld_p >= 0 && a->bs_q >= 0 && a->ld_q >= 0 && a->ld_u >= 0, "verify_drafts: negative stride");
    const size_t need = mm_verify_drafts_workspace(a->B, a->V);
    MM_CHECK(need == 0 || (a->workspace && a->workspace_bytes >= need && ((uintptr_t)a->workspace % 8) == 0), "verify_drafts: workspace too small or not aligned");
    const int sub = (int)verify_sub(a->V), parts = verify_parts(a->B, a->V);
    VerifyP p{a->drafts, a->p, a->K ? a->q : nullptr, a->u, a->counts, a->tokens, a->accepted, (double*)a->workspace, (int)a->K, (int)a->V,
              (int)cdiv(a->V, 256 * (int64_t)sub), sub, parts, (long)a->ld_drafts, (long)a->bs_p, (long)a->ld_p, (long)a->bs_q, (long)a->ld_q, (long)a->ld_u};
    hipStream_t st = (hipStream_t)stream;
    if (parts > 1) {
        hipLaunchKernelGGL(verify_totals_k, dim3((unsigned)parts, (unsigned)a->B), dim3(256), 0, st, p);
        MM_LAUNCH_CHECK();
    }
    if (a->V <= 4096 || parts > 1) hipLaunchKernelGGL(verify_k<4>, dim3((unsigned)a->B), dim3(256), 0, st, p);
    else hipLaunchKernelGGL(verify_k<16>, dim3((unsigned)a->B), dim3(1024), 0, st, p);
    MM_LAUNCH_CHECK();
    return MM_OK;
}
