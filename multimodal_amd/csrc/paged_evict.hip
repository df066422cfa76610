// Eviction from a paged key-value cache by accumulated attention weight (include/mmhip.h).
//
// Per (row, KV head): the A = budget - recent greatest of `old` weights, then as few moves as possible.  Attention does not ask for an
// order of the slots, so survivors among the first A slots stay; the i-th hole there takes the i-th survivor from behind.  Sources (>= A)
// and targets (< A) are disjoint: all moves are independent.  The newest slots shift down by n - budget; a slot's target is the
// source of the slot n - budget before it, so the slots of one residue class mod n - budget form a chain, and a thread that walks its
// chain in order needs no one else.  Of the survivors only those in slots that the shift overwrites are in its way: the first slot of a chain,
// which its walker moves before it begins.  So moves and shift are one launch.  HBM bounds it: 4 d values per slot moved (K and V, read and
// written).
//
// Selection: weights as ordered 32-bit keys, the A-th greatest found bit by bit, from the first bit in which they differ: count the keys
// >= candidate by ballots (no histogram: its bins collide where weights are alike, and equal weights are the rule at the start).  Once at most
// 64 keys are left in question each wave settles the rest alone (4 rows and heads of 40000 to 60000 slots, cut to 20000: 155 -> 136 us in all; of
// 80000 to 100000: 486 -> 410).  Up to 65536 slots stay in registers, longer rows are read again in every pass.  384 heads of up to 8192
// slots take 26 us: a workgroup loads for 3, counts for 8 (13 passes, each a barrier), settles the last 64 keys in 2, finds the places in 4 and the
// moves' rows in 1; the rest is the launch and the longest rows.
#include "paged.h"

// Order of weights as unsigned integers: greater weight, greater key; NaN above everything, -0 = 0, a slot that does not exist lowest (0).
__device__ __forceinline__ unsigned weight_key(float x) {
    if (x != x) return 0xffffffffu;
    const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
struct EvictP {
    char* kpool; char* vpool; float* w; int* lengths; int* kept; PagedMap map;
    char* ws; int room;            // per (row, KV head): {slots, moves, of them by the shift}; pool rows to [room] and from [room] of the moves;
                                   // where the shift moves what it finds, pool rows [recent] or -1; the moves as slots (without a room none of them)
    int units, budget, recent;                                                 // units: 16- or 8-byte pieces of a slot's K
    __device__ __forceinline__ int* head(long bh) const { return (int*)(ws + bh * (24L * room + (room ? 8L * recent : 0) + 16)); }
    __device__ __forceinline__ long* rows(long bh) const { return (long*)(head(bh) + 4); }
    __device__ __forceinline__ long* dest(long bh) const { return rows(bh) + 2L * room; }
    __device__ __forceinline__ int* slots(long bh) const { return (int*)(dest(bh) + recent); }
};

// ------------------------------------------------------------------------------------------------ selection (NW waves)
template <int NW> __device__ __forceinline__ int block_count(int c, int* red, int& buf) {       // c: wave-uniform
    int* r = red + (buf ^= NW);
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = c;
    __syncthreads();
    int t = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) t += r[i];
    return t;
}
// exclusive prefix of v over the workgroup's threads, and the total
template <int NW> __device__ __forceinline__ int block_scan(int v, int* red, int& buf, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int t = __shfl_up(s, o); if (lane >= o) s += t; }
    int* r = red + (buf ^= NW);
    if (lane == 63) r[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) { before += i < wave ? r[i] : 0; total += r[i]; }
    return before + s - v;
}

// R registers of keys a thread (four consecutive slots a round), R = 0: read again in every pass.  SPLIT: moves and shift run side by side
template <int NW, int R, bool SPLIT> __device__ __forceinline__ void evict_select(const EvictP& p, int b, int h, int* red) {
    constexpr int ROUND = NW * 256;
    const long bh = (long)b * p.map.Hkv + h;
    const int tid = threadIdx.x, n = min(p.lengths[b], p.map.capacity());
    int* kept = p.kept + bh * p.budget;
    int* hd = p.head(bh);
    if (tid == 0) { hd[0] = n; hd[1] = 0; hd[2] = 0; }
    if (n <= p.budget) return;
    const int A = p.budget - p.recent, old = n - p.recent, rounds = (old + ROUND - 1) / ROUND;
    // the moves as slots: in LDS where they fit (at most half of the slots move)
    constexpr int LIST = R > 0 && NW * R * 64 <= 8192 ? NW * R * 32 : 0;
    __shared__ int list[LIST ? 2 * LIST : 1];
    int* to = LIST ? list : p.slots(bh); int* from = to + (LIST ? LIST : p.room);
    auto load = [&](int r, unsigned (&k)[4]) {
        const int s = r * ROUND + tid * 4;                                     // four slots of one page
        const long row = s < old ? p.map.row(b, h, s) : -1;
        mm_f4_t w = {0.f, 0.f, 0.f, 0.f};
        if (row >= 0) w = *reinterpret_cast<const mm_f4_t*>(p.w + row);
#pragma unroll
        for (int i = 0; i < 4; i++) k[i] = row >= 0 && s + i < old ? weight_key(w[i]) : 0u;
    };
    constexpr int RR = R ? R / 4 : 1;
    unsigned key[RR][4];
    if constexpr (R > 0) {
#pragma unroll
        for (int r = 0; r < RR; r++) load(r, key[r]);
    }
    auto each = [&](auto&& f) {                                                // f(round, its keys)
        if constexpr (R > 0) {
#pragma unroll
            for (int r = 0; r < RR; r++) f(r, key[r]);
        } else
            for (int r = 0; r < rounds; r++) { unsigned k[4]; load(r, k); f(r, k); }
    };
    auto count = [&](unsigned t) {                                             // keys >= t (t > 0), over the wave
        int c = 0, all = 0;
        if constexpr (R > 4) {                                                 // a lane's count first, its bits by ballots: fewer of them
            each([&](int, const unsigned (&k)[4]) {
#pragma unroll
                for (int i = 0; i < 4; i++) c += k[i] >= t;
            });
#pragma unroll
            for (int e = 0; 1 << e <= R; e++) all += __popcll(__ballot(c >> e & 1)) << e;
        } else
            each([&](int, const unsigned (&k)[4]) {
#pragma unroll
                for (int i = 0; i < 4; i++) all += __popcll(__ballot(k[i] >= t));
            });
        return all;
    };
    __shared__ unsigned ends[2 * NW], few[64];
    __shared__ int nfew;
    int buf = 0, ge = old, above = 0, bit = 31;                                // keys >= T; keys beyond those in question
    int ties = 0x7fffffff;                                                     // how many keys equal to T are kept, lowest slots first
    unsigned T = 0;
    if (A == 0) { T = 0xffffffffu; ge = 0; }                                   // nothing of the old is kept
    else {
        if (tid == 0) nfew = 0;
        if constexpr (R == 4) __syncthreads();
        else {                                                                 // with few keys it costs more than the rounds it saves
            unsigned top = 0, low = 0;                                         // greatest key, greatest complement
            each([&](int r, const unsigned (&k)[4]) {
#pragma unroll
                for (int i = 0; i < 4; i++) if (r * ROUND + tid * 4 + i < old) { top = max(top, k[i]); low = max(low, ~k[i]); }
            });
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) { top = max(top, (unsigned)__shfl_xor((int)top, o)); low = max(low, (unsigned)__shfl_xor((int)low, o)); }
            if ((tid & 63) == 0) { ends[tid >> 6] = top; ends[NW + (tid >> 6)] = low; }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NW; i++) { top = max(top, ends[i]); low = max(low, ends[NW + i]); }
            const unsigned differ = top ^ ~low;
            bit = differ ? 31 - __clz((int)differ) : -1;
            T = bit == 31 ? 0u : top >> (bit + 1) << (bit + 1);
        }
        for (; bit >= 0 && ge != A && ge - above > 64; bit--) {
            const unsigned t = T | 1u << bit;
            const int c = block_count<NW>(count(t), red, buf);
            if (c >= A) { T = t; ge = c; } else above = c;
        }
        if (bit >= 0 && ge != A) {
            const unsigned last = T | ((2u << bit) - 1u);
            each([&](int r, const unsigned (&k)[4]) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (k[i] >= T && k[i] <= last && r * ROUND + tid * 4 + i < old) few[atomicAdd(&nfew, 1)] = k[i];   // their order does not matter
            });
            __syncthreads();
            const bool real = (tid & 63) < nfew;
            const unsigned mine = real ? few[tid & 63] : 0u;
            for (; bit >= 0 && ge != A; bit--) {
                const unsigned t = T | 1u << bit;
                const int c = above + __popcll(__ballot(real && mine >= t));
                if (c >= A) { T = t; ge = c; }
            }
            if (ge != A) ties = A - above - __popcll(__ballot(real && mine > T));
        } else if (ge != A) ties = A - (T == 0xffffffffu ? 0 : block_count<NW>(count(T + 1), red, buf));
    }
    int equal = 0, holes = 0, late = 0;                                        // so far, in slot order
    auto place = [&](int r, const unsigned (&k)[4]) {
        const int s = r * ROUND + tid * 4;
        bool keep[4];
        int eq = 0, total;
        if (ties != 0x7fffffff) {
#pragma unroll
            for (int i = 0; i < 4; i++) eq += k[i] == T && s + i < old;
            eq = equal + block_scan<NW>(eq, red, buf, total);
            equal += total;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool is = k[i] == T && s + i < old;
            keep[i] = A && s + i < old && (k[i] > T || (is && eq < ties));
            eq += is;
        }
        int c = 0;                                                             // holes | survivors behind A << 16 (a round has at most 4096 slots)
#pragma unroll
        for (int i = 0; i < 4; i++) c += s + i < A ? !keep[i] : keep[i] ? 1 << 16 : 0;
        const int pre = block_scan<NW>(c, red, buf, total);
        int hole = holes + (pre & 0xffff), sur = late + (int)((unsigned)pre >> 16);
        holes += total & 0xffff; late += (int)((unsigned)total >> 16);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (s + i < A) {
                if (keep[i]) kept[s + i] = s + i;
                else { if (hole < p.room) to[hole] = s + i; hole++; }
            } else if (keep[i]) { if (sur < p.room) from[sur] = s + i; sur++; }
        }
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int r = 0; r < RR; r++) if (r < rounds) place(r, key[r]);
    } else
        for (int r = 0; r < rounds; r++) { unsigned k[4]; load(r, k); place(r, k); }
    long* rows = p.rows(bh); long* dest = p.dest(bh);                          // looked up once here, not once a piece
    for (int j = A + tid; j < p.budget; j += NW * 64) { kept[j] = n - p.budget + j; if (SPLIT && p.room) dest[j - A] = -1; }
    __syncthreads();                                                           // the lists are written
    const int moves = min(holes, late);
    if (tid == 0) hd[1] = moves;
    constexpr int N = 4;
    for (int i0 = tid; i0 < moves; i0 += NW * 64 * N) {
        int ts[N], fs[N];
        long rt[N], rf[N];
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int i = i0 + j * NW * 64;
            ts[j] = i < moves ? to[i] : -1; fs[j] = i < moves ? from[i] : -1;
        }
#pragma unroll
        for (int j = 0; j < N; j++) { rt[j] = p.map.row(b, h, ts[j]); rf[j] = p.map.row(b, h, fs[j]); }
#pragma unroll
        for (int j = 0; j < N; j++)
            if (ts[j] >= 0) {
                const int i = i0 + j * NW * 64;
                kept[ts[j]] = fs[j];
                if (rf[j] < 0) rt[j] = -1;
                rows[i] = rt[j]; rows[p.room + i] = rf[j];
                if (SPLIT && fs[j] < p.budget) {                                   // sources ascend: these are the first moves
                    dest[fs[j] - A] = rt[j];
                    if (i + 1 == moves || from[i + 1] >= p.budget) hd[2] = i + 1;
                }
            }
    }
}

// ------------------------------------------------------------------------------------------------ moving
// the moves of a (row, KV head) that the shift does not make, one piece of K and of V a thread; `step` threads share the work.
// ST: past the last-level cache (non-temporal)
template <typename U, bool ST> __device__ __forceinline__ void evict_moves(const EvictP& p, int b, int h, int t, int step) {
    const long bh = (long)b * p.map.Hkv + h;
    const int first = p.head(bh)[2];
    const long* to = p.rows(bh) + first; const long* from = to + p.room;
    const unsigned total = (unsigned)(p.head(bh)[1] - first) * (unsigned)p.units;
    U* K = (U*)p.kpool; U* V = (U*)p.vpool;
    constexpr int N = 4;                                                       // in flight
    for (unsigned i0 = t; i0 < total; i0 += (unsigned)step * N) {
        U k[N], v[N];
        long d[N];
        int piece[N];
        float w[N];
#pragma unroll
        for (int j = 0; j < N; j++) {
            const unsigned i = i0 + (unsigned)(j * step);
            d[j] = -1;
            if (i < total) {
                const unsigned m = i / (unsigned)p.units;
                piece[j] = (int)(i - m * (unsigned)p.units);
                const long s = from[m];
                d[j] = to[m];
                if (d[j] >= 0) {
                    const U* ks = K + s * p.units + piece[j]; const U* vs = V + s * p.units + piece[j];
                    k[j] = ST ? __builtin_nontemporal_load(ks) : *ks; v[j] = ST ? __builtin_nontemporal_load(vs) : *vs;
                    if (piece[j] == 0) w[j] = p.w[s];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < N; j++)
            if (d[j] >= 0) {
                U* kd = K + d[j] * p.units + piece[j]; U* vd = V + d[j] * p.units + piece[j];
                if constexpr (ST) { __builtin_nontemporal_store(k[j], kd); __builtin_nontemporal_store(v[j], vd); }
                else { *kd = k[j]; *vd = v[j]; }
                if (piece[j] == 0) p.w[d[j]] = w[j];
            }
    }
}
// The newest slots, down by n - budget, by `blocks` workgroups of NT threads: a chain (residue class) and piece a thread where there are enough
// of them.  The survivor in a chain's first slot goes to its hole first.  Few chains are long ones (one token over the budget: one chain of all the newest slots): then one workgroup moves tile
// after tile instead, all loads of a tile before its stores, which only overwrite what has been loaded (96 heads of 964 newest slots, some
// rows one slot over: 550 us in chains).
template <typename U, int NT, bool SPLIT> __device__ __forceinline__ void evict_shift(const EvictP& p, int b, int h, int block, int blocks) {
    const int n = p.head((long)b * p.map.Hkv + h)[0];
    if (n <= p.budget || !p.recent) return;
    const int by = n - p.budget, first = n - p.recent, tid = threadIdx.x;
    const long* dest = p.dest((long)b * p.map.Hkv + h);
    const unsigned total = (unsigned)min(by, p.recent) * (unsigned)p.units, all = (unsigned)p.recent * (unsigned)p.units;
    U* K = (U*)p.kpool; U* V = (U*)p.vpool;
    constexpr int N = 4;
    auto take = [&](long j, int piece, long& d, U& k, U& v, float& w) {
        const long s = p.map.row(b, h, first + (int)j);
        d = -1;
        if (s >= 0) {
            d = p.map.row(b, h, first + (int)j - by);
            k = K[s * p.units + piece]; v = V[s * p.units + piece];
            if (piece == 0) w = p.w[s];
        }
    };
    auto put = [&](int piece, long d, const U& k, const U& v, float w) {
        if (d < 0) return;
        K[d * p.units + piece] = k; V[d * p.units + piece] = v;
        if (piece == 0) p.w[d] = w;
    };
    auto clear = [&](int c, int piece, long& d, U& k, U& v, float& w) {        // the survivor in the first slot of chain c
        d = SPLIT && p.room ? dest[c] : -1;
        if (d < 0) return;
        const long s = p.map.row(b, h, first + c - by);
        k = K[s * p.units + piece]; v = V[s * p.units + piece];
        if (piece == 0) w = p.w[s];
    };
    if (total >= all || total >= NT / 2) {
        for (unsigned i = (unsigned)(block * NT + tid); i < total; i += (unsigned)(blocks * NT)) {
            const unsigned c = i / (unsigned)p.units;
            const int piece = (int)(i - c * (unsigned)p.units);
            U k0, v0;
            float w0;
            long d0;
            clear((int)c, piece, d0, k0, v0, w0);
            for (long j0 = c; j0 < p.recent; j0 += (long)N * by) {
                U k[N], v[N];
                float w[N];
                long d[N];
#pragma unroll
                for (int e = 0; e < N; e++) { const long j = j0 + (long)e * by; d[e] = -1; if (j < p.recent) take(j, piece, d[e], k[e], v[e], w[e]); }
                if (j0 == c) put(piece, d0, k0, v0, w0);
#pragma unroll
                for (int e = 0; e < N; e++) put(piece, d[e], k[e], v[e], w[e]);
            }
        }
    } else if (block == 0) {
        if ((unsigned)tid < total) {
            const int c = tid / p.units, piece = tid - c * p.units;
            U k0, v0;
            float w0;
            long d0;
            clear(c, piece, d0, k0, v0, w0);
            put(piece, d0, k0, v0, w0);
        }
        for (unsigned i0 = 0; i0 < all; i0 += NT * N) {
            U k[N], v[N];
            float w[N];
            long d[N];
            int piece[N];
#pragma unroll
            for (int e = 0; e < N; e++) {
                const unsigned i = i0 + (unsigned)(e * NT + tid), j = i / (unsigned)p.units;
                piece[e] = (int)(i - j * (unsigned)p.units);
                d[e] = -1;
                if (i < all) take(j, piece[e], d[e], k[e], v[e], w[e]);
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < N; e++) put(piece[e], d[e], k[e], v[e], w[e]);
        }
    }
}

// ------------------------------------------------------------------------------------------------ kernels
constexpr int MOVERS = 1024;                                                   // 512: few long chains 50 us for 40 (12 rows of 8 heads of 964 newest slots)
// A workgroup per (row, KV head).  ALL: it moves and shifts as well.
template <int NW, int R, typename U, bool ALL> __global__ __launch_bounds__(NW * 64) void evict_select_k(const EvictP p) {
    __shared__ int red[2 * NW];
    const int b = blockIdx.x, h = blockIdx.y, n = min(p.lengths[b], p.map.capacity());
    if (n <= p.budget) {
        int* kept = p.kept + ((long)b * p.map.Hkv + h) * p.budget;
        for (int j = threadIdx.x; j < p.budget; j += NW * 64) kept[j] = j < n ? j : -1;
    }
    evict_select<NW, R, !ALL>(p, b, h, red);
    if constexpr (ALL) {
        __syncthreads();
        evict_moves<U, false>(p, b, h, threadIdx.x, NW * 64);
        __syncthreads();                                                       // targets of the shift were sources of the moves
        evict_shift<U, NW * 64, false>(p, b, h, 0, 1);
    }
}
// Only the selection reads the old lengths.
__device__ __forceinline__ void evict_length(const EvictP& p, int b) {
    if (blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0 && p.head((long)b * p.map.Hkv)[0] > p.budget) p.lengths[b] = p.budget;
}
// shifters workgroups of each (row, KV head) shift, the others move
template <typename U, bool ST> __global__ __launch_bounds__(MOVERS) void evict_move_k(const EvictP p, int shifters) {
    if ((int)blockIdx.z < shifters) evict_shift<U, MOVERS, true>(p, blockIdx.x, blockIdx.y, blockIdx.z, shifters);
    else evict_moves<U, ST>(p, blockIdx.x, blockIdx.y, (blockIdx.z - shifters) * MOVERS + threadIdx.x, (gridDim.z - shifters) * MOVERS);
    evict_length(p, blockIdx.x);
}
__global__ __launch_bounds__(64) void evict_lengths_k(const EvictP p) { evict_length(p, blockIdx.x); }

static int64_t evict_room(int64_t page, int64_t width, int64_t budget, int64_t recent) {
    const int64_t cap = page * width, A = budget - recent;
    return cap <= budget ? 0 : A < cap - A ? A : cap - A;                      // moves: at most the holes, at most the survivors behind them
}
extern "C" size_t mm_paged_evict_workspace(int64_t B, int64_t Hkv, int64_t page, int64_t width, int64_t budget, int64_t recent) {
    if (B <= 0 || Hkv <= 0 || page <= 0 || width <= 0 || recent < 0 || budget < recent) return 0;
    const int64_t room = evict_room(page, width, budget, recent);
    return (size_t)(B * Hkv) * (size_t)(24 * room + (room ? 8 * recent : 0) + 16);
}

template <typename U> static void evict_launch(const EvictP& p, int64_t B, int64_t cap, bool past, hipStream_t st) {
    const dim3 grid((unsigned)B, (unsigned)p.map.Hkv);
    const int64_t heads = B * p.map.Hkv;
    // Rows and heads that fill the card with a workgroup each: one launch moves and shifts as well, where that is little (microseconds in one
    // launch and in two: 768 heads cut from up to 300 slots of 256 bytes to 128 26 and 28, 1600 heads from 600 to 300 52 and 62, 9600 heads from
    // 300 to 128 200 and 270).  Else the moves and the shift spread over the card in a launch of their own (32 heads from 300 to 128 17 and 15,
    // 512 heads from 600 to 300 29 and 28, 128 heads from 1000 to 500 27 and 18, 384 heads from 8192 to 4096 217 and 170).
    const bool all = heads >= 768 && ((int64_t)p.room + p.recent) * p.units <= 8192;
#define MM_SELECT(NW_, R_) do { if (all) hipLaunchKernelGGL((evict_select_k<NW_, R_, U, true>), grid, dim3(NW_ * 64), 0, st, p); \
                                     else hipLaunchKernelGGL((evict_select_k<NW_, R_, U, false>), grid, dim3(NW_ * 64), 0, st, p); } while (0)
    if (cap <= 1024) MM_SELECT(4, 4);
    else if (cap <= 8192) MM_SELECT(8, 16);                               // eight waves: 26 us for 384 heads of 8192 slots, 16 waves 37, four 33
    else if (cap <= 32768) MM_SELECT(16, 32);
    else if (cap <= 65536) MM_SELECT(16, 64);
    else MM_SELECT(16, 0);
#undef MM_SELECT
    auto split = [&](int64_t items, int64_t each, int64_t in_all) {            // workgroups per (row, KV head), `each` pieces a thread where they suffice
        const int64_t w = cdiv(items, MOVERS * each), most = cdiv(in_all, heads);
        return (unsigned)(w < most ? w : most);
    };
    if (!all) {
        const unsigned shifters = split((int64_t)p.recent * p.units, 2, 1024), movers = split((int64_t)p.room * p.units, 4, 2048);
        const dim3 g(grid.x, grid.y, shifters + movers);
        // Where the rows' slots are more than the last-level cache holds, what is moved goes past it (384 heads halved from up to 8192 slots of 512
        // bytes: 170 us, 178 through it; 128 heads from 2000 to 1024, which it holds: 33 and 29).
        if (past) hipLaunchKernelGGL((evict_move_k<U, true>), g, dim3(MOVERS), 0, st, p, (int)shifters);
        else hipLaunchKernelGGL((evict_move_k<U, false>), g, dim3(MOVERS), 0, st, p, (int)shifters);
    }
    if (all) hipLaunchKernelGGL(evict_lengths_k, dim3(grid.x), dim3(64), 0, st, p);
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
    MM_CHECK(((uintptr_t)weights % 16) == 0, "paged_evict: weights must be 16-byte aligned");
    MM_CHECK(workspace_bytes >= mm_paged_evict_workspace(B, Hkv, page, width, budget, recent) && ((uintptr_t)workspace % 16) == 0,
             "paged_evict: workspace too small or not 16-byte aligned");
    const int64_t bytes = d * (dtype == MM_BF16 ? 2 : 4), room = evict_room(page, width, budget, recent);
    const int piece = bytes % 16 == 0 ? 16 : 8;
    MM_CHECK((room + recent) * (bytes / piece) < (1LL << 31), "paged_evict: too many slots for one call");
    EvictP p{};
    p.kpool = (char*)kpool; p.vpool = (char*)vpool; p.w = weights; p.lengths = lengths; p.kept = kept;
    p.map = {page_table, (long)ld_table, (int)width, paged_shift(page), (int)n_pages, (int)Hkv};
    p.ws = (char*)workspace; p.room = (int)room; p.units = (int)(bytes / piece); p.budget = (int)budget; p.recent = (int)recent;
    const bool past = paged_past_cache(B, Hkv, d, page, n_pages, width, dtype);
    hipStream_t st = (hipStream_t)stream;
    if (piece == 16) evict_launch<mm_u4_t>(p, B, page * width, past, st);
    else evict_launch<mm_u2_t>(p, B, page * width, past, st);
    MM_LAUNCH_CHECK();
    return MM_OK;
}
