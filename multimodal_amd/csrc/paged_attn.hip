// Attention of one token over a paged key-value cache, with its append, and the storing of runs (include/mmhip.h).
//
//   x_hs = q'_h . K_s / sqrt(d),  p = softmax_s(x) | stablemax_s(x),  o_h = sum_s p_hs V_s
//
// The cache is read once: 2 d values per slot and KV head against 4 d operations per query head, so HBM bounds it as long as the
// operations are cheap.  On the vector units they are not (shared heads: 2 G operations per byte in bf16, and the unpacking on top);
// on the matrix units a 16 x 16 tile costs the same for 1 to 16 query heads, a few per cent of the time its bytes need.  So:
//   - the query heads of a KV head are the 16 columns of a tile, 16 slots its rows: S = K Q^T;
//   - a lane's S values (column = its head, rows 4 g .. 4 g + 3 of each tile) are exactly the B operand of O^T = V^T P^T when
//     the 32 slots of a step are taken in the order (tile, group, row): probabilities never leave their lane;
//   - V comes straight from global memory too: a lane loads 16 bytes of each of "its" eight slots (a row is read whole by 16 lanes) and
//     transposes 8 x 8 values in registers (32 v_perm per 128 columns), which is the A operand.  No LDS traffic in the loop.
// The rotated q is kept as three bf16 terms (24 bits) and p as two (15 bits): the products are then as good as float32 ones, and what is
// rounded is what the caller asked to be rounded (stored keys, the output).  Each term but the last is truncated, so that all have one
// sign, and none is 0 unless the value is: an infinite query, key or value gives what it gives in one product (inf - inf and 0 * inf do not arise).
// A term that would be 0 beside one that is not is the least normal number, 2^-126, which is also where exp and the reciprocal end.
// float32 runs the same walk on the f32 matrix instruction.
// A workgroup is four waves that take 32 slots each in turn, with their own running maximum and sum, merged at the end; long caches
// are split over workgroups and a second kernel joins them (and adds the weights up).  The token's own key and value are taken
// from the inputs, not from the cache, so nothing waits for the append.  In a step's turn the next step's K is on its way while the
// softmax runs, and its V once this V has been used: 8 to 16 KB a wave, 8 to 12 waves a CU.
// Measured (a large copy: 5.1 TB/s): 1024 rows of 160 to 238 slots, 8 heads of 128, bf16: 849 MB in 150 us = 5.7 TB/s; 256 rows of 1000 to
// 2000: 6.1 TB/s; 32 rows of 300 to 16384, 8 KV heads shared by 4: 188 us = 5.8 TB/s, with weights 248 (scores and weights are
// another 90 MB); one row of 65551, 4 KV heads shared by 8: 36 us = 3.7 TB/s (two launches); float32, 64 rows of 1000 to 2000: 5.5 TB/s.
#include "paged.h"
#include <type_traits>

typedef __attribute__((ext_vector_type(4))) unsigned u4_t;
typedef __attribute__((ext_vector_type(2))) unsigned u2_t;
typedef u4_t __attribute__((aligned(8))) u4_8_t;
typedef u4_t __attribute__((aligned(2))) u4_2_t;                    // rows that are read once need no alignment beyond a value's
typedef u2_t __attribute__((aligned(2))) u2_2_t;
typedef f32x4_t __attribute__((aligned(4))) f4_4_t;

struct PagedP {
    const void* q; const void* kn; const void* vn; void* kpool; void* vpool; void* o; float* w; const int* lengths; const int* positions;
    const float* cos_t; const float* sin_t; PagedMap map;
    float* part; float2* stat; float* sc; float* sc_own;   // per (row, head, split): unscaled output [d], (max, sum); scores [row][head][capacity], [row][head]
    int B, H, Hkv, G, d, rot, n_pos, chunk, nsplit, ctiles, heads, units, stable; long ld_q, ld_k, ld_v; float scale;
};

// Slots of row b that the call attends over (its own token among them), and how they are split: into ceil(cover / chunk) even parts, in whole
// rounds of 128 slots.
__device__ __forceinline__ int paged_cover(const PagedP& p, int len) {
    const int cap = p.map.capacity();
    return len < 0 ? 0 : min(min(len, cap) + (p.kn ? 1 : 0), cap);
}
__device__ __forceinline__ int paged_part(const PagedP& p, int cover) {
    const int ns = max(1, (cover + p.chunk - 1) / p.chunk);
    return max(128, ((cover + ns - 1) / ns + 127) & ~127);
}

__device__ __forceinline__ int paged_pos(const int* positions, const int* lengths, bool append, int n_pos, int b) {
    const int n = lengths[b];
    const int pos = positions ? positions[b] : (append ? n : n - 1);
    return min(max(pos, 0), n_pos - 1);
}
// VE consecutive values from any address a value may have
template <int VE> __device__ __forceinline__ void load_any(const bf16* x, float (&v)[VE]) {
    unsigned w[VE / 2];
    if constexpr (VE == 8) {
        const u4_t t = *reinterpret_cast<const u4_2_t*>(x);
        w[0] = t[0]; w[1] = t[1]; w[2] = t[2]; w[3] = t[3];
    } else {
        const u2_t t = *reinterpret_cast<const u2_2_t*>(x);
        w[0] = t[0]; w[1] = t[1];
    }
#pragma unroll
    for (int i = 0; i < VE / 2; i++) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
template <int VE> __device__ __forceinline__ void load_any(const float* x, float (&v)[VE]) {
#pragma unroll
    for (int e = 0; e < VE; e += 4) {
        const f32x4_t t = *reinterpret_cast<const f4_4_t*>(x + e);
#pragma unroll
        for (int i = 0; i < 4; i++) v[e + i] = t[i];
    }
}
// the same of a row of d, 0 past its end (d % 4 == 0)
template <typename T, int VE> __device__ __forceinline__ void raw_piece(const T* x, int c, int d, float (&v)[VE]) {
    if (c + VE <= d) load_any(x + c, v);
    else
#pragma unroll
        for (int e = 0; e < VE; e++) v[e] = c + e < d ? to_f(x[c + e]) : 0.f;
}
// what rotates the values c .. c + VE - 1 of a row (half layout over its first rot values): partners and angles
template <typename T, int VE> struct Turn {
    float o[VE], cv[VE], sv[VE];
    bool low;
    int n;                                                                     // how many of the values are rotated
    // cs / sn: the tables' row of the position
    __device__ __forceinline__ void load(const T* x, int c, int rot, const float* cs, const float* sn) {
        n = min(max(rot - c, 0), VE);
        if (n == 0) return;
        const int half = rot >> 1;
        low = c < half;
        if (low ? c + VE <= half : c + VE <= rot) {                            // within one half: partners and angles are consecutive too
            const int i = low ? c : c - half;
            load_any(x + (low ? c + half : i), o);
            load_any(cs + i, cv);
            load_any(sn + i, sv);
            return;
        }
#pragma unroll
        for (int e = 0; e < VE; e++) {
            const bool first = c + e < half;
            const int i = c + e >= rot ? 0 : first ? c + e : c + e - half;
            o[e] = to_f(x[first ? i + half : i]);
            if (first != low) o[e] = -o[e];
            cv[e] = cs[i]; sv[e] = sn[i];
        }
    }
    __device__ __forceinline__ void apply(float (&v)[VE]) const {
#pragma unroll
        for (int e = 0; e < VE; e++) v[e] = e < n ? fmaf(v[e], cv[e], low ? -(o[e] * sv[e]) : o[e] * sv[e]) : v[e];
    }
};
// stablemax's s(x); the reciprocal is within one unit in the last place
__device__ __forceinline__ float stable_s(float x) { return x < 0.f ? __builtin_amdgcn_rcpf(1.f - x + 1e-9f) : x + 1.f; }

// over the four lanes that hold a head's values (lane ^ 16, lane ^ 32)
__device__ __forceinline__ float quad_max(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(c[0]), __uint_as_float(c[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    return v;
}
// barrier that orders LDS only: loads from global memory stay in flight across it
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// ------------------------------------------------------------------------------------------------ operands of one step (16 NT slots)
// VE: columns a lane loads of a V row (16 lanes x VE = one slab), NS: slabs of a head, NT: tiles of 16 slots in a step, AL: what a row of K
// is made of: 2 = whole 16-byte pieces, 1 = 8-byte pieces, 0 = one 8-byte piece.  K of the whole step is in registers; of V up to two
// slabs, the others follow as those are used up (a head of 512 would need 512 registers for its step otherwise).
template <typename T, int VE_, int NS_, int NT_, int AL, bool ST> struct Step {
    static constexpr bool BF = std::is_same<T, bf16>::value;
    static constexpr int VE = VE_, NS = NS_, NT = NT_, J = 4 * NT, DP = 16 * VE * NS;
    static constexpr int PE = BF ? 8 : 4, CW = 4 * PE, KC = DP / CW;           // values in a lane's piece of K, columns of a matrix instruction
    static constexpr int QT = BF ? 3 : 1, QS = DP + PE;                        // terms of q; a head's row in LDS (one piece of padding: no bank conflicts)
    static constexpr int VB = NS < 2 ? NS : 2;
    typedef typename std::conditional<VE * sizeof(T) == 16, u4_t, u2_t>::type v_t;
    template <typename V> static __device__ __forceinline__ V read(const T* p) {
        if constexpr (ST) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
        else return *reinterpret_cast<const V*>(p);
    }
    typedef __attribute__((ext_vector_type(8))) __bf16 frag_t;
    u4_t k[NT][KC];
    v_t v[VB][J];

    __device__ __forceinline__ void load_k(const T* pool, const long (&row)[NT], int d, int g) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const T* r = pool + row[t] * d;
#pragma unroll
            for (int c = 0; c < KC; c++) {
                const int col = c * CW + g * PE;
                if constexpr (AL == 2) k[t][c] = read<u4_t>(r + (col < d ? col : 0));
                else if constexpr (AL == 1) k[t][c] = read<u4_8_t>(r + min(col, d - 8));      // the last half piece: trim_k takes it from the end
                else { const u2_t a = read<u2_t>(r); k[t][c] = u4_t{a[0], a[1], 0u, 0u}; }
            }
        }
    }
    // pieces past column d become 0 (their q is 0 too, but 0 * inf is not)
    __device__ __forceinline__ void trim_k(int d, int g) {
#pragma unroll
        for (int c = 0; c < KC; c++)
            if (c * CW + CW > d) {
                const int col = c * CW + g * PE;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if (col >= d) k[t][c] = u4_t{0u, 0u, 0u, 0u};
                    else if (AL == 1 && col + 4 >= d) k[t][c] = u4_t{k[t][c][2], k[t][c][3], 0u, 0u};
                }
            }
    }
    __device__ __forceinline__ void load_slab(int s, const T* pool, const long (&row)[NT], int d, int li) {
        const int col = (s * 16 + li) * VE, cc = col < d ? col : 0;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) v[s % VB][t * 4 + i] = read<v_t>(pool + (row[t] + i) * d + cc);
    }
    __device__ __forceinline__ void load_v(const T* pool, const long (&row)[NT], int d, int li) {
#pragma unroll
        for (int s = 0; s < VB; s++) load_slab(s, pool, row, d, li);
    }
    // the token's own key, from LDS, as slot 0 of the step
    __device__ __forceinline__ void own_k(const T* ks, int li, int g) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int c = 0; c < KC; c++) k[t][c] = u4_t{0u, 0u, 0u, 0u};
        if (li == 0)
#pragma unroll
            for (int c = 0; c < KC; c++) k[0][c] = *reinterpret_cast<const u4_t*>(ks + c * CW + g * PE);
    }
    // piece c .. c + PE - 1 of a head's q, as QT terms: rows [term][heads]
    static __device__ __forceinline__ void put_q(T* lds, int heads, int head, int c, float (&x)[PE]) {
        T* f = lds + head * QS + c;
        if constexpr (!BF) { *reinterpret_cast<f32x4_t*>(f) = f32x4_t{x[0], x[1], x[2], x[3]}; }
        else {
            float least[PE];
#pragma unroll
            for (int e = 0; e < PE; e++) least[e] = x[e] == 0.f ? 0.f : copysignf(0x1p-126f, x[e]);
#pragma unroll
            for (int t = 0; t < QT; t++) {
                unsigned w[PE];
#pragma unroll
                for (int e = 0; e < PE; e++) {
                    const float h = __uint_as_float(__float_as_uint(x[e]) & 0xffff0000u);
                    w[e] = __float_as_uint(t && h == 0.f ? least[e] : h);
                    x[e] = x[e] == h ? 0.f : x[e] - h;                             // inf leaves nothing
                }
                *reinterpret_cast<u4_t*>(f + t * heads * QS) =
                    u4_t{w[0] >> 16 | w[1], w[2] >> 16 | w[3], w[4] >> 16 | w[5], w[6] >> 16 | w[7]};
            }
        }
    }
    // the scores of the step's tiles; q: this lane's head and piece in LDS.  Columns that are not rotated are exact in q's first term.
    __device__ __forceinline__ void scores(const T* q, int heads, int rot, f32x4_t (&s)[NT]) const {
        f32x4_t even[NT];                                                      // two chains of sums: a product's result takes several cycles
#pragma unroll
        for (int h = 0; h < NT; h++) { s[h] = f32x4_t{0.f, 0.f, 0.f, 0.f}; even[h] = s[h]; }
        int z = 0;
        asm volatile("" : "+v"(z));                                            // read again every step: registers are for the cache's rows
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int t = 0; t < QT; t++) {
                if (t && c * CW >= rot) break;
                const u4_t qf = *reinterpret_cast<const u4_t*>(q + (t * heads * QS + c * CW) + z);
#pragma unroll
                for (int h = 0; h < NT; h++) {
                    if constexpr (BF) {
                        s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(frag_t, k[h][c]), __builtin_bit_cast(frag_t, qf), s[h], 0, 0, 0);
                    } else {
                        const f32x4_t kf = __builtin_bit_cast(f32x4_t, k[h][c]), qq = __builtin_bit_cast(f32x4_t, qf);
#pragma unroll
                        for (int j = 0; j < 4; j += 2) {
                            s[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j], qq[j], s[h], 0, 0, 0);
                            even[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j + 1], qq[j + 1], even[h], 0, 0, 0);
                        }
                    }
                }
            }
        if constexpr (!BF)
#pragma unroll
            for (int h = 0; h < NT; h++) s[h] += even[h];
    }
    // acc[slab][column][4] += V^T P^T over one slab; slots whose bit is not set have p = 0, and their V must not be inf or NaN
    __device__ __forceinline__ void slab(int s, const float (&p)[J], unsigned ok, f32x4_t (&acc)[NS][VE]) {
        v_t (&w)[J] = v[s % VB];
        if (__ballot(ok != (1u << J) - 1)) {
#pragma unroll
            for (int j = 0; j < J; j++) if (!(ok >> j & 1)) w[j] = v_t{};
        }
        if constexpr (BF) {
            typedef __attribute__((ext_vector_type(2))) float f2_t;
            typedef __attribute__((ext_vector_type(2))) __bf16 b2_t;
            constexpr int W = J / 2;                                           // 32-bit words of an operand: 4 (32 slots) or 2 (16)
            unsigned hi[W], lo[W];
#pragma unroll
            for (int m = 0; m < W; m++) {
                const unsigned a = __float_as_uint(p[2 * m]), b = __float_as_uint(p[2 * m + 1]);
                hi[m] = __builtin_amdgcn_perm(b, a, 0x07060302u);
                lo[m] = __builtin_bit_cast(unsigned, __builtin_convertvector(
                    (f2_t{fmaxf(p[2 * m] - __uint_as_float(a & 0xffff0000u), fminf(p[2 * m], 0x1p-126f)),
                          fmaxf(p[2 * m + 1] - __uint_as_float(b & 0xffff0000u), fminf(p[2 * m + 1], 0x1p-126f))}), b2_t));
            }
#pragma unroll
            for (int e = 0; e < VE; e++) {
                unsigned x[W];
#pragma unroll
                for (int m = 0; m < W; m++)                                    // two slots' halfwords side by side
                    x[m] = __builtin_amdgcn_perm(w[2 * m + 1][e >> 1], w[2 * m][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
                if constexpr (NT == 2) {
                    const frag_t a = __builtin_bit_cast(frag_t, (u4_t{x[0], x[1], x[2], x[3]}));
                    acc[s][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(frag_t, (u4_t{hi[0], hi[1], hi[2], hi[3]})), acc[s][e], 0, 0, 0);
                    acc[s][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(frag_t, (u4_t{lo[0], lo[1], lo[2], lo[3]})), acc[s][e], 0, 0, 0);
                } else {
                    const bf16x4_t a = __builtin_bit_cast(bf16x4_t, (u2_t{x[0], x[1]}));
                    acc[s][e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, __builtin_bit_cast(bf16x4_t, (u2_t{hi[0], hi[1]})), acc[s][e], 0, 0, 0);
                    acc[s][e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, __builtin_bit_cast(bf16x4_t, (u2_t{lo[0], lo[1]})), acc[s][e], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < J; j++) {
                const f32x4_t x = __builtin_bit_cast(f32x4_t, w[j]);
#pragma unroll
                for (int e = 0; e < VE; e++) acc[s][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], p[j], acc[s][e], 0, 0, 0);
            }
        }
    }
    __device__ __forceinline__ void gather(const float (&p)[J], unsigned ok, const T* pool, const long (&row)[NT], int d, int li, f32x4_t (&acc)[NS][VE]) {
#pragma unroll
        for (int s = 0; s < NS; s++) {
            slab(s, p, ok, acc);
            if (s + VB < NS) load_slab(s + VB, pool, row, d, li);
        }
    }
    // the token's own value, from LDS
    __device__ __forceinline__ void gather_own(const float (&p)[J], const T* vs, int li, int g, f32x4_t (&acc)[NS][VE]) {
#pragma unroll
        for (int s = 0; s < NS; s++) {
#pragma unroll
            for (int j = 0; j < J; j++) v[s % VB][j] = v_t{};
            if (g == 0) v[s % VB][0] = *reinterpret_cast<const v_t*>(vs + (s * 16 + li) * VE);
            slab(s, p, (1u << J) - 1, acc);
        }
    }
};

// ------------------------------------------------------------------------------------------------ the walk
// WPR: waves that share a (row, KV head, split): 4 (merged through LDS), or 1 (four of them side by side in a workgroup).  ST: the cache is
// read past the last-level cache (non-temporal).  Waves a SIMD: three for heads up to 128, two up to 192, one beyond, where registers
// would spill -- but for short rows, which wait more than they read (8192 rows and heads of 256, 10 slots: 98 us with one, 68 with two;
// of 200 to 400 slots 125 and 139).
template <typename T, int VE, int NS, int NT, int AL, int WPR, bool ST>
__global__ __launch_bounds__(256, (VE * NS * sizeof(T) * NT <= 32 ? 3 : VE * NS * sizeof(T) * NT <= (WPR == 1 ? 64 : 48) ? 2 : 1)) void paged_attn_k(const PagedP p) {
    typedef Step<T, VE, NS, NT, AL, ST> S_t;
    constexpr int SW = 16 * VE, DP = SW * NS, SL = 16 * NT, RD = WPR * SL, J = 4 * NT;    // a wave's step, a round of the waves of a row
    constexpr int TEAMS = 4 / WPR, TT = 64 * WPR;
    extern __shared__ __attribute__((aligned(16))) char lds[];                            // q of the teams; at the end the waves' outputs
    const int HEADS = p.heads, QB = S_t::QT * HEADS * S_t::QS * (int)sizeof(T);           // query heads of a tile
    __shared__ __attribute__((aligned(16))) T own_kv[TEAMS][2][DP];
    __shared__ float st_m[4][16], st_l[4][16];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g = lane >> 4;
    const int team = wv / WPR, wave = wv % WPR, tid = threadIdx.x % TT;                   // threads and waves of one team
    T* qlds = (T*)(lds + team * QB);
    T* own_k = own_kv[team][0]; T* own_v = own_kv[team][1];
    auto sync = [&]() {                                                                   // the team's LDS is written
        if constexpr (WPR == 4) lds_barrier();
        else { __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local"); __builtin_amdgcn_wave_barrier(); __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local"); }
    };
    unsigned id = blockIdx.x * TEAMS + team;
    if (WPR == 1 && id >= (unsigned)p.units) return;
    // An odd number of workgroups a tile: they go round the eight XCDs, and with an even one those of the splits that short rows do not have stood
    // idle (452 rows and heads of 360 to 857 slots in up to two splits: 51 us; 40).
    const unsigned step = (unsigned)p.nsplit | 1u;
    const int split = (int)(id % step); id /= step;
    if (split >= p.nsplit) return;
    const int ct = (int)(id % (unsigned)p.ctiles); id /= (unsigned)p.ctiles;
    const int hk = (int)(id % (unsigned)p.Hkv), b = (int)(id / (unsigned)p.Hkv);
    const int d = p.d, cap = p.map.capacity(), len = p.lengths[b];
    const int h0 = hk * p.G + ct * 16, nh = min(16, p.G - ct * 16);                     // this tile's query heads
    const int n = min(max(len, 0), cap);                                                // slots in the cache
    const int cover = paged_cover(p, len), part = paged_part(p, cover);
    const int lo = split * part, hi = min(n, lo + part);
    if (split && lo >= cover) return;
    const bool mine = p.kn && len >= 0 && len < cap && len >= lo && len < lo + part;    // the new token falls into this split
    const long own_row = mine ? p.map.row(b, hk, len) : -1;
    const T* kp = (const T*)p.kpool; const T* vp = (const T*)p.vpool;
    const int shift = p.map.shift, mask = (1 << shift) - 1;
    const int* table = p.map.table + (long)b * p.map.ld;

    // page numbers of a step's slots: k the K rows of this lane (slot tile * 16 + li), v its four S / V slots (tile * 16 + 4 g)
    struct Pages { int k[NT], v[NT]; };
    auto fetch = [&](int s0, Pages& e) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            e.k[t] = table[min((s0 + t * 16 + li) >> shift, p.map.width - 1)];
            e.v[t] = table[min((s0 + t * 16 + g * 4) >> shift, p.map.width - 1)];
        }
    };
    auto row_of = [&](int e, int slot) -> long {                                        // slots that do not exist read row 0 of the pool and weigh nothing
        const bool ok = slot < hi && (unsigned)e < (unsigned)p.map.n_pages;
        return ok ? (((long)e * p.Hkv + hk) << shift) + (slot & mask) : 0;
    };
    S_t st;
    auto load_k = [&](int s0, const Pages& e) {
        long r[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) r[t] = row_of(e.k[t], s0 + t * 16 + li);
        st.load_k(kp, r, d, g);
    };
    unsigned ok = 0;                                                                    // bit t * 4 + i: slot exists
    long vrow[NT];
    auto load_v = [&](int s0, const Pages& e) {
        ok = 0;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            vrow[t] = row_of(e.v[t], s0 + t * 16 + g * 4);
            const int left = hi - (s0 + t * 16 + g * 4);
            if ((unsigned)e.v[t] < (unsigned)p.map.n_pages && left > 0) ok |= (left >= 4 ? 15u : (1u << left) - 1u) << (t * 4);
        }
        st.load_v(vp, vrow, d, li);
    };
    // ---- q (and the new key), rotated: loaded beside the page numbers, which the cache's rows wait for, and stored while those are under way
    // (loaded behind the rows it came after them).  Columns past d are zero, as in trim_k.
    constexpr int PE = S_t::PE, PIECES = DP / PE;
    const long trow = (long)paged_pos(p.positions, p.lengths, p.kn != nullptr, p.n_pos, b) * (p.rot >> 1);
    const float* cs = p.cos_t + trow; const float* sn = p.sin_t + trow;
    const int pieces = (nh + (mine ? 1 : 0)) * PIECES;                                  // the new key: behind the last head
    struct Item { float x[PE], y[PE]; Turn<T, PE> turn; };
    auto take = [&](int i, Item& t) {
        const int h = i / PIECES, c = i % PIECES * PE;
        const T* row = h < nh ? (const T*)p.q + (long)b * p.ld_q + (long)(h0 + h) * d : (const T*)p.kn + (long)b * p.ld_k + (long)hk * d;
        raw_piece(row, c, d, t.x);
        t.turn.load(row, c, p.rot, cs, sn);
        if (h == nh) raw_piece((const T*)p.vn + (long)b * p.ld_v + (long)hk * d, c, d, t.y);
    };
    auto put = [&](int i, Item& t) {
        const int h = i / PIECES, c = i % PIECES * PE;
        t.turn.apply(t.x);
        if (h < nh) { S_t::put_q(qlds, HEADS, h, c, t.x); return; }
        VecIO<T, PE>::store(own_k + c, t.x); VecIO<T, PE>::store(own_v + c, t.y);       // the key rounded to the cache's type, as it is stored
        if (own_row >= 0 && ct == 0) {
            T* kd = (T*)p.kpool + own_row * d + c; T* vd = (T*)p.vpool + own_row * d + c;
#pragma unroll
            for (int e = 0; e < PE; e += 4)
                if (c + e < d) {
                    const float a[4] = {t.x[e], t.x[e + 1], t.x[e + 2], t.x[e + 3]}, w[4] = {t.y[e], t.y[e + 1], t.y[e + 2], t.y[e + 3]};
                    VecIO<T, 4>::store(kd + e, a); VecIO<T, 4>::store(vd + e, w);
                }
        }
    };
    Pages e0, e1;
    Item item;
    int s0 = lo + wave * SL;
    const bool any = s0 < hi;                                                           // wave-uniform
    if (any) { fetch(s0, e0); fetch(s0 + RD, e1); }
    if (tid < pieces) take(tid, item);
    if (any) { load_k(s0, e0); load_v(s0, e0); }
    if (tid < pieces) put(tid, item);
    for (int i = tid + TT; i < pieces; i += TT) { take(i, item); put(i, item); }
    sync();
    const T* q = qlds + min(li, nh - 1) * S_t::QS + g * S_t::PE;                        // columns past the last head repeat it; nothing reads them

    f32x4_t acc[NS][VE];
#pragma unroll
    for (int s = 0; s < NS; s++)
#pragma unroll
        for (int e = 0; e < VE; e++) acc[s][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const float sc = p.stable ? p.scale : p.scale * 1.44269504088896340736f;            // softmax in base 2
    float* srow = p.sc + ((long)b * p.H + h0 + li) * cap;
    // from the scores of a step to its probabilities (relative to the running maximum), which rescale what was gathered before
    auto weigh = [&](f32x4_t (&s)[NT], unsigned okb, float (&pr)[J]) {
        float x[J];
#pragma unroll
        for (int j = 0; j < J; j++) { x[j] = s[j >> 2][j & 3] * sc; s[j >> 2][j & 3] = x[j]; }
        if (p.stable) {
#pragma unroll
            for (int j = 0; j < J; j++) { pr[j] = okb >> j & 1 ? stable_s(x[j]) : 0.f; l += pr[j]; }
            return;
        }
        float mx = m;
#pragma unroll
        for (int j = 0; j < J; j++) { x[j] = okb >> j & 1 ? x[j] : -INFINITY; mx = fmaxf(mx, x[j]); }
        mx = quad_max(mx);
        const float base = mx == -INFINITY ? 0.f : mx;
        const float al = __builtin_amdgcn_exp2f(m - base);
        if (__ballot(mx != m)) {                                                        // someone's maximum grew
            l *= al;
#pragma unroll
            for (int a = 0; a < NS; a++)
#pragma unroll
                for (int e = 0; e < VE; e++) acc[a][e] *= al;
        }
        m = mx;
#pragma unroll
        for (int j = 0; j < J; j++) { pr[j] = okb >> j & 1 ? __builtin_amdgcn_exp2f(x[j] - base) : 0.f; l += pr[j]; }
    };
    // the scores, for the weights: four slots at once, those past the end among them (nothing reads them).  The new token's score goes to a place
    // of its own, as its slot is among another wave's four.
    auto keep = [&](const f32x4_t (&s)[NT], int slot) {
        if (p.sc && li < nh) {
#pragma unroll
            for (int t = 0; t < NT; t++) if (slot + t * 16 + g * 4 < hi) *reinterpret_cast<f32x4_t*>(srow + slot + t * 16 + g * 4) = s[t];
        }
    };
    f32x4_t s[NT];
    float pr[J];
    const bool trim = d < DP;
    if (any) {
        // Memory operations complete in order, so each is issued where what waits for an earlier one does not wait for it too: the page numbers
        // before the V rows (K rows wait for them), the scores behind the use of V (stored before it they made it wait for the next K rows:
        // 249 us for 235 with 32 rows of 300 to 16384 slots).
        for (; s0 + RD < hi; s0 += RD) {
            if (trim) st.trim_k(d, g);
            st.scores(q, HEADS, p.rot, s);
            load_k(s0 + RD, e1);
            weigh(s, ok, pr);
            st.gather(pr, ok, vp, vrow, d, li, acc);
            keep(s, s0);
            fetch(s0 + 2 * RD, e0);
            load_v(s0 + RD, e1);
            e1 = e0;
        }
        if (trim) st.trim_k(d, g);
        st.scores(q, HEADS, p.rot, s);
        weigh(s, ok, pr);
        st.gather(pr, ok, vp, vrow, d, li, acc);
        keep(s, s0);
    }
    if (mine && own_row >= 0 && wave == (n - lo + SL - 1) / SL % WPR) {                   // the new token: the wave whose turn it is
        st.own_k(own_k, li, g);
        st.scores(q, HEADS, p.rot, s);
        weigh(s, lane < 16 ? 1u : 0u, pr);
        st.gather_own(pr, own_v, li, g, acc);
        if (p.sc && lane < nh) p.sc_own[b * p.H + h0 + lane] = s[0][0];
    }
    l = quad_sum(l);
    const bool single = p.nsplit == 1;
    if constexpr (WPR == 1) {
        const float inv = single ? (p.stable ? 1.f / fmaxf(l, 1e-9f) : l == 0.f ? 0.f : 1.f / l) : 1.f;
        if (li >= nh) return;
        const long bh = (long)b * p.H + h0 + li;
        if (p.stat && g == 0) p.stat[bh * p.nsplit + split] = make_float2(p.stable ? 0.f : m, l);
#pragma unroll
        for (int a = 0; a < NS; a++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int e = 0; e < VE; e += 4) {
                    const int c = a * SW + (g * 4 + r) * VE + e;
                    const float x[4] = {acc[a][e][r] * inv, acc[a][e + 1][r] * inv, acc[a][e + 2][r] * inv, acc[a][e + 3][r] * inv};
                    if (c >= d) continue;
                    if (single) VecIO<T, 4>::store((T*)p.o + bh * d + c, x);
                    else VecIO<float, 4>::store(p.part + (bh * p.nsplit + split) * d + c, x);
                }
        return;
    }
    // ---- the four waves' parts; a wave without slots has m = -inf, l = 0 and weighs nothing
    if (g == 0) { st_m[wave][li] = m; st_l[wave][li] = l; }
    lds_barrier();                                                                      // also: q has been read
    float M = 0.f, L = 0.f, f = 1.f;
    if (!p.stable) {
        M = fmaxf(fmaxf(st_m[0][li], st_m[1][li]), fmaxf(st_m[2][li], st_m[3][li]));
        const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < 4; w++) L += st_l[w][li] * __builtin_amdgcn_exp2f(st_m[w][li] - base);
        f = __builtin_amdgcn_exp2f(m - base);
    } else {
#pragma unroll
        for (int w = 0; w < 4; w++) L += st_l[w][li];
    }
    if (p.stat && wave == 0 && g == 0 && li < nh) p.stat[((long)b * p.H + h0 + li) * p.nsplit + split] = make_float2(M, L);
    if (single) f *= p.stable ? 1.f / fmaxf(L, 1e-9f) : L == 0.f ? 0.f : 1.f / L;
    float* out = (float*)lds;
#pragma unroll
    for (int a = 0; a < NS; a++) {
        if (a) lds_barrier();
        if (li < nh)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int e = 0; e < VE; e += 4)
                    *reinterpret_cast<f32x4_t*>(out + (wave * HEADS + li) * SW + (g * 4 + r) * VE + e) =
                        f32x4_t{acc[a][e][r] * f, acc[a][e + 1][r] * f, acc[a][e + 2][r] * f, acc[a][e + 3][r] * f};
        lds_barrier();
        for (int i = tid; i < nh * (SW / 4); i += 256) {
            const int h = i / (SW / 4), c = (i % (SW / 4)) * 4;
            if (a * SW + c >= d) continue;
            f32x4_t v = *reinterpret_cast<f32x4_t*>(out + h * SW + c);
#pragma unroll
            for (int w = 1; w < 4; w++) v += *reinterpret_cast<f32x4_t*>(out + (w * HEADS + h) * SW + c);
            const float r[4] = {v[0], v[1], v[2], v[3]};
            const long bh = (long)b * p.H + h0 + h;
            if (single) VecIO<T, 4>::store((T*)p.o + bh * d + a * SW + c, r);
            else VecIO<float, 4>::store(p.part + (bh * p.nsplit + split) * d + a * SW + c, r);
        }
    }
}

// ------------------------------------------------------------------------------------------------ joining the splits, adding the weights up
// Final maximum and 1 / sum of a head over its splits, by one wave (lanes take the splits in turn): every lane gets them.
__device__ __forceinline__ void paged_final(const PagedP& p, long bh, int ns, float& base, float& inv) {
    const int lane = threadIdx.x & 63;
    const float2* st = p.stat + bh * p.nsplit;
    float M = -INFINITY, L = 0.f;
    if (!p.stable) {
        for (int s = lane; s < ns; s += 64) M = fmaxf(M, st[s].x);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
    }
    base = p.stable || M == -INFINITY ? 0.f : M;
    for (int s = lane; s < ns; s += 64) { const float2 e = st[s]; L = fmaf(e.y, p.stable ? 1.f : __builtin_amdgcn_exp2f(e.x - base), L); }
    L = wave_sum(L);
    inv = p.stable ? 1.f / fmaxf(L, 1e-9f) : L == 0.f ? 0.f : 1.f / L;
}
// Workgroups below `joins`: one (row, head): the splits' outputs, 256 / (d / 4) of them at a time, d / 4 lanes of 16 bytes each.
// The others: 1024 slots of one (row, KV head): p = exp2(x - max) / sum (| s(x) / sum) of the group's heads, added to the slots' weights.
template <typename T, int NTH> __global__ __launch_bounds__(NTH) void paged_join_k(const PagedP p, int joins, int wchunks) {
    __shared__ __attribute__((aligned(16))) float red[NTH * 4];
    __shared__ float hb[64], hi[64];
    const int tid = threadIdx.x, wave = tid >> 6;
    if ((int)blockIdx.x < joins) {
        const int bh = blockIdx.x, b = bh / p.H, cols = p.d >> 2, per = NTH / cols;
        const int c = tid % cols, gr = tid / cols;
        const int cover = paged_cover(p, p.lengths[b]), part = paged_part(p, cover), ns = (cover + part - 1) / part;
        float base, inv;
        paged_final(p, bh, ns, base, inv);
        const float2* st = p.stat + (long)bh * p.nsplit;
        const float* from = p.part + (long)bh * p.nsplit * p.d + c * 4;
        f32x4_t a = {0.f, 0.f, 0.f, 0.f};
        if (gr < per) {
#pragma unroll 4
            for (int s = gr; s < ns; s += per)
                a += *reinterpret_cast<const f32x4_t*>(from + (long)s * p.d) * (p.stable ? 1.f : __builtin_amdgcn_exp2f(st[s].x - base));
        }
        *reinterpret_cast<f32x4_t*>(red + tid * 4) = a;
        __syncthreads();
        if (gr == 0) {
            for (int k = 1; k < per; k++) a += *reinterpret_cast<f32x4_t*>(red + (k * cols + c) * 4);
            const float r[4] = {a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv};
            VecIO<T, 4>::store((T*)p.o + (long)bh * p.d + c * 4, r);
        }
        return;
    }
    const int id = blockIdx.x - joins, ch = id % wchunks, bk = id / wchunks, b = bk / p.Hkv, hk = bk % p.Hkv;
    const int len = p.lengths[b], n = paged_cover(p, len), s0 = ch * (NTH * 4);
    if (s0 >= n) return;
    const int part = paged_part(p, n), ns = (n + part - 1) / part, cap = p.map.capacity();
    const int slot = s0 + tid * 4;
    const long row = slot < n ? p.map.row(b, hk, slot) : -1;                            // four slots of one page (page >= 4)
    const int fresh = p.kn ? len - slot : -1;                                           // which of the four is the new token
    f32x4_t old = {0.f, 0.f, 0.f, 0.f}, add = old;
    if (row >= 0) old = *reinterpret_cast<const f32x4_t*>(p.w + row);
    for (int g0 = 0; g0 < p.G; g0 += 64) {
        const int ng = min(64, p.G - g0);
        const long bh = (long)b * p.H + hk * p.G + g0;
        if (g0) __syncthreads();
        for (int h = wave; h < ng; h += NTH / 64) {
            float base, inv;
            paged_final(p, bh + h, ns, base, inv);
            if ((tid & 63) == 0) { hb[h] = base; hi[h] = inv; }
        }
        __syncthreads();
        if (row >= 0)
#pragma unroll 4
            for (int h = 0; h < ng; h++) {
                f32x4_t x = *reinterpret_cast<const f32x4_t*>(p.sc + (bh + h) * cap + slot);
                if (fresh >= 0 && fresh < 4) x[fresh] = p.sc_own[bh + h];
#pragma unroll
                for (int i = 0; i < 4; i++) add[i] += (p.stable ? stable_s(x[i]) : __builtin_amdgcn_exp2f(x[i] - hb[h])) * hi[h];
            }
    }
    if (row < 0) return;
    if (slot + 4 <= n && !(fresh >= 0 && fresh < 4)) {
        *reinterpret_cast<f32x4_t*>(p.w + row) = old + add;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (slot + i < n) p.w[row + i] = i == fresh ? add[i] : old[i] + add[i];
    }
}

// The most slots of a part, a whole number of rounds of 128.  Not split: up to 512 slots (a second launch costs more than it saves: 24.7 us
// against 33.5 for 32 rows of 16 heads and 500 slots), and up to 2048 where there are rows and heads for a workgroup a CU (512
// of 1000 to 2000 slots: 75 us, 84 in two parts; 452 heads of 256 and up to 857: 67, 78).  Else parts for about 768 workgroups (16 rows
// of up to 3000 slots, 8 heads: 35 us in parts of 512, 42 of 768; one row of 65551, 4 KV heads: 37 us in 384, 41 in 256, 45 in 1024),
// of at most 1024, which evens out rows of different lengths (32 rows of 300 to 16384, 8 KV heads: 188 us; 213 in 512, 209 in 4096).
static int paged_chunk(int64_t tiles, int64_t cap) {
    int64_t chunk = cdiv(cap * tiles, 768);
    if (chunk > 1024) chunk = 1024;
    if (cap <= 512 || (cap <= 2048 && tiles >= 256)) chunk = cap;
    return (int)(cdiv(chunk, 128) * 128);
}
// Joining many splits takes a workgroup of 1024 threads (171 splits of 32 heads: 11 us with 256).
static bool paged_wide_join(int nsplit) { return nsplit > 32; }
struct PagedPlan { int chunk, nsplit; size_t part, stat, sc, own; };
static PagedPlan paged_plan(const mm_paged_attn_args* a) {
    const int64_t cap = a->width * a->page, tiles = a->B * a->Hkv * cdiv(a->H / a->Hkv, 16);
    PagedPlan r;
    r.chunk = paged_chunk(tiles, cap);
    r.nsplit = (int)cdiv(cap, r.chunk);
    r.part = r.nsplit > 1 ? (size_t)(a->B * a->H) * r.nsplit * a->d * sizeof(float) : 0;
    r.stat = r.nsplit > 1 || a->weights ? (size_t)(a->B * a->H) * r.nsplit * sizeof(float2) : 0;
    r.stat = (r.stat + 255) / 256 * 256;                                                // whole cache lines of scores
    r.sc = a->weights ? (size_t)(a->B * a->H) * cap * sizeof(float) : 0;
    r.own = a->weights ? (size_t)(a->B * a->H) * sizeof(float) : 0;
    return r;
}

extern "C" size_t mm_paged_decode_attn_workspace(const mm_paged_attn_args* a) {
    if (!a || a->B <= 0 || a->H <= 0 || a->Hkv <= 0 || a->H < a->Hkv || a->d <= 0 || a->width <= 0 || a->page <= 0) return 0;
    const PagedPlan r = paged_plan(a);
    return r.part + r.stat + r.sc + r.own;
}

template <typename T, int VE, int NS, int NT, int AL> static void paged_launch(const PagedP& p, bool lone, bool past, hipStream_t st) {
    typedef Step<T, VE, NS, NT, AL, false> S_t;
    const size_t qb = (size_t)S_t::QT * p.heads * S_t::QS * sizeof(T), merge = (size_t)4 * p.heads * 16 * VE * sizeof(float);
    const size_t lds = lone ? 4 * qb : qb > merge ? qb : merge;                // at most 58 KB
#define MM_PAGED(WPR_, ST_) hipLaunchKernelGGL((paged_attn_k<T, VE, NS, NT, AL, WPR_, ST_>), dim3((unsigned)cdiv(p.units, WPR_ == 1 ? 4 : 1)), dim3(256), lds, st, p)
    if (lone) { if (past) MM_PAGED(1, true); else MM_PAGED(1, false); }
    else { if (past) MM_PAGED(4, true); else MM_PAGED(4, false); }
#undef MM_PAGED
}

extern "C" int mm_paged_decode_attn(const mm_paged_attn_args* a, void* stream) {
    MM_CHECK(a, "paged_decode_attn: null arguments");
    int rc = paged_check("paged_decode_attn", a->kpool, a->vpool, a->page_table, a->B, a->Hkv, a->d, a->page, a->n_pages, a->width, a->ld_table, a->dtype);
    if (rc != MM_OK) return rc;
    if (a->B == 0) return MM_OK;
    MM_CHECK(a->q && a->o && a->lengths && (!a->k_new == !a->v_new), "paged_decode_attn: null pointer");
    MM_CHECK(a->H > 0 && a->H <= 65535 && a->H % a->Hkv == 0, "paged_decode_attn: %lld query heads over %lld KV heads", (long long)a->H, (long long)a->Hkv);
    MM_CHECK(a->rot >= 0 && a->rot <= a->d && a->rot % 2 == 0 && (a->rot == 0 || (a->cos_t && a->sin_t && a->n_pos > 0 && a->n_pos < (1LL << 31))),
             "paged_decode_attn: bad rot/tables");
    MM_CHECK(a->ld_q >= 0 && a->ld_k >= 0 && a->ld_v >= 0, "paged_decode_attn: negative row stride");
    MM_CHECK(a->mode == MM_ATTN_SOFTMAX || a->mode == MM_ATTN_STABLEMAX, "paged_decode_attn: bad mode %d", a->mode);
    MM_CHECK((((uintptr_t)a->o | (uintptr_t)a->weights) % 16) == 0, "paged_decode_attn: o and weights must be 16-byte aligned");
    const PagedPlan r = paged_plan(a);
    const size_t need = r.part + r.stat + r.sc + r.own;
    MM_CHECK(need == 0 || (a->workspace && a->workspace_bytes >= need && ((uintptr_t)a->workspace % 16) == 0), "paged_decode_attn: workspace too small or not 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    PagedP p{};
    p.q = a->q; p.kn = a->k_new; p.vn = a->v_new; p.kpool = a->kpool; p.vpool = a->vpool; p.o = a->o; p.w = a->weights;
    p.lengths = a->lengths; p.positions = a->positions; p.cos_t = a->cos_t; p.sin_t = a->sin_t;
    p.map = {a->page_table, (long)a->ld_table, (int)a->width, paged_shift(a->page), (int)a->n_pages, (int)a->Hkv};
    char* ws = (char*)a->workspace;
    p.part = r.part ? (float*)ws : nullptr; p.stat = r.stat ? (float2*)(ws + r.part) : nullptr; p.sc = r.sc ? (float*)(ws + r.part + r.stat) : nullptr;
    p.sc_own = (float*)(ws + r.part + r.stat + r.sc);
    p.B = (int)a->B; p.H = (int)a->H; p.Hkv = (int)a->Hkv; p.G = (int)(a->H / a->Hkv); p.d = (int)a->d; p.rot = (int)a->rot;
    p.n_pos = a->rot ? (int)a->n_pos : 1; p.ld_q = a->ld_q; p.ld_k = a->ld_k; p.ld_v = a->ld_v; p.scale = (float)(1.0 / sqrt((double)a->d));
    p.chunk = r.chunk; p.nsplit = r.nsplit; p.ctiles = (int)cdiv(p.G, 16); p.heads = p.G < 16 ? p.G : 16; p.stable = a->mode == MM_ATTN_STABLEMAX;
    const int64_t blocks = a->B * a->Hkv * p.ctiles * (p.nsplit | 1);
    const int wchunks = a->weights ? (int)cdiv(a->width * a->page, paged_wide_join(r.nsplit) ? 4096 : 1024) : 0, joins = p.nsplit > 1 ? (int)(a->B * a->H) : 0;
    const int64_t blocks2 = joins + a->B * a->Hkv * wchunks;
    MM_CHECK(a->B * a->H < (1LL << 31) && blocks < (1LL << 31) && blocks2 < (1LL << 31), "paged_decode_attn: too many rows and heads for one call");
    p.units = (int)blocks;
    // Many short rows: a wave each (1024 rows of 160 to 238 slots, 8 heads: 164 us, four waves a row 173; 256 rows of 900, 8 KV heads: 150 and 140).
    // Four times q in LDS: not for more than four query heads a KV head unless the head is small.
    const bool lone = (p.G <= 4 || a->d <= 64) && r.nsplit == 1 && a->width * a->page <= 512 && blocks >= 2048;
    // A cache that the last-level cache (256 MB) cannot hold until the next call is read past it: 154 us for 164 at 849 MB; at 69 MB it
    // would be 39 for 26.  It goes by the pool, not by rows and their width alone, as rows may share pages or be the same row: five tokens of
    // each of 128 rows of 240 slots, 8 heads of 128, a pool of 126 MB: 73 us, 98 past the cache.
    const bool past = paged_past_cache(a->B, a->Hkv, a->d, a->page, a->n_pages, a->width, a->dtype);
    const int64_t d = a->d;
    if (a->dtype == MM_F32) {
        if (d <= 64) paged_launch<float, 4, 1, 1, 2>(p, lone, past, st);
        else if (d <= 128) paged_launch<float, 4, 2, 1, 2>(p, lone, past, st);
        else if (d <= 192) paged_launch<float, 4, 3, 1, 2>(p, lone, past, st);
        else if (d <= 256) paged_launch<float, 4, 4, 1, 2>(p, lone, past, st);
        else paged_launch<float, 4, 8, 1, 2>(p, lone, past, st);
    } else if (d % 8 == 0) {
        if (d <= 64) paged_launch<bf16, 4, 1, 2, 2>(p, lone, past, st);
        else if (d <= 128) paged_launch<bf16, 8, 1, 2, 2>(p, lone, past, st);
        else if (d <= 192) paged_launch<bf16, 4, 3, 2, 2>(p, lone, past, st);
        else if (d <= 256) paged_launch<bf16, 8, 2, 2, 2>(p, lone, past, st);
        else paged_launch<bf16, 8, 4, 1, 2>(p, lone, past, st);
    } else {                                                                            // rows of whole 8-byte pieces only
        if (d == 4) paged_launch<bf16, 4, 1, 2, 0>(p, lone, past, st);
        else if (d <= 64) paged_launch<bf16, 4, 1, 2, 1>(p, lone, past, st);
        else if (d <= 128) paged_launch<bf16, 4, 2, 2, 1>(p, lone, past, st);
        else if (d <= 192) paged_launch<bf16, 4, 3, 2, 1>(p, lone, past, st);
        else if (d <= 256) paged_launch<bf16, 4, 4, 2, 1>(p, lone, past, st);
        else paged_launch<bf16, 4, 8, 1, 1>(p, lone, past, st);
    }
    MM_LAUNCH_CHECK();
    if (blocks2) {
#define MM_JOIN(T_) do { if (paged_wide_join(r.nsplit)) hipLaunchKernelGGL((paged_join_k<T_, 1024>), dim3((unsigned)blocks2), dim3(1024), 0, st, p, joins, wchunks); \
                         else hipLaunchKernelGGL((paged_join_k<T_, 256>), dim3((unsigned)blocks2), dim3(256), 0, st, p, joins, wchunks); } while (0)
        if (a->dtype == MM_F32) MM_JOIN(float); else MM_JOIN(bf16);
        MM_LAUNCH_CHECK();
    }
    return MM_OK;
}

// ------------------------------------------------------------------------------------------------ runs of keys and values
// A copy: keys and values are read once and written once, which HBM bounds: 1125 MB (1024 rows of 100 to 159 tokens, 8 heads of 128, bf16) in
// 213 us = 5.3 TB/s.  A lane moves VE consecutive values of one head of one token (16 bytes; 8 where a bf16 row is no multiple of 16);
// for a rotated key it also reads the partner values (the other half: in the same row, so from the cache that has just fetched it), which
// spares an exchange between lanes.  One piece a lane: with two or four in flight the large case took 230 and 271 us.
struct FillP {
    const void* k; const void* v; void* kpool; void* vpool; float* w; const int* start; const int* counts; const int* positions;
    const float* cos_t; const float* sin_t; PagedMap map; int S, Hkv, d, rot, n_pos; long ld_k, bs_k, ld_v, bs_v;
};
template <typename T, int VE> __global__ __launch_bounds__(256) void paged_fill_k(const FillP p) {
    const int b = blockIdx.y;
    const unsigned pieces = (unsigned)p.d / VE, per = pieces * (unsigned)p.Hkv;
    const unsigned idx = blockIdx.x * 256u + threadIdx.x;                // over [S][Hkv][d / VE]; fits (checked by the launch)
    const int s = (int)(idx / per);
    const unsigned rem = idx - (unsigned)s * per;
    const int h = (int)(rem / pieces), c = (int)(rem - (unsigned)h * pieces) * VE;
    const int st = p.start ? p.start[b] : 0, n = p.counts ? min(p.counts[b], p.S) : p.S;
    if (st < 0 || s >= n || s > 0x7fffffff - st) return;
    const T* k = (const T*)p.k + (long)b * p.bs_k + (long)s * p.ld_k + (long)h * p.d;
    const T* v = (const T*)p.v + (long)b * p.bs_v + (long)s * p.ld_v + (long)h * p.d;
    float x[VE], y[VE];
    load_any(k + c, x);
    load_any(v + c, y);
    if (c < p.rot) {
        const long pos = p.positions ? (long)p.positions[b] + s : (long)st + s;
        const long t = min(max(pos, 0L), (long)p.n_pos - 1) * (p.rot >> 1);
        Turn<T, VE> turn;
        turn.load(k, c, p.rot, p.cos_t + t, p.sin_t + t);
        turn.apply(x);
    }
    const long row = p.map.row(b, h, st + s);
    if (row < 0) return;
    VecIO<T, VE>::store((T*)p.kpool + row * p.d + c, x);
    VecIO<T, VE>::store((T*)p.vpool + row * p.d + c, y);
    if (p.w && c == 0) p.w[row] = 0.f;
}

extern "C" int mm_paged_cache_fill(const mm_paged_fill_args* a, void* stream) {
    MM_CHECK(a, "paged_cache_fill: null arguments");
    int rc = paged_check("paged_cache_fill", a->kpool, a->vpool, a->page_table, a->B, a->Hkv, a->d, a->page, a->n_pages, a->width, a->ld_table, a->dtype);
    if (rc != MM_OK) return rc;
    MM_CHECK(a->S >= 0 && a->S < (1LL << 30), "paged_cache_fill: S=%lld", (long long)a->S);
    if (a->B == 0 || a->S == 0) return MM_OK;
    MM_CHECK(a->k && a->v, "paged_cache_fill: null pointer");
    MM_CHECK(a->rot >= 0 && a->rot <= a->d && a->rot % 2 == 0 && (a->rot == 0 || (a->cos_t && a->sin_t && a->n_pos > 0 && a->n_pos < (1LL << 31))),
             "paged_cache_fill: bad rot/tables");
    MM_CHECK(a->ld_k >= 0 && a->ld_v >= 0 && a->bs_k >= 0 && a->bs_v >= 0, "paged_cache_fill: negative stride");
    FillP p{};
    p.k = a->k; p.v = a->v; p.kpool = a->kpool; p.vpool = a->vpool; p.w = a->weights; p.start = a->start; p.counts = a->counts; p.positions = a->positions;
    p.cos_t = a->cos_t; p.sin_t = a->sin_t; p.map = {a->page_table, (long)a->ld_table, (int)a->width, paged_shift(a->page), (int)a->n_pages, (int)a->Hkv};
    p.S = (int)a->S; p.Hkv = (int)a->Hkv; p.d = (int)a->d; p.rot = (int)a->rot; p.n_pos = a->rot ? (int)a->n_pos : 1;
    p.ld_k = a->ld_k; p.bs_k = a->bs_k; p.ld_v = a->ld_v; p.bs_v = a->bs_v;
    const int VE = a->dtype == MM_BF16 && a->d % 8 == 0 ? 8 : 4;
    const int64_t items = a->S * a->Hkv * (a->d / VE);
    MM_CHECK(items < (1LL << 31), "paged_cache_fill: too many tokens for one call");
    const dim3 grid((unsigned)cdiv(items, 256), (unsigned)a->B);
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == MM_F32) hipLaunchKernelGGL((paged_fill_k<float, 4>), grid, dim3(256), 0, st, p);
    else if (VE == 8) hipLaunchKernelGGL((paged_fill_k<bf16, 8>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((paged_fill_k<bf16, 4>), grid, dim3(256), 0, st, p);
    MM_LAUNCH_CHECK();
    return MM_OK;
}
