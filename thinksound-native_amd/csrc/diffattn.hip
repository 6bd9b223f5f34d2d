// diffattn.hip — differential attention for gfx950: the difference of two softmax maps times one V,
//     lambda = exp(lq1.lk1) - exp(lq2.lk2) + lambda_init
//     o = softmax(s q1 k1^T) v - lambda softmax(s q2 k2^T) v,   out = (1 - lambda_init) RMS(o) w, or o.
// One pass over the keys: each map keeps its running maximum, sum and product with V (the online
// softmax), and the two are joined once both sums are known.
//
// Work of a pair (row, key) that a head sees: 4 hd operations for both maps' scores, 8 hd for their products with V (joined
// before it the maps need 4 hd, but both sums first, so the scores twice: 12 hd as well), two exponentials. Long contexts
// are bound by these under the card's power limit, one new row by reading its cache.
#include <math.h>

#include <algorithm>

#include "kernels.h"

#include "dpp.h"
#include "elems.h"

namespace tsn {

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// rows and keys of a sample, inside what the call gives it
__device__ __forceinline__ int q_rows(const DiffAttnArgs &a, int b) {
    return a.q_len ? min(max(a.q_len[b], 0), (int)a.Sq) : (int)a.Sq;
}
__device__ __forceinline__ int kv_rows(const DiffAttnArgs &a, int b) {
    return a.kv_len ? min(max(a.kv_len[b], 0), (int)a.Sk) : (int)a.Sk;
}
// lambda of head h, by a whole wave: lane i takes element i of the vectors
__device__ __forceinline__ float wave_lambda(const DiffAttnArgs &a, int h, int lane) {
    const int hd = (int)a.hd;
    const float *l = a.lam + (a.lam_heads > 1 ? (long long)h * 4 * hd : 0);
    const bool in = lane < hd;
    const float d1 = wave_sum(in ? l[lane] * l[hd + lane] : 0.0f);
    const float d2 = wave_sum(in ? l[2 * hd + lane] * l[3 * hd + lane] : 0.0f);
    return expf(d1) - expf(d2) + a.lambda_init;
}

// What scores are multiplied with before exp2. A scale of 0 must not meet a masked score's infinity: the smallest float
// makes finite products of q and k less than 2^-21 (zero queries instead cost a single row 0.2 of 12.3 us).
__device__ __forceinline__ float score_factor(const DiffAttnArgs &a) { return a.scale > 0.0f ? a.scale * LOG2E : 0x1p-149f; }

// What the RMS norm multiplies a row of these squares with. Squares below f32's range (bf16 values under 2^-75) leave eps
// alone; a row without keys stays zero also where eps is.
template <int HD>
__device__ __forceinline__ float rms_factor(const DiffAttnArgs &a, float squares) {
    const float ms = squares / (float)(2 * HD) + a.eps;
    return ms == 0.0f ? 0.0f : (1.0f - a.lambda_init) / sqrtf(ms);
}

// Any stride and alignment (two samples of 397 rows, 8 heads, f16: 133 us; whole chunks 11): one wave a row and head. A
// block of 64 keys at a time, lane j takes the scores of key j;
// the probabilities go through LDS, then the lanes take the columns of V.
template <typename T, int HD>
__global__ __launch_bounds__(256) void diff_attn_any_kernel(const DiffAttnArgs a) {
    constexpr int NV = 2 * HD / 64;   // columns of V a lane
    __shared__ float sq[4][2 * HD];
    __shared__ float sp[4][2][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long n_items = (long long)a.B * a.Sq * a.nh;
    for (long long id = (long long)blockIdx.x * 4 + wave; id < n_items; id += (long long)gridDim.x * 4) {   // no barrier: a wave uses its own LDS
        const int h = (int)(id % a.nh);
        const long long br = id / a.nh;
        const int b = (int)(br / a.Sq), r = (int)(br - (long long)b * a.Sq);
        const int nq = q_rows(a, b), nk = kv_rows(a, b);
        if (r >= nq) continue;
        const int g = h / (int)(a.nh / a.nkv);
        int keys = nk;
        if (a.causal) keys = min(nk, max(0, r + nk - nq + 1));
        const T *q = (const T *)a.q + (long long)b * a.bsq + (long long)r * a.ldq + (long long)h * 2 * HD;
        const T *k = (const T *)a.k + (long long)b * a.bsk + (long long)g * 2 * HD;
        const T *v = (const T *)a.v + (long long)b * a.bsv + (long long)g * 2 * HD;
        for (int i = lane; i < 2 * HD; i += 64) sq[wave][i] = (float)q[i] * a.scale * LOG2E;
        __builtin_amdgcn_wave_barrier();   // a wave's LDS accesses are done in their order
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[2][NV] = {};
        for (int k0 = 0; k0 < keys; k0 += 64) {
            const int n = min(64, keys - k0);
            float s[2] = {-INFINITY, -INFINITY};
            if (lane < n) {
                const T *kr = k + (long long)(k0 + lane) * a.ldk;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float d = 0.0f;
                    for (int i = 0; i < HD; ++i) d += sq[wave][j * HD + i] * (float)kr[j * HD + i];
                    s[j] = d;
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float mn = fmaxf(m[j], wave_max(s[j]));
                const float al = exp2f(m[j] - mn), p = lane < n ? exp2f(s[j] - mn) : 0.0f;
                m[j] = mn;
                l[j] = l[j] * al + wave_sum(p);
                for (int c = 0; c < NV; ++c) o[j][c] *= al;
                sp[wave][j][lane] = p;
            }
            __builtin_amdgcn_wave_barrier();
            for (int t = 0; t < n; ++t) {
                const T *vr = v + (long long)(k0 + t) * a.ldv;
#pragma unroll
                for (int c = 0; c < NV; ++c) {
                    const float x = (float)vr[lane + 64 * c];
                    o[0][c] += sp[wave][0][t] * x;
                    o[1][c] += sp[wave][1][t] * x;
                }
            }
        }
        const float lam = wave_lambda(a, h, lane);
        const float r0 = l[0] > 0.0f ? 1.0f / l[0] : 0.0f, r1 = l[1] > 0.0f ? lam / l[1] : 0.0f;
        float ss = 0.0f, y[NV];
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            y[c] = o[0][c] * r0 - o[1][c] * r1;
            ss += y[c] * y[c];
        }
        const float f = a.norm_w ? rms_factor<HD>(a, wave_sum(ss)) : 1.0f;
        T *out = (T *)a.out + (long long)b * a.bso + (long long)r * a.ldo + (long long)h * 2 * HD;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int i = lane + 64 * c;
            out[i] = (T)(a.norm_w ? y[c] * f * a.norm_w[i] : y[c]);
        }
    }
}

/* ---------------- MFMA kernels ---------------- */
//
// The rows of a key/value head are its nh/nkv heads' rows, heads next to each other: row x is query x / G of head
// g*G + x % G, so heads that share keys share a tile of them. A wave takes 32 rows and computes (32x32x16 MFMA, A row
// and B column = lane & 31, K group = lane >> 5, D[8*(r>>2) + 4*(lane>>5) + (r&3)][lane & 31], r = 0..15)
//   S^T = K Q^T  for 32 keys and each map: A = K rows from LDS, B = the wave's Q rows in registers. K rows are taken in
//                the order key_of(i), so that a lane ends with keys 16c + 8*(lane>>5) + 0..7, c = 0, 1, of query lane & 31:
//   O^T += V^T P^T: B = these probabilities as they lie in registers, A = V^T by transposing LDS reads
//                (ds_read_b64_tr_b16: a 16-lane group reads four keys of 16 columns and gets column lane & 15).
// Both maps multiply the same V fragments. A query's statistics and its O columns are in lanes q and q + 32.
//
// LDS rows (2 HD elements of one key) are 16-byte chunks; chunk c of row r sits at slot c ^ swizzle(r), so that the 16
// rows of a K read and the four rows of a V read fall in distinct banks.

typedef __attribute__((address_space(3))) char lds_char;
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) i32x4 lds_i32x4;
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ floatx16 mfma32(i32x4 a, i32x4 b, floatx16 c, half_t) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mfma32(i32x4 a, i32x4 b, floatx16 c, bf16_t) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// two values rounded to nearest even, in one register
template <typename T> struct Pair;
template <> struct Pair<half_t> { typedef half2_t type; };
template <> struct Pair<bf16_t> { typedef bf16x2 type; };
template <typename T>
__device__ __forceinline__ int pack2(float a, float b) {
    return __builtin_bit_cast(int, __builtin_convertvector((floatx2{a, b}), typename Pair<T>::type));
}
__device__ __forceinline__ floatx16 zero16() {
    return floatx16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
}
// both lanes of a query (l, l ^ 32) get the maximum, the sum
__device__ __forceinline__ float pair_max(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// A buffer of `bytes` (at most 2^30) bytes: loads from behind its end read as zero
__device__ __forceinline__ i32x4 buffer(const void *base, unsigned bytes) {
    const unsigned long long p = (unsigned long long)base;
    return i32x4{(int)__builtin_amdgcn_readfirstlane((unsigned)p), (int)(__builtin_amdgcn_readfirstlane((unsigned)(p >> 32)) & 0xFFFF),
                 (int)__builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
// 16 bytes a lane at voff + soff, global -> LDS slot (lane) of the 1 KB block at address lds; once: past the caches. Ordered
// by explicit vmcnt waits; s_nop 0 covers the M0 -> LDS-DMA hazard.
__device__ __forceinline__ void dma16(i32x4 rs, unsigned voff, unsigned soff, unsigned lds, bool once = false) {
    const unsigned l = __builtin_amdgcn_readfirstlane(lds), so = __builtin_amdgcn_readfirstlane(soff);
    if (once)
        asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen nt lds"
                     :
                     : "v"(voff), "s"(rs), "s"(so), "s"(l)
                     : "memory");
    else
        asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                     :
                     : "v"(voff), "s"(rs), "s"(so), "s"(l)
                     : "memory");
}
template <int N>
__device__ __forceinline__ void wait_vmcnt() {   // at most N vector loads of this wave still under way
    static_assert(N < 64, "vmcnt has six bits");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (0xF << 8));
    asm volatile("" ::: "memory");
}
// this wave's LDS reads have completed before any wave passes: a stage refilled after it is not still being read
__device__ __forceinline__ void block_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);   // vmcnt 63, expcnt 7: no wait; lgkmcnt 0
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// consecutive logical workgroups run on one XCD (dispatch is round-robin over the 8): the row tiles of a key/value
// head read its keys through one L2
__device__ __forceinline__ unsigned xcd_remap(unsigned bid, unsigned n) {
    const unsigned xcd = bid & 7, idx = bid >> 3, base = n >> 3, rem = n & 7;
    return (xcd < rem ? xcd * (base + 1) : rem * (base + 1) + (xcd - rem) * base) + idx;
}

template <int HD>
struct Lay {
    static constexpr int ROW = 4 * HD;         // bytes of a key's row of K or V (2 HD elements)
    static constexpr int CPR = ROW / 16;       // its chunks
    static constexpr int RPB = 64 / CPR;       // rows of a 1 KB block
    static constexpr int DT = 2 * HD / 32;     // 32-column tiles of V
    static constexpr int KS = HD / 16;         // MFMA steps of a map's width
    static __device__ __forceinline__ int ksw(int r) { return HD == 64 ? r & 15 : (r >> 1) & 7; }
    static __device__ __forceinline__ int vsw(int r) { return HD == 64 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; }
};
__device__ __forceinline__ int key_of(int i) { return 16 * (i >> 4) + 8 * ((i >> 2) & 1) + 4 * ((i >> 3) & 1) + (i & 3); }

// What a wave holds of its 32 rows: queries, running reference (log2 units), each lane's share of the sums, products
template <int HD>
struct Rows {
    i32x4 q[2][Lay<HD>::KS];
    float m[2], l[2];
    floatx16 o[2][Lay<HD>::DT];
    int lim;   // keys that the lane's row sees
};

// The lane's share of a tile's loads. Block i of a wave's holds rows r0 + i*RPB.. of the tile; row r's chunk c goes to
// slot c ^ swizzle(r). The K swizzle of block i is that of block 0 ^ 4i, the V swizzle the same for all.
template <int HD, int NB>
struct Loads {
    unsigned k[NB], v;   // byte offsets in the tile: K for each block, V (blocks RPB rows apart)
};
template <int HD, int NB>
__device__ __forceinline__ Loads<HD, NB> lane_loads(int row0, unsigned ldk, unsigned ldv, int lane) {
    using L = Lay<HD>;
    Loads<HD, NB> o;
    const int r = row0 + lane / L::CPR, c = lane % L::CPR;
#pragma unroll
    for (int i = 0; i < NB; ++i) o.k[i] = (unsigned)r * ldk + ((c ^ L::ksw(r + i * L::RPB)) << 4);
    o.v = (unsigned)r * ldv + ((c ^ L::vsw(r)) << 4);
    return o;
}
// the wave's NB blocks of K to lds, NB of V to lds + v_off; `rows` of the tile are there, the others read as zero
template <int HD, int NB>
__device__ __forceinline__ void load_tile(const Loads<HD, NB> &o, const char *kt, const char *vt, unsigned ldk, unsigned ldv, int rows,
                                          unsigned lds, unsigned v_off) {
    using L = Lay<HD>;
    const int n = rows - 1;
    const i32x4 rk = buffer(kt, n < 0 ? 0u : (unsigned)n * ldk + L::ROW), rv = buffer(vt, n < 0 ? 0u : (unsigned)n * ldv + L::ROW);
#pragma unroll
    for (int i = 0; i < NB; ++i) dma16(rk, o.k[i], i * L::RPB * ldk, lds + i * 1024);
#pragma unroll
    for (int i = 0; i < NB; ++i) dma16(rv, o.v, i * L::RPB * ldv, lds + v_off + i * 1024);
}

// LDS addresses of the lane's part of a tile of 32 rows: K row key_of(lane & 31), V row 8*(lane>>5) + (lane&15)/4. Other
// chunks are reached by ^ (bits 4 to 7), other rows, blocks and stages by +: they do not meet.
template <int HD>
__device__ __forceinline__ unsigned k_lane(int lane) {
    const int r = key_of(lane & 31);
    return r * Lay<HD>::ROW + (((lane >> 5) ^ Lay<HD>::ksw(r)) << 4);
}
template <int HD>
__device__ __forceinline__ unsigned v_lane(int lane) {
    const int r = 8 * (lane >> 5) + ((lane & 15) >> 2);
    return r * Lay<HD>::ROW + (((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ Lay<HD>::vsw(r)) << 4) + (lane & 1) * 8;
}
// S^T of both maps for 32 keys, k = k_lane + the K tile's address
template <typename T, int HD>
__device__ __forceinline__ void scores(const Rows<HD> &w, unsigned k, floatx16 (&s)[2]) {
    using L = Lay<HD>;
    i32x4 f[2][L::KS];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int ks = 0; ks < L::KS; ++ks) f[j][ks] = *(lds_i32x4 *)(k ^ ((j * (HD / 8) + ks * 2) << 4));
    __builtin_amdgcn_sched_barrier(0);   // all reads under way before the first product waits for one
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j] = zero16();
#pragma unroll
    for (int ks = 0; ks < L::KS; ++ks)   // the maps in turn: a product does not wait for the one before it
#pragma unroll
        for (int j = 0; j < 2; ++j) s[j] = mfma32(f[j][ks], w.q[j][ks], s[j], T());
}
// scores of keys that the lane's row does not see: key 0 of the 32 at k0
template <int HD>
__device__ __forceinline__ void mask_scores(const Rows<HD> &w, floatx16 (&s)[2], int k0, int lane) {
    const int left = w.lim - k0 - 8 * (lane >> 5);
#pragma unroll
    for (int r = 0; r < 16; ++r)
        if (16 * (r >> 3) + (r & 7) >= left) s[0][r] = s[1][r] = -INFINITY;
}
// sum + the two values of a register of probabilities: numerator and denominator see the same rounding
__device__ __forceinline__ float dot_ones(int v, float sum, half_t) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, v), half2_t{1, 1}, sum, false);
}
__device__ __forceinline__ float dot_ones(int v, float sum, bf16_t) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, v), bf16x2{1, 1}, sum, false);
}
// exp2(c s - m) of 16 scores, rounded, and their sum
template <typename T>
__device__ __forceinline__ float exp_scores(const floatx16 &s, float c, float m, i32x4 (&p)[2]) {
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
        const int v = pack2<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -m)), __builtin_amdgcn_exp2f(__builtin_fmaf(s[r + 1], c, -m)));
        p[r >> 3][(r & 7) >> 1] = v;
        sum = dot_ones(v, sum, T());
    }
    return sum;
}
// Probabilities of 32 keys, to the reference m of earlier ones. A reference may lie below a score as long as no
// probability nears f16's range: a lane's 16 add up to no more than `most`. Only where one exceeds that (the first block:
// m = -1e30) are the maxima taken, the references moved and O and the sums scaled; most blocks take no maximum at all.
// For f16 a reference is set 2^8 (`below`) under the maximum, so that probabilities are subnormal, in steps of 2^-24 of 1,
// from 2^-22 of the largest down (15.2 nats) and not from 2^-14: with one key 14.2 nats above 700 others of equal scores
// the others' joint weight was off by 3.7% of itself. It takes 1% (12289 rows: references at the maximum and sums to 2^12 946
// us, 2^8 under it 957, 2^10 under it 959 to 964: the further down, the more often they move). bf16 has f32's range.
template <typename T> struct Reference;
template <> struct Reference<half_t> { static constexpr float below = 8.0f, most = 32768.0f; };
template <> struct Reference<bf16_t> { static constexpr float below = 0.0f, most = 4096.0f; };
template <typename T, int HD>
__device__ __forceinline__ void probs(Rows<HD> &w, const floatx16 (&s)[2], i32x4 (&p)[2][2], float c) {
    float sum[2] = {exp_scores<T>(s[0], c, w.m[0], p[0]), exp_scores<T>(s[1], c, w.m[1], p[1])};
    if (__builtin_amdgcn_ballot_w64(!(fmaxf(sum[0], sum[1]) <= Reference<T>::most)) != 0) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float t = fmaxf(fmaxf(s[j][0], s[j][1]), s[j][2]);
#pragma unroll
            for (int r = 3; r < 15; r += 2) t = fmaxf(fmaxf(t, s[j][r]), s[j][r + 1]);
            const float mn = fmaxf(w.m[j], pair_max(fmaxf(t, s[j][15])) * c - Reference<T>::below);
            const float al = __builtin_amdgcn_exp2f(w.m[j] - mn);
            w.m[j] = mn;
            w.l[j] *= al;
#pragma unroll
            for (int d = 0; d < Lay<HD>::DT; ++d) w.o[j][d] *= al;
            sum[j] = exp_scores<T>(s[j], c, mn, p[j]);
        }
    }
    w.l[0] += sum[0];
    w.l[1] += sum[1];
}
// O^T += V^T P^T for 32 keys, v = v_lane + the V tile's address: A row = column 32d + (lane & 31) of V, keys
// 16h + 8*(lane>>5) + 0..7 by two transposing reads of four
template <typename T, int HD>
__device__ __forceinline__ void product(Rows<HD> &w, unsigned v, const i32x4 (&p)[2][2]) {
    using L = Lay<HD>;
#pragma unroll
    for (int d = 0; d < L::DT; ++d) {
        const unsigned vd = v ^ (d << 6);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int2 lo = __builtin_bit_cast(int2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vd + 16 * h * L::ROW)));
            const int2 hi = __builtin_bit_cast(int2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vd + (16 * h + 4) * L::ROW)));
            const i32x4 vf = i32x4{lo.x, lo.y, hi.x, hi.y};
            w.o[0][d] = mfma32(vf, p[0][h], w.o[0][d], T());
            w.o[1][d] = mfma32(vf, p[1][h], w.o[1][d], T());
        }
    }
}
// Row x of a key/value head: its query and head within the group
struct RowOf {
    int qi, hg;
};
__device__ __forceinline__ RowOf row_of(int x, int G) {
    const int qi = G == 1 ? x : x / G;
    return RowOf{qi, x - qi * G};
}

template <typename T, int HD>
__device__ __forceinline__ void load_rows(Rows<HD> &w, const DiffAttnArgs &a, int b, int g, int G, int x, int nq, int nk, int lane) {
    using L = Lay<HD>;
    const RowOf ro = row_of(x, G);
    const bool in = ro.qi < nq;   // other lanes compute with query 0 and are not stored
    const T *q = (const T *)a.q + (long long)b * a.bsq + (long long)(in ? ro.qi : 0) * a.ldq + (g * G + (in ? ro.hg : 0)) * 2 * HD + 8 * (lane >> 5);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int ks = 0; ks < L::KS; ++ks) w.q[j][ks] = *(const i32x4 *)(q + j * HD + ks * 16);
        w.m[j] = -1e30f;
        w.l[j] = 0.0f;
#pragma unroll
        for (int d = 0; d < L::DT; ++d) w.o[j][d] = zero16();
    }
    w.lim = !in ? 0 : a.causal ? min(nk, max(0, ro.qi + nk - nq + 1)) : nk;
}

// lambda of the lane's head
__device__ __forceinline__ float row_lambda(const DiffAttnArgs &a, int g, int G, int hg, int lane) {
    if (a.lam_heads == 1) return wave_lambda(a, 0, lane);
    float lam = 0.0f;
    for (int i = 0; i < G; ++i) {
        const float v = wave_lambda(a, g * G + i, lane);
        if (hg == i) lam = v;
    }
    return lam;
}

// How a launch's work is cut. A tile is TR rows of one key/value head of one sample, its keys are units of KB. The first
// `full` tiles have a workgroup each. The units of the others, one after the other, are shared out evenly among `shared`
// workgroups; their pieces of tiles go to the workspace and are joined by diff_attn_join_kernel. A piece's place there is
// its workgroup's number plus its tile's: both only grow along the units, and one of them does at every cut.
struct DiffPlan {
    int ntile;          // tiles of a key/value head
    int tiles, units;   // of all heads and samples; of a tile (by Sk)
    int full, shared;
    int by_len;         // full = 0 and lengths are given: the units are counted by them
    int ranked;         // causal, full = tiles, lengths that differ or heads that do not go round the XCDs: see ranked_part
    int groups;         // workgroups of a tile that join its rows
    float *o;           // [piece][row of the tile][map][2 HD]: products with V, not divided
    float4 *st;         // [piece][row of the tile]: reference and sum of each map
};
struct Share {   // shared workgroup p's units begin at p*q + min(p, r)
    unsigned q, r;
    __device__ __forceinline__ unsigned begin(unsigned p) const { return p * q + min(p, r); }
    __device__ __forceinline__ unsigned holder(unsigned u) const { return u < r * (q + 1) ? u / (q + 1) : r + (u - r * (q + 1)) / q; }
};
// sum over the lanes up to this one: within rows of 16, then from row to row
__device__ __forceinline__ unsigned lane_prefix(unsigned v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}
// The samples' units by their lengths, 64 samples at a time: lane i looks at sample b0 + i, which has nkv * tiles * n
// units (tiles of a head, units of a tile)
template <int TR, int KB>
struct ByLen {
    int b0, nq, nk, tiles;
    unsigned n, own, upto;   // units of the lane's sample, and up to and with it of the 64
    __device__ __forceinline__ void look(const DiffAttnArgs &a, int from, int lane) {
        b0 = from;
        const int b = min(from + lane, (int)a.B - 1);
        nq = q_rows(a, b);
        nk = kv_rows(a, b);
        tiles = (int)(((unsigned)nq * (a.nh / a.nkv) + TR - 1) / TR);
        n = (unsigned)max(1, (nk + KB - 1) / KB);
        own = from + lane < (int)a.B ? a.nkv * tiles * n : 0;
        upto = lane_prefix(own);
    }
    __device__ __forceinline__ unsigned all() const { return __builtin_amdgcn_readlane(upto, 63); }
    // of all samples; the first 64 are being looked at before and after
    __device__ __forceinline__ unsigned total(const DiffAttnArgs &a, int lane) {
        unsigned t = all();
        for (int from = 64; from < (int)a.B; from += 64) {
            ByLen x;
            x.look(a, from, lane);
            t += x.all();
        }
        return t;
    }
};
// A tile and some of its units
struct Part {
    int b, g, tile, nq, nk, u0, u1, n, place;   // n: units of the tile; place: the tile's number among all (static)
};
__device__ __forceinline__ int tile_order(const DiffAttnArgs &a, int heads, int i) { return a.causal ? heads - 1 - i : i; }   // the longest first
// unit u and what follows it in its tile, up to unit end
template <int TR, int KB>
__device__ __forceinline__ Part part_at(const DiffAttnArgs &a, const DiffPlan &pl, const ByLen<TR, KB> &first64, unsigned u, unsigned end, int lane) {
    Part p;
    int heads = pl.ntile, in_sample;
    if (pl.by_len) {
        ByLen<TR, KB> x = first64;
        unsigned before = 0;
        while (u >= before + x.all() && x.b0 + 64 < (int)a.B) {
            before += x.all();
            x.look(a, x.b0 + 64, lane);
        }
        const int i = __ffsll((unsigned long long)__builtin_amdgcn_ballot_w64(before + x.upto > u)) - 1;
        p.b = x.b0 + i;
        p.nq = __builtin_amdgcn_readlane(x.nq, i);
        p.nk = __builtin_amdgcn_readlane(x.nk, i);
        p.n = __builtin_amdgcn_readlane(x.n, i);
        heads = __builtin_amdgcn_readlane(x.tiles, i);
        const unsigned in = u - before - __builtin_amdgcn_readlane(x.upto - x.own, i);
        in_sample = (int)(in / (unsigned)p.n);
        p.u0 = (int)(in - in_sample * (unsigned)p.n);
        p.g = in_sample / heads;
    } else {
        const int ts = (int)(u / (unsigned)pl.units), t = pl.full + ts, bg = t / pl.ntile;
        p.u0 = (int)(u - (unsigned)ts * pl.units);
        p.n = pl.units;
        p.b = bg / (int)a.nkv;
        p.g = bg - p.b * (int)a.nkv;
        p.nq = q_rows(a, p.b);
        p.nk = kv_rows(a, p.b);
        in_sample = t - p.b * (int)a.nkv * pl.ntile;
    }
    const int i = in_sample - p.g * heads;
    p.tile = tile_order(a, heads, i);
    p.u1 = (int)min((unsigned)p.n, p.u0 + (end - u));
    p.place = (p.b * (int)a.nkv + p.g) * pl.ntile + tile_order(a, pl.ntile, p.tile) - pl.full;
    return p;
}

// Causal tiles are up to twice the mean length, and a CU's workgroups share it: started longest first, a CU gets two or
// three of the longest and works on them when the others have ended. Lengths of 677 to 2047 rows, hd 32: 65.5 us in
// the order of the static shapes, 51 as below; two samples of 8192 and 5620 rows, 2 heads of 4: 498, 325.
//
// Blocks of n workgroups of `all` behind the first turned round: n CUs get one of each block, the one with the longest of
// the first the shortest of the others (every other block turned round: 2% slower)
__device__ __forceinline__ int mirrored(int i, int n, int all) {
    const int block = i / n, first = block * n;
    return block ? first + min(n, all - first) - 1 - (i - first) : i;
}
// Causal tiles of up to 64 samples of unequal length, longest first over all: a sample's tiles end at level
// nk*G/TR, one level apart. Sets b, nq, nk, g, tile and returns whether there is a tile of the workgroup's rank. Samples
// of a multiple of eight heads give each XCD an eighth of them, and it ranks its own.
template <int TR, int WAVES>
__device__ __forceinline__ bool ranked_part(const DiffAttnArgs &a, const DiffPlan &pl, Part &p, int lane) {
    const int xcds = a.nkv % 8 == 0 ? 8 : 1, nkv = (int)a.nkv / xcds, cus = 256 / xcds, all = pl.full / xcds;
    int i = (int)blockIdx.x / xcds;
    const int b = min(lane, (int)a.B - 1), G = (int)(a.nh / a.nkv);
    const int nq = q_rows(a, b), nk = kv_rows(a, b);
    const int tiles = lane < (int)a.B ? (int)(((unsigned)nq * G + TR - 1) / TR) : 0, top = (int)((unsigned)nk * G / TR);
    auto from = [&](int level) {   // tiles of the level and above, up to and with the lane's sample
        return lane_prefix((unsigned)(nkv * min(max(top - level + 1, 0), tiles)));
    };
    int lo = -(int)pl.ntile, hi = (int)(a.Sk * G / TR);   // every tile is at lo or above, none above hi
    const int n = (int)__builtin_amdgcn_readlane(from(lo), 63);
    if (n <= WAVES * cus) i = mirrored(i, cus, all);
    if (i >= n) return false;
    while (lo < hi) {   // the highest level with more than i tiles from it on
        const int mid = lo + (hi - lo + 1) / 2;
        if ((int)__builtin_amdgcn_readlane(from(mid), 63) > i) lo = mid;
        else hi = mid - 1;
    }
    const unsigned above = __builtin_amdgcn_readlane(from(lo + 1), 63), rest = (unsigned)i - above;
    const unsigned own = top - lo >= 0 && top - lo < tiles ? nkv : 0, upto = lane_prefix(own);
    const int at = __ffsll((unsigned long long)__builtin_amdgcn_ballot_w64(upto > rest)) - 1;
    p.b = at;
    p.nq = __builtin_amdgcn_readlane(nq, at);
    p.nk = __builtin_amdgcn_readlane(nk, at);
    p.g = (int)(rest - __builtin_amdgcn_readlane(upto - own, at)) * xcds + (int)blockIdx.x % xcds;
    p.tile = __builtin_amdgcn_readlane(tiles - 1 - (top - lo), at);
    return true;
}

// A workgroup's worker: 128 rows, 32 a wave. The four waves share K and V tiles of 64 keys, two stages in LDS: the next is
// loaded while one is worked on. Two workgroups a CU (hd 32: three), one's matrix products cover the other's softmax.
// Measured (calls in a row; the first hundred after a pause take up to 18% longer, until the clocks have settled): 12289
// rows and keys, 8 heads, hd 64, f16: 950 to 967 us, 960 to 980 TFLOP/s of the 12 hd operations a pair (matrix units half
// busy at 1.9 GHz, which the power limit leaves; a library bf16 product of 8192^3 reaches 1259). 1101 rows, 128 heads, bf16: 149
// to 152 us, 790 (matrix units 0.31 busy: half a round of tiles at the end, 18 key tiles between a tile's start and end). One
// wave a SIMD, the products of a step beside the softmax of the one before: 1500 us for the first; 64 rows a workgroup and
// two waves that share the keys: spills. Causal, hd 32, 677 to 2047 rows of four heads a key, f16: 50.3 us.
template <typename T, int HD>
struct Wide {
    using L = Lay<HD>;
    static constexpr int TR = 128, KB = 64;
    static constexpr int OP = KB * L::ROW, STAGE = 2 * OP, SUB = 32 * L::ROW;
    static constexpr int NB = OP / 1024 / 4;         // 1 KB blocks of K, of V, a wave and unit
    static constexpr int LDS = 2 * STAGE, WAVES = HD == 32 ? 3 : 2;

    // units of a tile; a piece of it (to the workspace) or, piece < 0, all of it
    static __device__ __forceinline__ void run(const DiffAttnArgs &a, const DiffPlan &pl, char *smem, const Part &t, int piece) {
        const unsigned lds = (unsigned)(unsigned long)(lds_char *)smem;
        const int lane = threadIdx.x & 63;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int b = t.b, g = t.g, G = (int)(a.nh / a.nkv), nq = t.nq, nk = t.nk;
        const int x0 = t.tile * TR;
        if (x0 / G >= nq) return;   // the whole workgroup: no row of the tile is there
        const int x = x0 + wave * 32 + (lane & 31);
        // keys that any row of the tile and every row of the wave sees
        auto limit = [&](int xr) {
            const int qi = min(row_of(xr, G).qi, nq - 1);
            return a.causal ? min(nk, max(0, qi + nk - nq + 1)) : nk;
        };
        const int keys = limit(x0 + TR - 1), all = limit(x0 + wave * 32);
        const char *kp = (const char *)((const T *)a.k + (long long)b * a.bsk + g * 2 * HD);
        const char *vp = (const char *)((const T *)a.v + (long long)b * a.bsv + g * 2 * HD);
        const unsigned ldk = a.ldk * 2, ldv = a.ldv * 2;
        const Loads<HD, NB> lo = lane_loads<HD, NB>(wave * NB * L::RPB, ldk, ldv, lane);
        const unsigned kl = lds + k_lane<HD>(lane), vl = lds + OP + v_lane<HD>(lane);
        auto issue = [&](int u) {
            const long long k0 = (long long)u * KB;
            load_tile<HD, NB>(lo, kp + k0 * ldk, vp + k0 * ldv, ldk, ldv, min(KB, nk - u * KB), lds + (u & 1) * STAGE + wave * NB * 1024, OP);
        };
        const float c = score_factor(a);
        const int end = min(t.u1, (keys + KB - 1) / KB);
        block_barrier();   // an earlier piece's LDS has been read
        if (t.u0 < end) issue(t.u0);
        Rows<HD> w;
        load_rows<T, HD>(w, a, b, g, G, x, nq, nk, lane);
        const RowOf ro = row_of(x, G);
        const float lam = piece < 0 ? row_lambda(a, g, G, ro.hg, lane) : 0.0f;   // loaded beside the first keys
        for (int u = t.u0; u < end; ++u) {
            wait_vmcnt<0>();
            block_barrier();
            if (u + 1 < end) issue(u + 1);
            const unsigned at = (u & 1) * STAGE;
#pragma unroll   // one block's start beside the other's end: hd 32, as above, 51.1 -> 48.6 us; hd 64 1 to 4%
            for (int i = 0; i < KB / 32; ++i) {
                const int k0 = u * KB + 32 * i;
                floatx16 s[2];
                i32x4 p[2][2];
                scores<T, HD>(w, kl + at + i * SUB, s);
                if (k0 + 32 > all) mask_scores<HD>(w, s, k0, lane);
                probs<T, HD>(w, s, p, c);
                product<T, HD>(w, vl + at + i * SUB, p);
            }
        }
        const float l0 = pair_sum(w.l[0]), l1 = pair_sum(w.l[1]);
        // value r of tile d is column 32d + 8(r>>2) + 4*(lane>>5) + (r&3)
        const int col0 = 4 * (lane >> 5);
        if (piece >= 0) {
            if (ro.qi >= nq) return;
            const long long row = (long long)piece * TR + wave * 32 + (lane & 31);
            if (lane < 32) pl.st[row] = make_float4(w.m[0], l0, w.m[1], l1);
            float *to = pl.o + row * (4 * HD) + col0;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int d = 0; d < L::DT; ++d)
#pragma unroll
                    for (int r = 0; r < 16; r += 4)
                        *(float4 *)(to + j * 2 * HD + 32 * d + 2 * r) = make_float4(w.o[j][d][r], w.o[j][d][r + 1], w.o[j][d][r + 2], w.o[j][d][r + 3]);
            return;
        }
        const float r0 = l0 > 0.0f ? 1.0f / l0 : 0.0f, r1 = l1 > 0.0f ? lam / l1 : 0.0f;
        float ss = 0.0f;
#pragma unroll
        for (int d = 0; d < L::DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float y = w.o[0][d][r] * r0 - w.o[1][d][r] * r1;
                w.o[0][d][r] = y;
                ss += y * y;
            }
        ss = pair_sum(ss);
        if (ro.qi >= nq) return;
        if (a.norm_w) {
            const float f = rms_factor<HD>(a, ss);
            const float *nw = a.norm_w + col0;
#pragma unroll
            for (int d = 0; d < L::DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) w.o[0][d][r] = w.o[0][d][r] * f * nw[32 * d + 8 * (r >> 2) + (r & 3)];
        }
        T *out = (T *)a.out + (long long)b * a.bso + (long long)ro.qi * a.ldo + (g * G + ro.hg) * 2 * HD + col0;
#pragma unroll
        for (int d = 0; d < L::DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *(int2 *)(out + 32 * d + 2 * r) = make_int2(pack2<T>(w.o[0][d][r], w.o[0][d][r + 1]), pack2<T>(w.o[0][d][r + 2], w.o[0][d][r + 3]));
    }
};

// A workgroup's worker for few rows: 16, the same in all four waves. Wave w takes keys 32w.. of every unit of 128, which it
// alone reads: it loads them into LDS of its own and waits for nothing but its own loads, K of the next unit under way
// as soon as this one's is in registers, V likewise. The waves' products are merged at the end through LDS.
// 16x16x32 MFMA (A row and B column = lane & 15, K group g = lane >> 4, D[4g + r][lane & 15], r = 0..3), operands as in
// the wide kernel: row i of the two products over 32 keys' K takes keys 8(i>>2) + (i&3) and 4 more, so that a lane has
// keys 8g + 0..7 of query lane & 15.
typedef floatx4 f32x4;
__device__ __forceinline__ f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c, half_t) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c, bf16_t) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// the four lanes of a query (l, l ^ 16, l ^ 32, l ^ 48) get the maximum, the sum
__device__ __forceinline__ float quad_max(float v) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return pair_max(fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1])));
}
__device__ __forceinline__ float quad_sum(float v) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return pair_sum(__uint_as_float(p[0]) + __uint_as_float(p[1]));
}
// Measured: 64 caches of 2048 to 8192 keys, 4 heads of 4 rows, bf16: 121 us with the join, 5.8 TB/s of K and V (a large copy
// on this card: 6.2); one row over 4099 keys, 8 heads: 12.3 us (traced: 8.6 and 4.2 for the join), all latency; two samples of 397
// rows, 8 heads: 11 us (32 rows a workgroup that share their tiles: 13.1).
template <typename T, int HD>
struct Few {
    using L = Lay<HD>;
    static constexpr int TR = 16, KB = 128;
    static constexpr int KS = HD / 32, DT = 2 * HD / 16;   // MFMA steps of a map's width; 16-column tiles of V
    static constexpr int OP = 32 * L::ROW, NB = OP / 1024; // a wave's K (V) tile and its 1 KB blocks
    static constexpr int NO = DT * 4, NQ = NO / 4;         // products of a lane and map; those that it has after the merge
    static constexpr int LDS = 8 * OP + 4 * 64 * 5 * 4, WAVES = HD == 32 ? 3 : 2;
    static_assert(4 * 2 * NO * 256 <= 8 * OP, "the products fit in the tiles");
    // the 16 K rows of a read differ in bits 0, 1, 3, 4, the 8 V rows of half a wave in bits 0, 1, 3 (32 bytes each)
    static __device__ __forceinline__ int ksw(int r) {
        return HD == 64 ? (r & 3) | ((r >> 3) & 3) << 2 : ((r >> 1) & 1) | ((r >> 3) & 3) << 1;
    }
    static __device__ __forceinline__ int vsw(int r) {
        return HD == 64 ? ((r & 3) | ((r >> 3) & 1) << 2) << 1 : (((r >> 1) & 1) | ((r >> 3) & 1) << 1) << 1;
    }

    static __device__ __forceinline__ float exps(const f32x4 (&s)[2], float c, float m, i32x4 &p) {
        float sum = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                const int v = pack2<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[h][r], c, -m)), __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][r + 1], c, -m)));
                p[2 * h + r / 2] = v;
                sum = dot_ones(v, sum, T());
            }
        return sum;
    }

    static __device__ __forceinline__ void run(const DiffAttnArgs &a, const DiffPlan &pl, char *smem, const Part &t, int piece) {
        const int lane = threadIdx.x & 63, g4 = lane >> 4, l16 = lane & 15;
        const int kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int b = t.b, g = t.g, G = (int)(a.nh / a.nkv), nq = t.nq, nk = t.nk;
        const int x0 = t.tile * TR;
        if (x0 / G >= nq) return;   // the whole workgroup: no row of the tile is there
        const RowOf ro = row_of(x0 + l16, G);
        const bool in = ro.qi < nq;   // other lanes compute with query 0 and are not stored
        auto limit = [&](int qi) { return a.causal ? min(nk, max(0, qi + nk - nq + 1)) : nk; };
        const int keys = limit(min(row_of(x0 + TR - 1, G).qi, nq - 1)), all = limit(row_of(x0, G).qi);
        const int lim = in ? limit(ro.qi) : 0;
        const int end = min(t.u1, (keys + KB - 1) / KB);
        // the wave's tiles, and the lane's share of their loads
        const unsigned sk = (unsigned)(unsigned long)(lds_char *)smem + kw * 2 * OP, sv = sk + OP;
        const char *kp = (const char *)((const T *)a.k + (long long)b * a.bsk + g * 2 * HD);
        const char *vp = (const char *)((const T *)a.v + (long long)b * a.bsv + g * 2 * HD);
        const unsigned ldk = a.ldk * 2, ldv = a.ldv * 2;
        const int lr = lane / L::CPR, lc = lane % L::CPR;
        unsigned ok[NB], ov[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int r = lr + i * L::RPB;
            ok[i] = (unsigned)r * ldk + ((lc ^ ksw(r)) << 4);
            ov[i] = (unsigned)r * ldv + ((lc ^ vsw(r)) << 4);
        }
        auto load = [&](int u, const char *p, unsigned ld, const unsigned (&o)[NB], unsigned to) {
            const int k0 = u * KB + 32 * kw, n = min(32, nk - k0) - 1;   // rows behind the last key read as zero
            const i32x4 rs = buffer(p + (long long)k0 * ld, n < 0 ? 0u : (unsigned)n * ld + L::ROW);
            // A head with one tile reads its keys once: past the caches, at every size. Bytes of K and V, us past them and
            // through them: 16.8 MB 12.9, 13.5; 67 MB 30.0, 31.4; 268 MB 46.6, 53.3; 1074 MB 168, 185, with other
            // caches read in between, as between the steps of a model. Read again at once: 10.9, 10.9; 28.9, 21.9; 46.0, 44.2.
            if (pl.ntile == 1) {
#pragma unroll
                for (int i = 0; i < NB; ++i) dma16(rs, o[i], 0, to + i * 1024, true);
            } else {
#pragma unroll
                for (int i = 0; i < NB; ++i) dma16(rs, o[i], 0, to + i * 1024);
            }
        };
        wait_vmcnt<0>();   // an earlier piece's stores are not counted among the loads below
        block_barrier();   // its LDS has been read
        if (t.u0 < end) {
            load(t.u0, kp, ldk, ok, sk);
            load(t.u0, vp, ldv, ov, sv);
        }
        const T *q = (const T *)a.q + (long long)b * a.bsq + (long long)(in ? ro.qi : 0) * a.ldq + (g * G + (in ? ro.hg : 0)) * 2 * HD + 8 * g4;
        i32x4 qf[2][KS];
        f32x4 o[2][DT];
        float m[2] = {-1e30f, -1e30f}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) qf[j][ks] = *(const i32x4 *)(q + j * HD + ks * 32);
#pragma unroll
            for (int d = 0; d < DT; ++d) o[j][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        // after the merge value i of the wave's is column 16*(d0 + i/4) + 4*g4 + i%4
        const int col0 = 16 * (DT / 4) * kw + 4 * g4;
        float lam = 0.0f, nw[NQ];
        if (piece < 0) {
            lam = row_lambda(a, g, G, ro.hg, lane);
#pragma unroll
            for (int i = 0; i < NQ; ++i) nw[i] = a.norm_w ? a.norm_w[col0 + 16 * (i >> 2) + (i & 3)] : 1.0f;
        }
        const float c = score_factor(a);
        // K row 8*(l16>>2) + (l16&3), chunk g4; V row 8*g4 + (l16>>2), column 4*(l16&3)
        const int kr = 8 * (l16 >> 2) + (l16 & 3), vr = 8 * g4 + (l16 >> 2);
        const unsigned kl = sk + kr * L::ROW + ((g4 ^ ksw(kr)) << 4);
        const unsigned vl = sv + vr * L::ROW + ((((l16 & 3) >> 1) ^ vsw(vr)) << 4) + (l16 & 1) * 8;
        asm volatile("" ::: "memory");
        for (int u = t.u0; u < end; ++u) {
            const bool more = u + 1 < end;
            wait_vmcnt<NB>();   // K is there; V's NB blocks may still be under way
            i32x4 kf[2][2][KS];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) kf[j][h][ks] = *(lds_i32x4 *)((kl ^ ((j * (HD / 8) + ks * 4) << 4)) + 4 * h * L::ROW);
            __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt 0: the tile is in registers
            asm volatile("" ::: "memory");
            if (more) load(u + 1, kp, ldk, ok, sk);
            f32x4 s[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) s[j][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) s[j][h] = mfma16(kf[j][h][ks], qf[j][ks], s[j][h], T());
            const int k0 = u * KB + 32 * kw;
            if (k0 + 32 > all) {
                const int left = lim - k0 - 8 * g4;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (4 * h + r >= left) s[0][h][r] = s[1][h][r] = -INFINITY;
            }
            i32x4 p[2];
            float sum[2] = {exps(s[0], c, m[0], p[0]), exps(s[1], c, m[1], p[1])};
            if (__builtin_amdgcn_ballot_w64(!(fmaxf(sum[0], sum[1]) <= Reference<T>::most)) != 0) {   // as in probs
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float top = fmaxf(fmaxf(fmaxf(s[j][0][0], s[j][0][1]), fmaxf(s[j][0][2], s[j][0][3])),
                                            fmaxf(fmaxf(s[j][1][0], s[j][1][1]), fmaxf(s[j][1][2], s[j][1][3])));
                    const float mn = fmaxf(m[j], quad_max(top) * c - Reference<T>::below);
                    const float al = __builtin_amdgcn_exp2f(m[j] - mn);
                    m[j] = mn;
                    l[j] *= al;
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[j][d] *= al;
                    sum[j] = exps(s[j], c, mn, p[j]);
                }
            }
            l[0] += sum[0];
            l[1] += sum[1];
            if (more) wait_vmcnt<NB>();   // V is there; the next K's NB blocks may still be under way
            else wait_vmcnt<0>();
            i32x4 vf[DT];
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const unsigned vd = vl ^ (d << 5);
                const int2 lo = __builtin_bit_cast(int2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)vd));
                const int2 hi = __builtin_bit_cast(int2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vd + 4 * L::ROW)));
                vf[d] = i32x4{lo.x, lo.y, hi.x, hi.y};
            }
            __builtin_amdgcn_s_waitcnt(0xC07F);
            asm volatile("" ::: "memory");
            if (more) load(u + 1, vp, ldv, ov, sv);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int j = 0; j < 2; ++j) o[j][d] = mfma16(vf[d], p[j], o[j][d], T());
        }
        // every wave leaves its products in LDS (a lane's four are 16 bytes, lanes next to each other) and takes a quarter of all
        float4 *prod = (float4 *)smem + lane;
        float4 *st = (float4 *)(smem + 8 * OP) + lane;
        block_barrier();   // the tiles have been read
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int d = 0; d < DT; ++d) prod[(kw * 2 * DT + j * DT + d) * 64] = make_float4(o[j][d][0], o[j][d][1], o[j][d][2], o[j][d][3]);
        st[kw * 64] = make_float4(m[0], quad_sum(l[0]), m[1], quad_sum(l[1]));
        block_barrier();
        float f[2][4], y[2][NQ];
        m[0] = m[1] = -1e30f;
        l[0] = l[1] = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float4 v = st[k * 64];
            m[0] = fmaxf(m[0], v.x);
            m[1] = fmaxf(m[1], v.z);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float4 v = st[k * 64];
            f[0][k] = __builtin_amdgcn_exp2f(v.x - m[0]);
            f[1][k] = __builtin_amdgcn_exp2f(v.z - m[1]);
            l[0] += v.y * f[0][k];
            l[1] += v.w * f[1][k];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < NQ; i += 4) {
                float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float4 v = prod[(k * 2 * DT + j * DT + kw * (DT / 4) + i / 4) * 64];
                    s.x += v.x * f[j][k];
                    s.y += v.y * f[j][k];
                    s.z += v.z * f[j][k];
                    s.w += v.w * f[j][k];
                }
                y[j][i] = s.x;
                y[j][i + 1] = s.y;
                y[j][i + 2] = s.z;
                y[j][i + 3] = s.w;
            }
        if (piece >= 0) {
            if (!in) return;
            const long long row = (long long)piece * TR + l16;
            if (g4 == 0 && kw == 0) pl.st[row] = make_float4(m[0], l[0], m[1], l[1]);
            float *to = pl.o + row * (4 * HD) + col0;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < NQ; i += 4) *(float4 *)(to + j * 2 * HD + 4 * i) = make_float4(y[j][i], y[j][i + 1], y[j][i + 2], y[j][i + 3]);
            return;
        }
        const float r0 = l[0] > 0.0f ? 1.0f / l[0] : 0.0f, r1 = l[1] > 0.0f ? lam / l[1] : 0.0f;
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            y[0][i] = y[0][i] * r0 - y[1][i] * r1;
            ss += y[0][i] * y[0][i];
        }
        if (a.norm_w) {   // the row's squares over the waves, in their order
            float *red = (float *)(smem + 8 * OP + 4 * 64 * 16) + lane;
            red[kw * 64] = quad_sum(ss);
            block_barrier();
            ss = ((red[0] + red[64]) + red[128]) + red[192];
            const float fn = rms_factor<HD>(a, ss);
#pragma unroll
            for (int i = 0; i < NQ; ++i) y[0][i] = y[0][i] * fn * nw[i];
        }
        if (!in) return;
        T *out = (T *)a.out + (long long)b * a.bso + (long long)ro.qi * a.ldo + (g * G + ro.hg) * 2 * HD + col0;
#pragma unroll
        for (int i = 0; i < NQ; i += 4)
            *(int2 *)(out + 4 * i) = make_int2(pack2<T>(y[0][i], y[0][i + 1]), pack2<T>(y[0][i + 2], y[0][i + 3]));
    }
};

template <int TR, int KB>
__device__ __forceinline__ Share shares(const DiffAttnArgs &a, const DiffPlan &pl, ByLen<TR, KB> &x, int lane) {
    unsigned U = (unsigned)(pl.tiles - pl.full) * pl.units;
    if (pl.by_len) {
        x.look(a, 0, lane);
        U = x.total(a, lane);
    }
    const unsigned q = U / (unsigned)pl.shared;
    return Share{q, U - q * pl.shared};
}

template <typename T, int HD, typename A>
__global__ __launch_bounds__(256, A::WAVES) void diff_attn_kernel(const DiffAttnArgs a, const DiffPlan pl) {
    __shared__ __attribute__((aligned(1024))) char smem[A::LDS];
    const int lane = threadIdx.x & 63, nkv = (int)a.nkv;
    if ((int)blockIdx.x < pl.full) {
        Part p;
        if (pl.ranked) {
            if (!ranked_part<A::TR, A::WAVES>(a, pl, p, lane)) return;
        } else {
            // workgroups go round the 8 XCDs in turn. A head's tiles stay on one, for its L2; heads go round too, so that a
            // short sample's are not all on one; causal tiles the longest first, over all the XCD's heads
            const int heads = nkv * (int)a.B;
            int bg, i;
            if (heads % 8 == 0 && pl.full == pl.tiles) {
                const int per = heads / 8, n = pl.full / 8;
                int idx = (int)blockIdx.x >> 3;
                if (a.causal && n <= A::WAVES * 32) idx = mirrored(idx, 32, n);
                i = a.causal ? idx / per : idx % pl.ntile;
                bg = (a.causal ? idx - i * per : idx / pl.ntile) * 8 + ((int)blockIdx.x & 7);
            } else {
                const int t = (int)xcd_remap(blockIdx.x, pl.full);
                bg = t / pl.ntile;
                i = t - bg * pl.ntile;
            }
            p.b = bg / nkv;
            p.g = bg - p.b * nkv;
            p.tile = tile_order(a, pl.ntile, i);
            p.nq = q_rows(a, p.b);
            p.nk = kv_rows(a, p.b);
        }
        p.u0 = 0;
        p.u1 = pl.units;
        A::run(a, pl, smem, p, -1);
        return;
    }
    const int p = (int)xcd_remap(blockIdx.x - pl.full, pl.shared);
    ByLen<A::TR, A::KB> first64{};
    const Share sh = shares(a, pl, first64, lane);
    const unsigned end = sh.begin(p + 1);
    for (unsigned u = sh.begin(p); u < end;) {
        const Part t = part_at(a, pl, first64, u, end, lane);
        u += t.u1 - t.u0;
        A::run(a, pl, smem, t, t.u0 == 0 && t.u1 == t.n ? -1 : p + t.place);
    }
}

// Joins the pieces of the shared tiles, in the order of their keys: HD/2 lanes a row, four columns of each map a lane.
// PG groups of lanes take a row's pieces in turn (as many as a workgroup has beside few rows) and are merged in LDS.
// A launch of its own: 4 us behind one row over 4099 keys. The last workgroup of a tile joining it instead, by tickets,
// takes device-wide fences that write back and drop an XCD's L2: 12.2 -> 15.3 us there, 140 -> 175 for 64 caches.
template <typename T, int HD, int TR, int KB, int PG>
__global__ __launch_bounds__(256) void diff_attn_join_kernel(const DiffAttnArgs a, const DiffPlan pl) {
    constexpr int LR = HD / 2, RPW = 256 / LR / PG;   // rows of a workgroup
    __shared__ float4 part[PG > 1 ? 2 * 256 : 1];
    __shared__ float4 stat[PG > 1 ? 256 / LR : 1];
    const int lane = threadIdx.x & (LR - 1), team = (int)threadIdx.x / LR, rr = team % RPW, pg = team / RPW;
    const int ts = (int)(blockIdx.x / (unsigned)pl.groups), r0 = (int)(blockIdx.x - (unsigned)ts * pl.groups) * RPW, r = r0 + rr;
    const int t = pl.full + ts, bg = t / pl.ntile, nkv = (int)a.nkv;
    const int b = bg / nkv, g = bg - b * nkv, G = (int)(a.nh / a.nkv);
    const int tile = tile_order(a, pl.ntile, t - bg * pl.ntile);
    const int nq = q_rows(a, b);
    if ((tile * TR + r0) / G >= nq) return;   // the whole workgroup
    ByLen<TR, KB> x{};
    const int wl = threadIdx.x & 63;
    const Share sh = shares(a, pl, x, wl);
    unsigned first = (unsigned)ts * pl.units, n = pl.units;
    if (pl.by_len) {
        unsigned before = 0;
        while (x.b0 + 64 <= b) {
            before += x.all();
            x.look(a, x.b0 + 64, wl);
        }
        const int i = b - x.b0, heads = __builtin_amdgcn_readlane(x.tiles, i);
        n = __builtin_amdgcn_readlane(x.n, i);
        first = before + __builtin_amdgcn_readlane(x.upto - x.own, i) + (unsigned)(g * heads + tile_order(a, heads, tile)) * n;
    }
    const int p0 = (int)sh.holder(first), p1 = (int)sh.holder(first + n - 1);
    if (p0 == p1) return;   // in one piece: written already
    const RowOf ro = row_of(tile * TR + r, G);
    const bool in = ro.qi < nq;
    const int h = g * G + (in ? ro.hg : 0);
    // loaded beside the pieces
    const float *lv = a.lam + (a.lam_heads > 1 ? (long long)h * 4 * HD : 0) + 2 * lane;
    const float2 lq1 = make_float2(lv[0], lv[1]), lk1 = make_float2(lv[HD], lv[HD + 1]);
    const float2 lq2 = make_float2(lv[2 * HD], lv[2 * HD + 1]), lk2 = make_float2(lv[3 * HD], lv[3 * HD + 1]);
    float nw[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) nw[e] = a.norm_w ? a.norm_w[4 * lane + e] : 1.0f;
    float m[2] = {-1e30f, -1e30f}, l[2] = {0.0f, 0.0f};
    float4 o[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    // one more part: the larger reference, what was before scaled to it
    auto add = [&](int j, float mp, float lp, float4 v) {
        const float mn = fmaxf(m[j], mp);
        const float f = __builtin_amdgcn_exp2f(m[j] - mn), w = __builtin_amdgcn_exp2f(mp - mn);
        m[j] = mn;
        l[j] = l[j] * f + lp * w;
        o[j] = make_float4(o[j].x * f + v.x * w, o[j].y * f + v.y * w, o[j].z * f + v.z * w, o[j].w * f + v.w * w);
    };
    if (in)
#pragma unroll 2
        for (int p = p0 + pg; p <= p1; p += PG) {
            const long long row = (long long)(p + ts) * TR + r;
            const float4 st = pl.st[row];
            const float4 *v = (const float4 *)(pl.o + row * (4 * HD)) + lane;
            const float4 v0 = v[0], v1 = v[HD / 2];
            add(0, st.x, st.y, v0);
            add(1, st.z, st.w, v1);
        }
    if constexpr (PG > 1) {
        part[threadIdx.x] = o[0];
        part[256 + threadIdx.x] = o[1];
        if (lane == 0) stat[team] = make_float4(m[0], l[0], m[1], l[1]);
        __syncthreads();
        if (pg > 0) return;
#pragma unroll
        for (int k = 1; k < PG; ++k) {
            const float4 st = stat[k * RPW + rr];
            add(0, st.x, st.y, part[k * RPW * LR + threadIdx.x]);
            add(1, st.z, st.w, part[256 + k * RPW * LR + threadIdx.x]);
        }
    }
    auto row_sum = [&](float v) {
        v = row16_sum(v);
        if constexpr (LR == 32) {
            const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
            v = __uint_as_float(q[0]) + __uint_as_float(q[1]);
        }
        return v;
    };
    const float d1 = row_sum(lq1.x * lk1.x + lq1.y * lk1.y), d2 = row_sum(lq2.x * lk2.x + lq2.y * lk2.y);
    const float lam = expf(d1) - expf(d2) + a.lambda_init;
    const float i0 = l[0] > 0.0f ? 1.0f / l[0] : 0.0f, i1 = l[1] > 0.0f ? lam / l[1] : 0.0f;
    float y[4] = {o[0].x * i0 - o[1].x * i1, o[0].y * i0 - o[1].y * i1, o[0].z * i0 - o[1].z * i1, o[0].w * i0 - o[1].w * i1};
    const float ss = row_sum((y[0] * y[0] + y[1] * y[1]) + (y[2] * y[2] + y[3] * y[3]));
    if (!in) return;
    if (a.norm_w) {
        const float f = rms_factor<HD>(a, ss);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = y[e] * f * nw[e];
    }
    T *out = (T *)a.out + (long long)b * a.bso + (long long)ro.qi * a.ldo + (long long)h * 2 * HD + 4 * lane;
    *(int2 *)out = make_int2(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]));
}

// the MFMA kernels read and write whole 16-byte chunks
bool chunked(const DiffAttnArgs &a) {
    return (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) & 15) == 0 &&
           ((a.ldq | a.ldk | a.ldv | a.ldo) & 7) == 0 && ((a.bsq | a.bsk | a.bsv | a.bso) & 7) == 0;
}

template <typename T, int HD, typename A>
int launch_plan(const DiffAttnArgs &a, DiffPlan &pl, hipStream_t st) {
    TSN_LAUNCH((diff_attn_kernel<T, HD, A>), dim3((unsigned)(pl.full + pl.shared)), dim3(256), 0, st, a, pl);
    TSN_HIP_CHECK(hipGetLastError());
    if (pl.shared > 0) {
        constexpr int PG = A::TR == 16 ? 8 : 1, RPW = 512 / HD / PG;
        const long long rows = std::min<long long>(A::TR, (long long)a.Sq * (a.nh / a.nkv));   // a tile has at most
        pl.groups = (int)((rows + RPW - 1) / RPW);
        TSN_LAUNCH((diff_attn_join_kernel<T, HD, A::TR, A::KB, PG>), dim3((unsigned)(pl.tiles - pl.full) * pl.groups), dim3(256), 0, st, a, pl);
        TSN_HIP_CHECK(hipGetLastError());
    }
    return TSN_OK;
}

template <typename T, int HD>
int launch_any(const DiffAttnArgs &a, hipStream_t st) {
    const unsigned long long n = (unsigned long long)a.B * a.Sq * a.nh;
    TSN_LAUNCH((diff_attn_any_kernel<T, HD>), dim3((unsigned)std::min<unsigned long long>((n + 3) / 4, 1 << 20)), dim3(256), 0, st, a);
    TSN_HIP_CHECK(hipGetLastError());
    return TSN_OK;
}

// the rows of a tile, and what of the tiles is shared out
struct DiffChoice {
    int rows, hd;
    DiffPlan pl;
    size_t pieces() const { return pl.shared ? (size_t)(pl.tiles - pl.full + pl.shared) : 0; }
    size_t bytes() const { return pieces() * rows * (4 * hd + 4) * sizeof(float); }
};

// The plan of the least estimated time (us, fitted to sweeps of 64 to 12289 rows and caches of 128 to 65536 keys; hd 32
// takes 0.55 of hd 64's time a unit). 256 CUs hold two workgroups each.
//  * wide tiles, a workgroup each: a unit takes 1.95 alone on a CU, 3.3 beside another
//  * few-row tiles, a workgroup each: 0.95, 1.35
//  * shared out: the same over 512 workgroups, and a second launch, and the pieces' way to memory and back
// Measured (us), two samples of 8 heads, hd 64, all keys: 397 rows 12 few, 20 wide; 1101 rows 41, 40; 4096 rows 328 few, 207
// wide. One row over 4099 keys, 8 heads: 47 few-row tiles of a workgroup each, 12 shared out; 16 rows of four heads a key
// over 2048 keys, 8 samples: 21, 24; 64 rows over 4096 keys, 4 samples of 8 heads: 37, 28. 64 caches of 8192 keys: 167,
// 181, and with caches of 2048 to 8192 keys, as they are when lengths are given, 129, 121.
DiffChoice choose(const DiffAttnArgs &a) {
    const long long rows = (long long)a.Sq * (a.nh / a.nkv), heads = (long long)a.nkv * a.B;
    const double h = a.hd == 64 ? 1.0 : 0.55;
    const double stream = (double)heads * a.Sk * 8 * a.hd / 5.5e6;   // K and V from memory
    const double seen = a.causal && a.Sq > a.Sk / 2 ? 0.55 : 1.0;    // of the keys, by many rows
    const double ragged = a.kv_len && rows <= 16 ? 0.8 : 1.0;        // a guess: a longer cache makes no one wait when shared
    DiffChoice best{};
    double least = 1e300;
    for (int tr : {128, 16}) {
        DiffChoice c{};
        c.rows = tr;
        c.hd = (int)a.hd;
        DiffPlan &p = c.pl;
        const int kb = tr == 16 ? 128 : 64;
        p.ntile = (int)((rows + tr - 1) / tr);
        p.tiles = (int)(p.ntile * heads);
        p.units = (int)((a.Sk + kb - 1) / kb);
        const double n = p.units, alone = (tr == 16 ? 0.95 : 1.95) * h, pair = (tr == 16 ? 1.35 : 3.3) * h;
        auto keep = [&](double us, int full, int shared) {
            if (us >= least) return;
            DiffChoice d = c;
            d.pl.full = full;
            d.pl.shared = shared;
            d.pl.by_len = full == 0 && (a.q_len || a.kv_len);
            d.pl.ranked = tr == 128 && full == p.tiles && a.causal && (a.q_len || a.kv_len || heads % 8) && a.B <= 64 &&
                          (unsigned long long)a.Sk * (a.nh / a.nkv) < (1ULL << 30);
            if (d.bytes() > ((size_t)256 << 20)) return;
            best = d;
            least = us;
        };
        double us;
        if (tr == 16) {
            const double r = p.tiles / 512.0, rounds = r <= 1 ? 1 : 0.5 * (r + ceil(r));
            us = 3 + std::max(rounds * (n * (p.tiles <= 256 ? alone : pair) * (r > 1 ? seen : 1) + 3), stream);
        } else {
            const int t = (p.tiles + 255) / 256;
            us = 7 + std::max(n * (t / 2 * pair + t % 2 * alone) * (t > 1 ? seen : 1), stream);
        }
        keep(us, p.tiles, 0);
        if ((long long)p.tiles * p.units >= (1LL << 31) || p.tiles >= (1 << 24)) continue;
        for (int wgs : {512, 256}) {   // all tiles, or those behind the last full round, shared out
            for (int full : {0, p.tiles / 512 * 512}) {
                const int rest = p.tiles - full;
                const long long units = (long long)rest * p.units;
                if (rest == 0 || (full == 0 && p.tiles > 512) || (full > 0 && tr == 16)) continue;
                const int shared = (int)std::min<long long>(wgs, units);
                const double part = ceil((double)units / shared) * (wgs == 512 ? pair : alone) * ragged;
                const double pieces = 2.0 * std::min<double>(shared + rest, units) * std::min<double>(tr, rows) * 16.25 * a.hd / 6e6;
                keep(10 + n * (full / 512) * pair + std::max(part, stream * ragged) + pieces + (tr == 16 ? rest / 40.0 : 0.0), full, shared);
            }
        }
    }
    return best;
}

} // namespace

int diff_attention_check(DiffAttnArgs &a) {
    TSN_REQUIRE(a.q && a.k && a.v && a.lam && a.out, "diff_attention: null tensor");
    TSN_REQUIRE(a.dt == DT_F16 || a.dt == DT_BF16, "diff_attention: dtype f16 or bf16");
    TSN_REQUIRE(a.B > 0 && a.Sq > 0 && a.Sk > 0 && a.nh > 0 && a.nkv > 0, "diff_attention: empty shape");
    if (a.hd != 32 && a.hd != 64) {
        set_error("diff_attention: hd must be 32 or 64");
        return TSN_ERR_UNSUPPORTED;
    }
    TSN_REQUIRE(a.nh % a.nkv == 0, "diff_attention: nh must be a multiple of nkv");
    TSN_REQUIRE(a.lam_heads == 1 || a.lam_heads == a.nh, "diff_attention: lambda vectors for one head or for each");
    TSN_REQUIRE(isfinite(a.scale) && a.scale >= 0.0f, "diff_attention: scale must be finite and not negative");
    TSN_REQUIRE(a.lambda_init >= 0.0f && a.lambda_init < 1.0f, "diff_attention: lambda_init must be in [0, 1)");
    TSN_REQUIRE(!a.norm_w || (isfinite(a.eps) && a.eps >= 0.0f), "diff_attention: eps must be finite and not negative");
    // the few-row kernel's tiles, 256 threads each, are less than 2^32 threads
    TSN_REQUIRE(a.nh <= (1u << 12) && a.Sq < (1u << 30) && a.Sk < (1u << 30) && a.B < (1u << 24) &&
                    ((unsigned long long)a.Sq * (a.nh / a.nkv) + 15) / 16 * a.nkv * a.B < (1ULL << 24),
                "diff_attention: sizes beyond the launch grid");
    const uint32_t wq = 2 * a.nh * a.hd, wk = 2 * a.nkv * a.hd;
    if (!a.ldq) a.ldq = wq;
    if (!a.ldk) a.ldk = wk;
    if (!a.ldv) a.ldv = wk;
    if (!a.ldo) a.ldo = wq;
    TSN_REQUIRE(a.ldq >= wq && a.ldk >= wk && a.ldv >= wk && a.ldo >= wq, "diff_attention: row stride below the row width");
    TSN_REQUIRE(a.ldq <= (1u << 22) && a.ldk <= (1u << 22) && a.ldv <= (1u << 22) && a.ldo <= (1u << 22),
                "diff_attention: row stride above 2^22 elements");
    if (!a.bsq) a.bsq = (uint64_t)a.Sq * a.ldq;
    if (!a.bsk) a.bsk = (uint64_t)a.Sk * a.ldk;
    if (!a.bsv) a.bsv = (uint64_t)a.Sk * a.ldv;
    if (!a.bso) a.bso = (uint64_t)a.Sq * a.ldo;
    TSN_REQUIRE(a.bsq < (1ULL << 40) && a.bsk < (1ULL << 40) && a.bsv < (1ULL << 40) && a.bso < (1ULL << 40),
                "diff_attention: sample stride above 2^40 elements");
    TSN_REQUIRE(a.B == 1 || a.bso >= (uint64_t)(a.Sq - 1) * a.ldo + wq || (a.bso >= wq && a.ldo >= (a.B - 1) * a.bso + wq),
                "diff_attention: the samples of out overlap");
    TSN_REQUIRE(((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) % 2 == 0 &&
                    ((uintptr_t)a.lam | (uintptr_t)a.norm_w | (uintptr_t)a.q_len | (uintptr_t)a.kv_len) % 4 == 0,
                "diff_attention: pointers must be aligned to their elements");
    const Window o = window(a.out, 2, wq, a.ldo, a.Sq, a.bso, a.B);
    TSN_REQUIRE(!windows_meet(o, window(a.q, 2, wq, a.ldq, a.Sq, a.bsq, a.B)) &&
                    !windows_meet(o, window(a.k, 2, wk, a.ldk, a.Sk, a.bsk, a.B)) &&
                    !windows_meet(o, window(a.v, 2, wk, a.ldv, a.Sk, a.bsv, a.B)),
                "diff_attention: out overlaps an input");
    const uint64_t nl = 4ULL * a.lam_heads * a.hd;
    struct { const void *p; unsigned long long n; } vec[4] = {
        {a.lam, nl}, {a.norm_w, 2ULL * a.hd}, {a.q_len, a.B}, {a.kv_len, a.B}};
    for (auto &v : vec)
        TSN_REQUIRE(!v.p || !windows_meet(o, window(v.p, 4, v.n, v.n, 1)), "diff_attention: out overlaps lam, norm_w or the lengths");
    return TSN_OK;
}

size_t diff_attention_bytes(const DiffAttnArgs &a) { return chunked(a) ? choose(a).bytes() : 0; }

int launch_diff_attention(const DiffAttnArgs &a, void *ws, size_t ws_bytes, hipStream_t st) {
    auto typed = [&](auto t) -> int {
        using T = decltype(t);
        if (!chunked(a)) return a.hd == 64 ? launch_any<T, 64>(a, st) : launch_any<T, 32>(a, st);
        DiffChoice c = choose(a);
        TSN_REQUIRE(c.bytes() <= ws_bytes && (c.bytes() == 0 || ((uintptr_t)ws & 15) == 0), "diff_attention: workspace");
        c.pl.st = (float4 *)ws;
        c.pl.o = (float *)ws + 4 * c.pieces() * c.rows;
        if (a.hd == 64) return c.rows == 128 ? launch_plan<T, 64, Wide<T, 64>>(a, c.pl, st) : launch_plan<T, 64, Few<T, 64>>(a, c.pl, st);
        return c.rows == 128 ? launch_plan<T, 32, Wide<T, 32>>(a, c.pl, st) : launch_plan<T, 32, Few<T, 32>>(a, c.pl, st);
    };
    return a.dt == DT_F16 ? typed(half_t()) : typed(bf16_t());
}

} // namespace tsn
