// diffattn.hip — differential attention for gfx950: the difference of two softmax maps times one V,
//     lambda = exp(lq1.lk1) - exp(lq2.lk2) + lambda_init
//     o = softmax(s q1 k1^T) v - lambda softmax(s q2 k2^T) v,   out = (1 - lambda_init) RMS(o) w, or o.
// One pass over the keys: each map keeps its running maximum, sum and product with V (the online
// softmax), and the two are joined once both sums are known.
#include <math.h>
#include <stdio.h>
#include <stdlib.h>

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

// Any stride and alignment: one wave a row and head. A block of 64 keys at a time, lane j takes the scores of key j;
// the probabilities go through LDS, then the lanes take the columns of V.
template <typename T, int HD>
__global__ __launch_bounds__(256) void diff_attn_any_kernel(const DiffAttnArgs a) {
    constexpr int NV = 2 * HD / 64;   // columns of V a lane
    __shared__ float sq[4][2 * HD];
    __shared__ float sp[4][2][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long id = (long long)blockIdx.x * 4 + wave;
    const long long n_items = (long long)a.B * a.Sq * a.nh;
    if (id >= n_items) return;   // no barrier below: a wave uses its own LDS
    const int h = (int)(id % a.nh);
    const long long br = id / a.nh;
    const int b = (int)(br / a.Sq), r = (int)(br - (long long)b * a.Sq);
    const int nq = q_rows(a, b), nk = kv_rows(a, b);
    if (r >= nq) return;
    const int g = h / (int)(a.nh / a.nkv);
    int keys = nk;
    if (a.causal) keys = min(nk, max(0, r + nk - nq + 1));
    const T *q = (const T *)a.q + (long long)b * a.bsq + (long long)r * a.ldq + (long long)h * 2 * HD;
    const T *k = (const T *)a.k + (long long)b * a.bsk + (long long)g * 2 * HD;
    const T *v = (const T *)a.v + (long long)b * a.bsv + (long long)g * 2 * HD;
    for (int i = lane; i < 2 * HD; i += 64) sq[wave][i] = (float)q[i] * a.scale * LOG2E;
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
    const float f = a.norm_w ? (1.0f - a.lambda_init) / sqrtf(wave_sum(ss) / (float)(2 * HD) + a.eps) : 1.0f;
    T *out = (T *)a.out + (long long)b * a.bso + (long long)r * a.ldo + (long long)h * 2 * HD;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
        const int i = lane + 64 * c;
        out[i] = (T)(a.norm_w ? y[c] * f * a.norm_w[i] : y[c]);
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
// 16 bytes a lane at voff + soff, global -> LDS slot (lane) of the 1 KB block at address lds. Ordered by explicit vmcnt
// waits; s_nop 0 covers the M0 -> LDS-DMA hazard.
__device__ __forceinline__ void dma16(i32x4 rs, unsigned voff, unsigned soff, unsigned lds) {
    const unsigned l = __builtin_amdgcn_readfirstlane(lds), so = __builtin_amdgcn_readfirstlane(soff);
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
// probability nears f16's range: a lane's 16 add up to no more than 2^12. Only where one exceeds that (the first block:
// m = -1e30) are the maxima taken, the references moved and O and the sums scaled; most blocks take no maximum at all.
template <typename T, int HD>
__device__ __forceinline__ void probs(Rows<HD> &w, const floatx16 (&s)[2], i32x4 (&p)[2][2], float c) {
    float sum[2] = {exp_scores<T>(s[0], c, w.m[0], p[0]), exp_scores<T>(s[1], c, w.m[1], p[1])};
    if (__builtin_amdgcn_ballot_w64(!(fmaxf(sum[0], sum[1]) <= 4096.0f)) != 0) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float t = fmaxf(fmaxf(s[j][0], s[j][1]), s[j][2]);
#pragma unroll
            for (int r = 3; r < 15; r += 2) t = fmaxf(fmaxf(t, s[j][r]), s[j][r + 1]);
            const float mn = fmaxf(w.m[j], pair_max(fmaxf(t, s[j][15])) * c);
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

// How a launch's work is cut. A tile is 32*RW rows of one key/value head of one sample, its keys are units of KB. The
// first `full` tiles have a workgroup each. The units of the others, one after the other, are shared out evenly among
// `shared` workgroups; their pieces of tiles go to the workspace and are joined by diff_attn_join_kernel. A piece's place
// there is its workgroup's number plus its tile's: both only grow along the units, and one of them does at every cut.
struct DiffPlan {
    int ntile;          // tiles of a key/value head
    int tiles, units;   // of all heads and samples; of a tile (by Sk)
    int full, shared;
    int by_len;         // full = 0 and lengths are given: the units are counted by them
    float *o;           // [piece][row of the tile][map][2 HD]: products with V, not divided
    float4 *st;         // [piece][row of the tile]: reference and sum of each map
};
struct Share {   // shared workgroup p's units begin at p*q + min(p, r)
    unsigned q, r;
    __device__ __forceinline__ unsigned begin(unsigned p) const { return p * q + min(p, r); }
    __device__ __forceinline__ unsigned holder(unsigned u) const { return u < r * (q + 1) ? u / (q + 1) : r + (u - r * (q + 1)) / q; }
};
// A unit's tile: sample, place among the sample's tiles (of which each head has `heads`), first unit, units of a tile
struct Spot {
    int b, tile, heads;
    unsigned first, n;
};
// By the lengths: a wave looks at 64 samples at a time. Of sample b, nkv * tiles * n units.
template <int RW, int KB>
struct ByLen {
    __device__ static __forceinline__ void sample(const DiffAttnArgs &a, int b, int &tiles, unsigned &n) {
        const int G = (int)(a.nh / a.nkv);
        tiles = (int)(((unsigned)q_rows(a, b) * G + 32 * RW - 1) / (32 * RW));
        n = (unsigned)max(1, (kv_rows(a, b) + KB - 1) / KB);
    }
    // units up to and with the lane's sample, of the 64 from b0 on
    __device__ static __forceinline__ unsigned scan(const DiffAttnArgs &a, int b0, int lane, unsigned &own) {
        int tiles = 0;
        unsigned n = 0;
        if (b0 + lane < (int)a.B) sample(a, b0 + lane, tiles, n);
        own = a.nkv * tiles * n;
        unsigned v = own;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const unsigned w = __shfl_up(v, d);
            if (lane >= d) v += w;
        }
        return v;
    }
    __device__ static __forceinline__ unsigned total(const DiffAttnArgs &a, int lane) {
        unsigned t = 0, own;
        for (int b0 = 0; b0 < (int)a.B; b0 += 64) t += __builtin_amdgcn_readlane(scan(a, b0, lane, own), 63);
        return t;
    }
    __device__ static __forceinline__ Spot find(const DiffAttnArgs &a, unsigned u, int lane) {
        unsigned before = 0;
        for (int b0 = 0; b0 < (int)a.B; b0 += 64) {
            unsigned own;
            const unsigned upto = scan(a, b0, lane, own), all = __builtin_amdgcn_readlane(upto, 63);
            if (u < before + all) {
                const int i = __ffsll((unsigned long long)__builtin_amdgcn_ballot_w64(before + upto > u)) - 1;
                Spot s;
                s.b = b0 + i;
                const unsigned start = before + __builtin_amdgcn_readlane(upto - own, i);
                sample(a, s.b, s.heads, s.n);
                s.tile = (int)((u - start) / s.n);
                s.first = start + s.tile * s.n;
                return s;
            }
            before += all;
        }
        return Spot{};   // u is below the total: not reached
    }
};

// One tile or piece of one: 32 rows a wave, RW waves side by side; KW waves share the rows of one and take every KW-th
// block of 32 keys, and are merged at the end through LDS. All four read the same K and V tiles, two stages in LDS: the
// next is loaded while one is worked on. RW = 4: two workgroups a CU, one's matrix products cover the other's softmax.
template <typename T, int HD, int RW, int KW>
struct Attn {
    using L = Lay<HD>;
    static constexpr int NSUB = KW > 2 ? KW : 2;     // blocks of 32 keys in a unit
    static constexpr int KB = 32 * NSUB;
    static constexpr int OP = KB * L::ROW, STAGE = 2 * OP, SUB = 32 * L::ROW;
    static constexpr int NB = OP / 1024 / 4;         // 1 KB blocks of K, of V, a wave and unit
    static constexpr int NO = L::DT * 16;            // products of a lane and map
    static constexpr int NQ = NO / KW;               // those that the lane has after the merge
    static constexpr int STATS = KW > 1 ? 4 * 64 * 5 * 4 : 0;
    static constexpr int LDS = 2 * STAGE + STATS;
    static_assert(RW * KW == 4 && (KW == 1 || KW * 2 * NO * 256 <= 2 * STAGE), "four waves, whose products fit in the stages");

    // Every wave leaves its products in LDS and takes values kw*NQ.. of all. Each lane's four are 16 bytes, lanes next to each other.
    static __device__ __forceinline__ void merge(Rows<HD> &w, float (&o)[2][NQ], char *smem, int kw, int lane) {
        float4 *all = (float4 *)smem + lane;
        float4 *st = (float4 *)(smem + 2 * STAGE) + lane;
        block_barrier();   // the key tiles have been read
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < NO; i += 4)
                all[(kw * (NO / 2) + (j * NO + i) / 4) * 64] = make_float4(w.o[j][i >> 4][i & 15], w.o[j][i >> 4][(i & 15) + 1],
                                                                           w.o[j][i >> 4][(i & 15) + 2], w.o[j][i >> 4][(i & 15) + 3]);
        st[kw * 64] = make_float4(w.m[0], w.l[0], w.m[1], w.l[1]);
        block_barrier();
        float f[2][KW];
        w.m[0] = w.m[1] = -1e30f;
        w.l[0] = w.l[1] = 0.0f;
#pragma unroll
        for (int k = 0; k < KW; ++k) {
            const float4 v = st[k * 64];
            w.m[0] = fmaxf(w.m[0], v.x);
            w.m[1] = fmaxf(w.m[1], v.z);
        }
#pragma unroll
        for (int k = 0; k < KW; ++k) {
            const float4 v = st[k * 64];
            f[0][k] = __builtin_amdgcn_exp2f(v.x - w.m[0]);
            f[1][k] = __builtin_amdgcn_exp2f(v.z - w.m[1]);
            w.l[0] += v.y * f[0][k];
            w.l[1] += v.w * f[1][k];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < NQ; i += 4) {
                float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int k = 0; k < KW; ++k) {
                    const float4 v = all[(k * (NO / 2) + (j * NO + kw * NQ + i) / 4) * 64];
                    t.x += v.x * f[j][k];
                    t.y += v.y * f[j][k];
                    t.z += v.z * f[j][k];
                    t.w += v.w * f[j][k];
                }
                o[j][i] = t.x;
                o[j][i + 1] = t.y;
                o[j][i + 2] = t.z;
                o[j][i + 3] = t.w;
            }
    }

    // units u0 to u1 of tile `tile` of head g of sample b; a piece of it (to the workspace) or, piece < 0, all of it
    static __device__ __forceinline__ void run(const DiffAttnArgs &a, const DiffPlan &pl, char *smem, int b, int g, int tile, int u0, int u1,
                                               int piece) {
        const unsigned lds = (unsigned)(unsigned long)(lds_char *)smem;
        const int lane = threadIdx.x & 63;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int rw = wave % RW, kw = wave / RW;
        const int G = (int)(a.nh / a.nkv);
        const int nq = q_rows(a, b), nk = kv_rows(a, b);
        const int x0 = tile * 32 * RW;
        if (x0 / G >= nq) return;   // the whole workgroup: no row of the tile is there
        const int x = x0 + rw * 32 + (lane & 31);
        // keys that any row of the tile and every row of the wave sees
        auto limit = [&](int xr) {
            const int qi = min(row_of(xr, G).qi, nq - 1);
            return a.causal ? min(nk, max(0, qi + nk - nq + 1)) : nk;
        };
        const int keys = limit(x0 + 32 * RW - 1), all = limit(x0 + rw * 32);
        const char *kp = (const char *)((const T *)a.k + (long long)b * a.bsk + g * 2 * HD);
        const char *vp = (const char *)((const T *)a.v + (long long)b * a.bsv + g * 2 * HD);
        const unsigned ldk = a.ldk * 2, ldv = a.ldv * 2;
        const Loads<HD, NB> lo = lane_loads<HD, NB>(wave * NB * L::RPB, ldk, ldv, lane);
        const unsigned kl = lds + k_lane<HD>(lane), vl = lds + OP + v_lane<HD>(lane);
        auto issue = [&](int u) {
            const long long k0 = (long long)u * KB;
            load_tile<HD, NB>(lo, kp + k0 * ldk, vp + k0 * ldv, ldk, ldv, min(KB, nk - u * KB), lds + (u & 1) * STAGE + wave * NB * 1024, OP);
        };
        const float c = a.scale > 0.0f ? a.scale * LOG2E : 1e-30f;   // a scale of 0 must not meet a masked score's infinity
        const int end = min(u1, (keys + KB - 1) / KB);
        block_barrier();   // an earlier piece's LDS has been read
        if (u0 < end) issue(u0);
        Rows<HD> w;
        load_rows<T, HD>(w, a, b, g, G, x, nq, nk, lane);
        const RowOf ro = row_of(x, G);
        // values i of a lane are columns 32(i>>4) + 8((i&15)>>2) + 4*(lane>>5) + (i&3)
        const int i0 = kw * NQ, col0 = 32 * (i0 >> 4) + 2 * (i0 & 15) + 4 * (lane >> 5);
        float lam = 0.0f, nw[KW > 1 ? NQ : 1];
        if (piece < 0) {   // loaded beside the first keys
            lam = row_lambda(a, g, G, ro.hg, lane);
            if constexpr (KW > 1) {
#pragma unroll
                for (int i = 0; i < NQ; ++i) nw[i] = a.norm_w ? a.norm_w[col0 + 32 * (i >> 4) + 8 * ((i & 15) >> 2) + (i & 3)] : 1.0f;
            }
        }
        for (int u = u0; u < end; ++u) {
            wait_vmcnt<0>();
            block_barrier();
            if (u + 1 < end) issue(u + 1);
            const unsigned at = (u & 1) * STAGE;
#pragma unroll 1
            for (int i = 0; i < NSUB / KW; ++i) {
                const int blk = i * KW + kw;
                const int k0 = u * KB + 32 * blk;
                floatx16 s[2];
                i32x4 p[2][2];
                scores<T, HD>(w, kl + at + blk * SUB, s);
                if (k0 + 32 > all) mask_scores<HD>(w, s, k0, lane);
                probs<T, HD>(w, s, p, c);
                product<T, HD>(w, vl + at + blk * SUB, p);
            }
        }
        float o[2][NQ];
        if constexpr (KW > 1) {
            merge(w, o, smem, kw, lane);
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < NQ; ++i) o[j][i] = w.o[j][i >> 4][i & 15];
        }
        const float l0 = pair_sum(w.l[0]), l1 = pair_sum(w.l[1]);
        if (piece >= 0) {
            if (ro.qi >= nq) return;
            const long long row = (long long)piece * (32 * RW) + rw * 32 + (lane & 31);
            if (lane < 32 && kw == 0) pl.st[row] = make_float4(w.m[0], l0, w.m[1], l1);
            float *to = pl.o + row * (4 * HD) + col0;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < NQ; i += 4)
                    *(float4 *)(to + j * 2 * HD + 32 * (i >> 4) + 2 * (i & 15)) = make_float4(o[j][i], o[j][i + 1], o[j][i + 2], o[j][i + 3]);
            return;
        }
        const float r0 = l0 > 0.0f ? 1.0f / l0 : 0.0f, r1 = l1 > 0.0f ? lam / l1 : 0.0f;
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            o[0][i] = o[0][i] * r0 - o[1][i] * r1;
            ss += o[0][i] * o[0][i];
        }
        ss = pair_sum(ss);
        if constexpr (KW > 1) {   // the row's squares over the waves, in their order
            float *red = (float *)(smem + 2 * STAGE + 4 * 64 * 16) + lane;
            red[kw * 64] = ss;
            block_barrier();
            ss = red[0];
#pragma unroll
            for (int k = 1; k < KW; ++k) ss += red[k * 64];
        }
        if (ro.qi >= nq) return;
        if (a.norm_w) {
            const float f = (1.0f - a.lambda_init) / sqrtf(ss / (float)(2 * HD) + a.eps);
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                if constexpr (KW > 1) o[0][i] = o[0][i] * f * nw[i];
                else o[0][i] = o[0][i] * f * a.norm_w[col0 + 32 * (i >> 4) + 8 * ((i & 15) >> 2) + (i & 3)];
            }
        }
        T *out = (T *)a.out + (long long)b * a.bso + (long long)ro.qi * a.ldo + (g * G + ro.hg) * 2 * HD + col0;
#pragma unroll
        for (int i = 0; i < NQ; i += 4)
            *(int2 *)(out + 32 * (i >> 4) + 2 * (i & 15)) = make_int2(pack2<T>(o[0][i], o[0][i + 1]), pack2<T>(o[0][i + 2], o[0][i + 3]));
    }
};

template <int RW, int KB>
__device__ __forceinline__ Share shares(const DiffAttnArgs &a, const DiffPlan &pl, int lane) {
    const unsigned U = pl.by_len ? ByLen<RW, KB>::total(a, lane) : (unsigned)(pl.tiles - pl.full) * pl.units;
    const unsigned q = U / (unsigned)pl.shared;
    return Share{q, U - q * pl.shared};
}
__device__ __forceinline__ int tile_order(const DiffAttnArgs &a, int heads, int i) { return a.causal ? heads - 1 - i : i; }   // the longest first

template <typename T, int HD, int RW, int KW>
__global__ __launch_bounds__(256, 2) void diff_attn_kernel(const DiffAttnArgs a, const DiffPlan pl) {
    using A = Attn<T, HD, RW, KW>;
    __shared__ __attribute__((aligned(1024))) char smem[A::LDS];
    const int lane = threadIdx.x & 63, nkv = (int)a.nkv;
    unsigned u = 0, end = 1;
    int p = (int)blockIdx.x - pl.full;
    if (p >= 0) {
        p = (int)xcd_remap((unsigned)p, pl.shared);
        const Share sh = shares<RW, A::KB>(a, pl, lane);
        u = sh.begin(p);
        end = sh.begin(p + 1);
    }
    while (u < end) {
        int bg, tile, u0 = 0, u1 = pl.units, piece = -1;
        if (p < 0) {
            const int t = (int)xcd_remap(blockIdx.x, pl.full);
            bg = t / pl.ntile;
            tile = tile_order(a, pl.ntile, t - bg * pl.ntile);
            u = end;
        } else {
            unsigned n = pl.units;
            if (pl.by_len) {
                const Spot s = ByLen<RW, A::KB>::find(a, u, lane);
                const int g = s.tile / s.heads;
                bg = s.b * nkv + g;
                tile = tile_order(a, s.heads, s.tile - g * s.heads);
                u0 = (int)(u - s.first);
                n = s.n;
            } else {
                const int ts = (int)(u / n), t = pl.full + ts;
                bg = t / pl.ntile;
                tile = tile_order(a, pl.ntile, t - bg * pl.ntile);
                u0 = (int)(u - ts * n);
            }
            u1 = (int)min(n, u0 + (end - u));
            u += u1 - u0;
            if (u0 > 0 || u1 < (int)n) piece = p + bg * pl.ntile + tile_order(a, pl.ntile, tile) - pl.full;
        }
        const int b = bg / nkv;
        A::run(a, pl, smem, b, bg - b * nkv, tile, u0, u1, piece);
    }
}

// Joins the pieces of the shared tiles: HD/2 lanes a row, four columns of each map a lane, pieces in the order of
// their keys.
template <typename T, int HD, int RW, int KB>
__global__ __launch_bounds__(256) void diff_attn_join_kernel(const DiffAttnArgs a, const DiffPlan pl) {
    constexpr int LR = HD / 2, RPW = 256 / LR, GROUPS = 32 * RW / RPW;   // workgroups of a tile
    const int lane = threadIdx.x & (LR - 1);
    const int ts = (int)(blockIdx.x / GROUPS), r = (int)(blockIdx.x % GROUPS) * RPW + (int)(threadIdx.x / LR);
    const int t = pl.full + ts, bg = t / pl.ntile, nkv = (int)a.nkv;
    const int b = bg / nkv, g = bg - b * nkv, G = (int)(a.nh / a.nkv);
    // the tile's order number among those of its head is turned round once more where the kernel's is
    int tile = tile_order(a, pl.ntile, t - bg * pl.ntile);
    const int nq = q_rows(a, b);
    if ((tile * 32 * RW + (int)(blockIdx.x % GROUPS) * RPW) / G >= nq) return;
    const Share sh = shares<RW, KB>(a, pl, threadIdx.x & 63);
    unsigned first = (unsigned)ts * pl.units, n = pl.units;
    if (pl.by_len) {
        // units before sample b
        unsigned before = 0, own;
        for (int b0 = 0; b0 + 64 <= b; b0 += 64) before += __builtin_amdgcn_readlane(ByLen<RW, KB>::scan(a, b0, threadIdx.x & 63, own), 63);
        const unsigned upto = ByLen<RW, KB>::scan(a, b & ~63, threadIdx.x & 63, own);
        before += __builtin_amdgcn_readlane(upto - own, b & 63);
        int heads;
        ByLen<RW, KB>::sample(a, b, heads, n);
        first = before + (unsigned)(g * heads + tile_order(a, heads, tile)) * n;
    }
    const int p0 = (int)sh.holder(first), p1 = (int)sh.holder(first + n - 1);
    if (p0 == p1) return;   // in one piece: written already
    const RowOf ro = row_of(tile * 32 * RW + r, G);
    const bool in = ro.qi < nq;
    const int h = g * G + (in ? ro.hg : 0);
    const long long row0 = (long long)ts * 32 * RW + r;
    float m[2] = {-1e30f, -1e30f}, l[2] = {0.0f, 0.0f}, o[2][4] = {};
    for (int p = in ? p0 : p1 + 1; p <= p1; ++p) {   // as over the keys: the larger reference, what was before scaled to it
        const long long row = row0 + (long long)p * 32 * RW;
        const float4 st = pl.st[row];
        const float ms[2] = {st.x, st.z}, ls[2] = {st.y, st.w};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float4 v = *(const float4 *)(pl.o + row * (4 * HD) + j * 2 * HD + 4 * lane);
            const float mn = fmaxf(m[j], ms[j]);
            const float f = __builtin_amdgcn_exp2f(m[j] - mn), w = __builtin_amdgcn_exp2f(ms[j] - mn);
            m[j] = mn;
            l[j] = l[j] * f + ls[j] * w;
            o[j][0] = o[j][0] * f + v.x * w;
            o[j][1] = o[j][1] * f + v.y * w;
            o[j][2] = o[j][2] * f + v.z * w;
            o[j][3] = o[j][3] * f + v.w * w;
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
    const float *lv = a.lam + (a.lam_heads > 1 ? (long long)h * 4 * HD : 0) + 2 * lane;
    const float d1 = row_sum(lv[0] * lv[HD] + lv[1] * lv[HD + 1]), d2 = row_sum(lv[2 * HD] * lv[3 * HD] + lv[2 * HD + 1] * lv[3 * HD + 1]);
    const float lam = expf(d1) - expf(d2) + a.lambda_init;
    const float r0 = l[0] > 0.0f ? 1.0f / l[0] : 0.0f, r1 = l[1] > 0.0f ? lam / l[1] : 0.0f;
    float y[4], ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        y[e] = o[0][e] * r0 - o[1][e] * r1;
        ss += y[e] * y[e];
    }
    ss = row_sum(ss);
    if (!in) return;
    if (a.norm_w) {
        const float f = (1.0f - a.lambda_init) / sqrtf(ss / (float)(2 * HD) + a.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = y[e] * f * a.norm_w[4 * lane + e];
    }
    T *out = (T *)a.out + (long long)b * a.bso + (long long)ro.qi * a.ldo + (long long)h * 2 * HD + 4 * lane;
    *(int2 *)out = make_int2(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]));
}

// the MFMA kernels read and write whole 16-byte chunks
bool chunked(const DiffAttnArgs &a) {
    return (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) & 15) == 0 &&
           ((a.ldq | a.ldk | a.ldv | a.ldo) & 7) == 0 && ((a.bsq | a.bsk | a.bsv | a.bso) & 7) == 0;
}

template <typename T, int HD, int RW, int KW>
int launch_plan(const DiffAttnArgs &a, const DiffPlan &pl, hipStream_t st) {
    TSN_LAUNCH((diff_attn_kernel<T, HD, RW, KW>), dim3((unsigned)(pl.full + pl.shared)), dim3(256), 0, st, a, pl);
    TSN_HIP_CHECK(hipGetLastError());
    if (pl.shared > 0) {
        constexpr int GROUPS = 32 * RW * HD / 512;
        TSN_LAUNCH((diff_attn_join_kernel<T, HD, RW, Attn<T, HD, RW, KW>::KB>), dim3((unsigned)(pl.tiles - pl.full) * GROUPS), dim3(256), 0, st, a, pl);
        TSN_HIP_CHECK(hipGetLastError());
    }
    return TSN_OK;
}

template <typename T, int HD>
int launch_any(const DiffAttnArgs &a, hipStream_t st) {
    const unsigned long long n = (unsigned long long)a.B * a.Sq * a.nh;
    TSN_LAUNCH((diff_attn_any_kernel<T, HD>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, a);
    TSN_HIP_CHECK(hipGetLastError());
    return TSN_OK;
}

// rows of a tile / 32, and what of the tiles is shared out
struct DiffChoice {
    int rw;
    DiffPlan pl;
    size_t bytes() const {
        return pl.shared ? (size_t)(pl.tiles - pl.full + pl.shared) * 32 * rw * (4 * hd + 4) * sizeof(float) : 0;
    }
    int hd;
};

DiffChoice choose(const DiffAttnArgs &a) {
    const long long rows = (long long)a.Sq * (a.nh / a.nkv);
    DiffChoice best{};
    double least = 1e30;
    for (int rw : {4, 1}) {
        DiffChoice c{};
        c.rw = rw;
        c.hd = (int)a.hd;
        DiffPlan &p = c.pl;
        const int kb = rw == 1 ? 128 : 64;
        p.ntile = (int)((rows + 32 * rw - 1) / (32 * rw));
        const long long tiles = (long long)p.ntile * a.nkv * a.B;
        if (tiles >= (1LL << 31)) continue;
        p.tiles = (int)tiles;
        p.units = (int)((a.Sk + kb - 1) / kb);
        const char *e = getenv("DA_PLAN");   // rw,full,shared
        int er = 4, ef = -1, es = 0;
        if (e) sscanf(e, "%d,%d,%d", &er, &ef, &es);
        if (er != rw) continue;
        p.full = ef < 0 ? p.tiles : ef < p.tiles ? ef : p.tiles;
        p.shared = p.full < p.tiles ? es : 0;
        if (p.shared > (long long)(p.tiles - p.full) * p.units) p.shared = (p.tiles - p.full) * p.units;
        p.by_len = p.full == 0 && p.shared > 0 && (a.q_len || a.kv_len);
        best = c;
        (void)least;
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
    TSN_REQUIRE(a.nh <= (1u << 12) && a.Sq < (1u << 30) && a.Sk < (1u << 30) &&
                    (unsigned long long)a.B * a.Sq * a.nh < (1ULL << 31),
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
        const size_t pieces = (size_t)(c.pl.tiles - c.pl.full + c.pl.shared) * 32 * c.rw;
        c.pl.st = (float4 *)ws;
        c.pl.o = (float *)ws + 4 * pieces;
        if (a.hd == 64)
            return c.rw == 4 ? launch_plan<T, 64, 4, 1>(a, c.pl, st) : launch_plan<T, 64, 1, 4>(a, c.pl, st);
        return c.rw == 4 ? launch_plan<T, 32, 4, 1>(a, c.pl, st) : launch_plan<T, 32, 1, 4>(a, c.pl, st);
    };
    return a.dt == DT_F16 ? typed(half_t()) : typed(bf16_t());
}

} // namespace tsn
