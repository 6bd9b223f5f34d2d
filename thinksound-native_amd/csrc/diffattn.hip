// diffattn.hip — differential attention for gfx950: the difference of two softmax maps times one V,
//     lambda = exp(lq1.lk1) - exp(lq2.lk2) + lambda_init
//     o = softmax(s q1 k1^T) v - lambda softmax(s q2 k2^T) v,   out = (1 - lambda_init) RMS(o) w, or o.
// One pass over the keys: each map keeps its running maximum, sum and product with V (the online
// softmax), and the two are joined once both sums are known.
#include <math.h>

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
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ floatx16 mfma32(s16x8 a, s16x8 b, floatx16 c, half_t) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mfma32(s16x8 a, s16x8 b, floatx16 c, bf16_t) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
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

// 16 bytes a lane, global -> LDS slot (lane) of the 1 KB block at lds; offsets past the resource's 2^31 bytes read as
// zero. Ordered by explicit vmcnt waits; s_nop 0 covers the M0 -> LDS-DMA hazard.
__device__ __forceinline__ void dma16(const void *base, unsigned voff, const lds_char *lds) {
    const unsigned l = __builtin_amdgcn_readfirstlane((unsigned)(unsigned long)lds);
    const unsigned long long p = (unsigned long long)base;
    const i32x4 rs = i32x4{(int)__builtin_amdgcn_readfirstlane((unsigned)p),
                           (int)(__builtin_amdgcn_readfirstlane((unsigned)(p >> 32)) & 0xFFFF), 0x7FFFFFFF, 0x00020000};
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                 :
                 : "v"(voff), "s"(rs), "s"(l)
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
    s16x8 q[2][Lay<HD>::KS];
    float m[2], l[2];
    floatx16 o[2][Lay<HD>::DT];
    int lim;   // keys that the lane's row sees
};

// NB blocks of 1 KB of one operand: rows row0 + blk*RPB.. of the tile that starts at `base`, into the tile at lds;
// rows from `valid` on read as zero
template <int HD, bool V>
__device__ __forceinline__ void load_block(const char *base, unsigned ld_bytes, int blk, int valid, const lds_char *tile, int lane) {
    using L = Lay<HD>;
    const int r = blk * L::RPB + lane / L::CPR;
    const int c = (lane % L::CPR) ^ (V ? L::vsw(r) : L::ksw(r));
    dma16(base, r < valid ? (unsigned)r * ld_bytes + c * 16 : 0x80000000u, tile + blk * 1024);
}

// Online softmax and products of 32 keys, key 0 of them at k0, K and V rows at the LDS tiles sK, sV. The reference m
// moves only when a score passes it by more than 2^8 (then O and the sums are rescaled): probabilities stay below 2^8,
// inside f16, and most steps skip it.
template <typename T, int HD>
__device__ __forceinline__ void step32(Rows<HD> &w, const lds_char *sK, const lds_char *sV, int k0, bool mask, float c, int lane) {
    using L = Lay<HD>;
    const int g = lane >> 5;
    const int kr = key_of(lane & 31);
    floatx16 s[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        s[j] = zero16();
#pragma unroll
        for (int ks = 0; ks < L::KS; ++ks) {
            const int slot = (j * (HD / 8) + ks * 2 + g) ^ L::ksw(kr);
            const s16x8 kf = *(const __attribute__((address_space(3))) s16x8 *)(sK + kr * L::ROW + slot * 16);
            s[j] = mfma32(kf, w.q[j][ks], s[j], T());
        }
    }
    if (mask) {   // the same for the whole wave
        const int left = w.lim - k0 - 8 * g;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (16 * (r >> 3) + (r & 7) >= left) s[0][r] = s[1][r] = -INFINITY;
    }
    float top[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float t = fmaxf(fmaxf(s[j][0], s[j][1]), s[j][2]);
#pragma unroll
        for (int r = 3; r < 15; r += 2) t = fmaxf(fmaxf(t, s[j][r]), s[j][r + 1]);
        top[j] = pair_max(fmaxf(t, s[j][15])) * c;
    }
    const bool up0 = top[0] > w.m[0] + 8.0f, up1 = top[1] > w.m[1] + 8.0f;
    if (__builtin_amdgcn_ballot_w64(up0 || up1) != 0) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float mn = (j ? up1 : up0) ? top[j] : w.m[j];
            const float al = __builtin_amdgcn_exp2f(w.m[j] - mn);
            w.m[j] = mn;
            w.l[j] *= al;
#pragma unroll
            for (int d = 0; d < L::DT; ++d) w.o[j][d] *= al;
        }
    }
    s16x8 p[2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r], c, -w.m[j]));
            sum += e;
            p[j][r >> 3][r & 7] = __builtin_bit_cast(short, (T)e);
        }
        w.l[j] += sum;
    }
    // A row = column 32d + (lane & 31) of V, keys 16*h + 8g + 0..7 by two transposing reads of four
    const int vr = 8 * g + ((lane & 15) >> 2);
    const int vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 0; d < L::DT; ++d) {
            s16x4 v[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 16 * h + vr + 4 * e;
                v[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s16x4 *)(sV + r * L::ROW + ((4 * d + vc) ^ L::vsw(r)) * 16 + (lane & 1) * 8));
            }
            const s16x8 vf = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
            w.o[0][d] = mfma32(vf, p[0][h], w.o[0][d], T());
            w.o[1][d] = mfma32(vf, p[1][h], w.o[1][d], T());
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
    const bool in = ro.qi < nq;
    const T *q = (const T *)a.q + (long long)b * a.bsq + (long long)ro.qi * a.ldq + (g * G + ro.hg) * 2 * HD + 8 * (lane >> 5);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int ks = 0; ks < L::KS; ++ks) {
            w.q[j][ks] = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
            if (in) w.q[j][ks] = *(const s16x8 *)(q + j * HD + ks * 16);
        }
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

// Many rows: 128 rows of one key/value head a workgroup, 32 a wave; the four waves share tiles of 64 keys, two stages
// in LDS, the next tile loaded while this one is multiplied.
template <typename T, int HD>
__global__ __launch_bounds__(256, HD == 64 ? 1 : 2) void diff_attn_rows_kernel(const DiffAttnArgs a, int ntile) {
    using L = Lay<HD>;
    constexpr int KB = 64, OP = KB * L::ROW, STAGE = 2 * OP;
    __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];
    const lds_char *lds = (const lds_char *)smem;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned wg = xcd_remap(blockIdx.x, gridDim.x);
    const unsigned bg = wg / (unsigned)ntile;
    const int tile = a.causal ? ntile - 1 - (int)(wg - bg * ntile) : (int)(wg - bg * ntile);   // causal: long rows first
    const int b = (int)(bg / a.nkv), g = (int)(bg - (unsigned)b * a.nkv), G = (int)(a.nh / a.nkv);
    const int nq = q_rows(a, b), nk = kv_rows(a, b);
    const int x0 = tile * 128;
    if (x0 / G >= nq) return;   // the whole workgroup: no row of it is left
    const int x = x0 + wave * 32 + (lane & 31);
    Rows<HD> w;
    load_rows<T, HD>(w, a, b, g, G, x, nq, nk, lane);
    // keys that any row of the workgroup, any row of the wave, and every row of the wave sees
    auto limit = [&](int xr) {
        const int qi = min(row_of(xr, G).qi, nq - 1);
        return a.causal ? min(nk, max(0, qi + nk - nq + 1)) : nk;
    };
    const int keys = limit(x0 + 127), wkeys = limit(x0 + wave * 32 + 31), all = limit(x0 + wave * 32);
    const char *kp = (const char *)((const T *)a.k + (long long)b * a.bsk + g * 2 * HD);
    const char *vp = (const char *)((const T *)a.v + (long long)b * a.bsv + g * 2 * HD);
    const unsigned ldk = a.ldk * 2, ldv = a.ldv * 2;
    auto issue = [&](int t, int stage) {
        const int k0 = t * KB;
        const char *kt = kp + (long long)k0 * ldk, *vt = vp + (long long)k0 * ldv;
        constexpr int PW = OP / 1024 / 4;   // 1 KB blocks of K, of V, a wave
#pragma unroll
        for (int i = 0; i < PW; ++i) load_block<HD, false>(kt, ldk, wave * PW + i, nk - k0, lds + stage * STAGE, lane);
#pragma unroll
        for (int i = 0; i < PW; ++i) load_block<HD, true>(vt, ldv, wave * PW + i, nk - k0, lds + stage * STAGE + OP, lane);
    };
    const float c = a.scale > 0.0f ? a.scale * LOG2E : 1e-30f;   // a scale of 0 must not meet a masked score's infinity
    const int nt = (keys + KB - 1) / KB;
    if (nt > 0) issue(0, 0);
    for (int t = 0; t < nt; ++t) {
        wait_vmcnt<0>();
        block_barrier();
        if (t + 1 < nt) issue(t + 1, (t + 1) & 1);
        const lds_char *sK = lds + (t & 1) * STAGE, *sV = sK + OP;
#pragma unroll 1
        for (int i = 0; i < KB / 32; ++i) {
            const int k0 = t * KB + 32 * i;
            if (k0 >= wkeys) break;
            step32<T, HD>(w, sK + 32 * i * L::ROW, sV + 32 * i * L::ROW, k0, k0 + 32 > all, c, lane);
        }
    }
    const RowOf ro = row_of(x, G);
    const float lam = row_lambda(a, g, G, ro.hg, lane);
    const float l0 = pair_sum(w.l[0]), l1 = pair_sum(w.l[1]);
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
    const float f = a.norm_w ? (1.0f - a.lambda_init) / sqrtf(ss / (float)(2 * HD) + a.eps) : 1.0f;
    T *out = (T *)a.out + (long long)b * a.bso + (long long)ro.qi * a.ldo + (g * G + ro.hg) * 2 * HD;
#pragma unroll
    for (int d = 0; d < L::DT; ++d)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const int col = 32 * d + 8 * q4 + 4 * (lane >> 5);
            s16x4 st;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float y = w.o[0][d][4 * q4 + e];
                st[e] = __builtin_bit_cast(short, (T)(a.norm_w ? y * f * a.norm_w[col + e] : y));
            }
            *(s16x4 *)(out + col) = st;
        }
}

// the MFMA kernels read and write whole 16-byte chunks
bool chunked(const DiffAttnArgs &a) {
    return (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) & 15) == 0 &&
           ((a.ldq | a.ldk | a.ldv | a.ldo) & 7) == 0 && ((a.bsq | a.bsk | a.bsv | a.bso) & 7) == 0;
}

template <typename T, int HD>
int launch_typed(const DiffAttnArgs &a, float *ws, size_t ws_bytes, hipStream_t st) {
    (void)ws;
    (void)ws_bytes;
    if (!chunked(a)) {
        const unsigned long long n = (unsigned long long)a.B * a.Sq * a.nh;
        TSN_LAUNCH((diff_attn_any_kernel<T, HD>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, a);
        TSN_HIP_CHECK(hipGetLastError());
        return TSN_OK;
    }
    const unsigned long long rows = (unsigned long long)a.Sq * (a.nh / a.nkv);
    const int ntile = (int)((rows + 127) / 128);
    TSN_LAUNCH((diff_attn_rows_kernel<T, HD>), dim3((unsigned)(a.B * a.nkv * ntile)), dim3(256), 0, st, a, ntile);
    TSN_HIP_CHECK(hipGetLastError());
    return TSN_OK;
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

int launch_diff_attention(const DiffAttnArgs &a, float *ws, size_t ws_bytes, hipStream_t st) {
    if (a.dt == DT_F16)
        return a.hd == 64 ? launch_typed<half_t, 64>(a, ws, ws_bytes, st) : launch_typed<half_t, 32>(a, ws, ws_bytes, st);
    return a.hd == 64 ? launch_typed<bf16_t, 64>(a, ws, ws_bytes, st) : launch_typed<bf16_t, 32>(a, ws, ws_bytes, st);
}

} // namespace tsn
