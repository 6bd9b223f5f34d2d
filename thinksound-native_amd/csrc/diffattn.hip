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

template <typename T> struct Elem;
template <> struct Elem<half_t> { static constexpr int dt = DT_F16; };
template <> struct Elem<bf16_t> { static constexpr int dt = DT_BF16; };

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

template <typename T, int HD>
int launch_typed(const DiffAttnArgs &a, float *ws, size_t ws_bytes, hipStream_t st) {
    (void)ws;
    (void)ws_bytes;
    const unsigned long long n = (unsigned long long)a.B * a.Sq * a.nh;
    TSN_LAUNCH((diff_attn_any_kernel<T, HD>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, a);
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
