// blockops.hip — row operators of a transformer block: rotary positions over several axes, and the norms
// after and before a block fused with its gate and residual scale. Both read each element once and
// write it once.
#include <math.h>

#include "kernels.h"

#include "dpp.h"
#include "elems.h"

namespace tsn {

namespace {

/* ---------------- rotary positions over several axes ---------------- */

// What the kernels read of a call. freq: turns of a pair per position, in 64 bits: a position of 10^6 times a
// frequency of one radian is off by a tenth of a radian in 32 bits. Pairs behind the last axis have frequency 0.
constexpr int MAX_PAIRS = 128;
struct RopeKernelArgs {
    const void *x;
    const int32_t *pos;
    void *y;
    int dt;
    unsigned rows, nh, hd, ldx, ldy, pos_rows, n_axes;
    unsigned start[4], dim[4];   // each axis' elements of a head
    unsigned total;              // elements of all axes
    int half_split;
    double freq[MAX_PAIRS];
};

// pair p of a head: its axis and the positions of its two elements
__device__ __forceinline__ void pair_at(const RopeKernelArgs &a, unsigned p, unsigned &axis, unsigned &e0, unsigned &e1) {
    axis = 0;
    e0 = 2 * p;
    e1 = 2 * p + 1;
    if (e0 >= a.total) return;
#pragma unroll
    for (unsigned i = 1; i < 4; ++i)
        if (i < a.n_axes && e0 >= a.start[i]) axis = i;
    if (a.half_split) {
        e0 = a.start[axis] + (p - a.start[axis] / 2);
        e1 = e0 + a.dim[axis] / 2;
    }
}
// cosine and sine of pair p at a position: whole turns are taken off in 64 bits
__device__ __forceinline__ void turn(double freq, int pos, float &cs, float &sn) {
    const double t = (double)pos * freq;
    sincospif(2.0f * (float)(t - rint(t)), &sn, &cs);
}

// Any width, stride and alignment: a thread turns pair p of one row in every head, so its sine and cosine
// are taken once.
__global__ __launch_bounds__(256) void rope_axes_any_kernel(const RopeKernelArgs a) {
    const unsigned np = a.hd / 2;
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long long)a.rows * np) return;
    const unsigned r = (unsigned)(id / np), p = (unsigned)(id - (long long)r * np);
    unsigned axis, e0, e1;
    pair_at(a, p, axis, e0, e1);
    float cs, sn;
    turn(a.freq[p], a.pos[(long long)(r % a.pos_rows) * a.n_axes + axis], cs, sn);
    const long long xr = (long long)r * a.ldx, yr = (long long)r * a.ldy;
    const bool turned = 2 * p < a.total;
    for (unsigned h = 0; h < a.nh; ++h) {
        const float v0 = load_elem(a.x, a.dt, xr + h * a.hd + e0), v1 = load_elem(a.x, a.dt, xr + h * a.hd + e1);
        store_elem(a.y, a.dt, yr + h * a.hd + e0, turned ? v0 * cs - v1 * sn : v0);
        store_elem(a.y, a.dt, yr + h * a.hd + e1, turned ? v0 * sn + v1 * cs : v1);
    }
}

/* ---------------- norms around a block ---------------- */

// sum over a workgroup of W waves; every thread gets the same value, combined in wave order
template <int W>
__device__ __forceinline__ float group_sum(float v, float *red) {
    v = wave_sum(v);
    if constexpr (W > 1) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();   // the previous sum has been read
        if ((threadIdx.x & 63) == 0) red[wave] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < W; ++w) v += red[w];
    }
    return v;
}

// Any width, stride and alignment: one workgroup a row, the row (f, then x_out) in LDS as f32.
__global__ __launch_bounds__(256) void gate_norm_any_kernel(const GateNormArgs a) {
    extern __shared__ float row[];
    __shared__ float red[4];
    const unsigned r = blockIdx.x, H = a.H;
    const int tid = threadIdx.x;
    const long long xr = (long long)r * a.ldx, fr = (long long)r * a.ldf, orow = (long long)r * a.ldo, yr = (long long)r * a.ldy;
    const float *mod = a.mod ? a.mod + (long long)(r / a.mod_rows) * a.chunks * H : nullptr;
    const float n = (float)H;
    // a thread reads back only elements that it wrote itself
    float s = 0.0f;
    for (unsigned i = tid; i < H; i += 256) {
        const float v = load_elem(a.f, a.fdt, fr + i);
        row[i] = v;
        s += a.post == NORM_LN ? v : v * v;
    }
    float mean = 0.0f, inv = 1.0f;
    if (a.post != NORM_NONE) {
        s = group_sum<4>(s, red);
        if (a.post == NORM_LN) {
            mean = s / n;
            s = 0.0f;
            for (unsigned i = tid; i < H; i += 256) {
                const float d = row[i] - mean;
                s += d * d;
            }
            s = group_sum<4>(s, red);
        }
        inv = 1.0f / sqrtf(s / n + a.post_eps);
    }
    s = 0.0f;
    for (unsigned i = tid; i < H; i += 256) {
        float z = (row[i] - mean) * inv;
        if (a.post_w) z *= a.post_w[i];
        if (a.post_b) z += a.post_b[i];
        const float g = a.f_scale * (a.gate >= 0 ? mod[(long long)a.gate * H + i] : 1.0f);
        const float v = a.x_scale * load_elem(a.x, a.xdt, xr + i) + g * z;
        store_elem(a.x_out, a.xdt, orow + i, v);
        row[i] = v;
        s += a.pre == NORM_LN ? v : v * v;
    }
    if (!a.y) return;
    mean = 0.0f;
    inv = 1.0f;
    if (a.pre != NORM_NONE) {
        s = group_sum<4>(s, red);
        if (a.pre == NORM_LN) {
            mean = s / n;
            s = 0.0f;
            for (unsigned i = tid; i < H; i += 256) {
                const float d = row[i] - mean;
                s += d * d;
            }
            s = group_sum<4>(s, red);
        }
        inv = 1.0f / sqrtf(s / n + a.pre_eps);
    }
    for (unsigned i = tid; i < H; i += 256) {
        float v = (row[i] - mean) * inv;
        if (a.pre_w) v *= a.pre_w[i];
        if (a.pre_b) v += a.pre_b[i];
        if (a.scale >= 0) v *= 1.0f + mod[(long long)a.scale * H + i];
        if (a.shift >= 0) v += mod[(long long)a.shift * H + i];
        store_elem(a.y, a.ydt, yr + i, v);
    }
}

} // namespace

int rope_axes_check(RopeAxesArgs &a) {
    TSN_REQUIRE(a.x && a.pos && a.y, "rope_axes: null tensor");
    TSN_REQUIRE(is_elem(a.dt), "rope_axes: dtype f32, f16 or bf16");
    TSN_REQUIRE(a.rows > 0 && a.nh > 0 && a.hd > 0, "rope_axes: empty shape");
    TSN_REQUIRE(a.hd % 2 == 0 && a.hd <= 2 * MAX_PAIRS, "rope_axes: hd must be even and at most 256");
    TSN_REQUIRE(a.n_axes >= 1 && a.n_axes <= 4, "rope_axes: one to four axes");
    unsigned long long total = 0;
    for (unsigned i = 0; i < a.n_axes; ++i) {
        TSN_REQUIRE(a.dim[i] % 2 == 0, "rope_axes: an axis turns an even number of elements");
        TSN_REQUIRE(isfinite(a.base[i]) && a.base[i] > 0.0f && isfinite(a.fscale[i]), "rope_axes: base must be positive, base and scale finite");
        total += a.dim[i];
    }
    TSN_REQUIRE(total <= a.hd, "rope_axes: the axes turn more than hd elements");
    const unsigned long long n = (unsigned long long)a.nh * a.hd;
    TSN_REQUIRE(n < (1ULL << 31) && (unsigned long long)a.rows * (a.hd / 2) < (1ULL << 31) * 128,
                "rope_axes: sizes beyond the launch grid");
    if (!a.ldx) a.ldx = (uint32_t)n;
    if (!a.ldy) a.ldy = (uint32_t)n;
    TSN_REQUIRE(a.ldx >= n && a.ldy >= n, "rope_axes: row stride below the row width");
    if (!a.pos_rows) a.pos_rows = a.rows;
    const size_t e = elem_bytes(a.dt);
    TSN_REQUIRE((uintptr_t)a.x % e == 0 && (uintptr_t)a.y % e == 0 && (uintptr_t)a.pos % 4 == 0,
                "rope_axes: pointers must be aligned to their elements");
    const Window x = window(a.x, e, n, a.ldx, a.rows), y = window(a.y, e, n, a.ldy, a.rows);
    TSN_REQUIRE((a.x == a.y && a.ldx == a.ldy) || !windows_meet(x, y), "rope_axes: y must be x or not overlap it");
    TSN_REQUIRE(!windows_meet(window(a.pos, 4, a.n_axes, a.n_axes, a.pos_rows), y), "rope_axes: y overlaps pos");
    return TSN_OK;
}

int launch_rope_axes(const RopeAxesArgs &c, hipStream_t st) {
    RopeKernelArgs a{};
    a.x = c.x; a.pos = c.pos; a.y = c.y; a.dt = c.dt;
    a.rows = c.rows; a.nh = c.nh; a.hd = c.hd; a.ldx = c.ldx; a.ldy = c.ldy; a.pos_rows = c.pos_rows; a.n_axes = c.n_axes;
    a.half_split = c.half_split;
    for (unsigned i = 0; i < c.n_axes; ++i) {
        a.start[i] = a.total;
        a.dim[i] = c.dim[i];
        for (unsigned p = 0; p < c.dim[i] / 2; ++p) {
            const double f = (double)c.fscale[i] * pow((double)c.base[i], -2.0 * p / c.dim[i]) / (2.0 * M_PI);
            a.freq[a.total / 2 + p] = c.inverse ? -f : f;
        }
        a.total += c.dim[i];
    }
    const unsigned long long n = (unsigned long long)c.rows * (c.hd / 2);
    TSN_LAUNCH(rope_axes_any_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
    TSN_HIP_CHECK(hipGetLastError());
    return TSN_OK;
}

int gate_add_norm_check(GateNormArgs &a) {
    TSN_REQUIRE(a.x && a.f && a.x_out, "gate_add_norm: null tensor");
    TSN_REQUIRE(is_elem(a.xdt) && is_elem(a.fdt) && is_elem(a.ydt), "gate_add_norm: dtypes f32, f16 or bf16");
    TSN_REQUIRE(a.post >= NORM_NONE && a.post <= NORM_LN && a.pre >= NORM_NONE && a.pre <= NORM_LN, "gate_add_norm: norm kind");
    TSN_REQUIRE(a.rows > 0 && a.H > 0, "gate_add_norm: empty shape");
    TSN_REQUIRE(a.rows < (1u << 31), "gate_add_norm: sizes beyond the launch grid");
    if (a.H > 16384) {
        set_error("gate_add_norm: H above 16384");
        return TSN_ERR_UNSUPPORTED;
    }
    TSN_REQUIRE(isfinite(a.x_scale) && isfinite(a.f_scale), "gate_add_norm: scales must be finite");
    TSN_REQUIRE((a.post == NORM_NONE || (isfinite(a.post_eps) && a.post_eps >= 0.0f)) &&
                    (a.pre == NORM_NONE || (isfinite(a.pre_eps) && a.pre_eps >= 0.0f)),
                "gate_add_norm: eps must be finite and not negative");
    for (int c : {a.gate, a.shift, a.scale}) {
        TSN_REQUIRE(c >= -1 && (c == -1 || (a.mod && (uint32_t)c < a.chunks)), "gate_add_norm: chunk index without its chunk of mod");
    }
    if (!a.ldx) a.ldx = a.H;
    if (!a.ldf) a.ldf = a.H;
    if (!a.ldo) a.ldo = a.H;
    if (!a.ldy) a.ldy = a.H;
    TSN_REQUIRE(a.ldx >= a.H && a.ldf >= a.H && a.ldo >= a.H && a.ldy >= a.H, "gate_add_norm: row stride below H");
    if (!a.mod_rows) a.mod_rows = a.rows;
    const size_t ex = elem_bytes(a.xdt), ef = elem_bytes(a.fdt), ey = elem_bytes(a.ydt);
    TSN_REQUIRE((uintptr_t)a.x % ex == 0 && (uintptr_t)a.f % ef == 0 && (uintptr_t)a.x_out % ex == 0 && (uintptr_t)a.y % ey == 0 &&
                    (uintptr_t)a.mod % 4 == 0 && (uintptr_t)a.post_w % 4 == 0 && (uintptr_t)a.post_b % 4 == 0 &&
                    (uintptr_t)a.pre_w % 4 == 0 && (uintptr_t)a.pre_b % 4 == 0,
                "gate_add_norm: pointers must be aligned to their elements");
    const Window x = window(a.x, ex, a.H, a.ldx, a.rows), f = window(a.f, ef, a.H, a.ldf, a.rows),
                 o = window(a.x_out, ex, a.H, a.ldo, a.rows), y = window(a.y, ey, a.H, a.ldy, a.rows);
    TSN_REQUIRE((a.x_out == a.x && a.ldo == a.ldx) || !windows_meet(o, x), "gate_add_norm: x_out must be x or not overlap it");
    TSN_REQUIRE(!windows_meet(o, f), "gate_add_norm: x_out overlaps f");
    if (a.y) {
        TSN_REQUIRE((a.y == a.f && a.ydt == a.fdt && a.ldy == a.ldf) || !windows_meet(y, f), "gate_add_norm: y must be f or not overlap it");
        TSN_REQUIRE(!windows_meet(y, x) && !windows_meet(y, o), "gate_add_norm: y overlaps x or x_out");
    }
    const unsigned long long mrows = (a.rows + a.mod_rows - 1ULL) / a.mod_rows;
    struct { const float *p; unsigned long long n; } vec[5] = {
        {a.mod, mrows * a.chunks * a.H}, {a.post_w, a.H}, {a.post_b, a.H}, {a.pre_w, a.H}, {a.pre_b, a.H}};
    for (auto &v : vec) {
        if (!v.p || !v.n) continue;
        const Window w = window(v.p, 4, v.n, v.n, 1);
        TSN_REQUIRE(!windows_meet(w, o) && !(a.y && windows_meet(w, y)), "gate_add_norm: an output overlaps mod or a weight");
    }
    return TSN_OK;
}

int launch_gate_add_norm(const GateNormArgs &a, hipStream_t st) {
    TSN_LAUNCH(gate_norm_any_kernel, dim3(a.rows), dim3(256), a.H * sizeof(float), st, a);
    TSN_HIP_CHECK(hipGetLastError());
    return TSN_OK;
}

} // namespace tsn
