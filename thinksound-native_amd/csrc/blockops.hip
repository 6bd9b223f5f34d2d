// blockops.hip — row operators of a transformer block: rotary positions over several axes, and the norms
// after and before a block fused with its gate and residual scale. Both read each element once and
// write it once.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"

#include "dpp.h"
#include "elems.h"

namespace tsn {

namespace {

// Whether a launch's traffic goes past the 256 MB last-level cache whatever it does: then loads and stores that leave
// the caches alone are faster (rotary positions, f16, 269 MB: 47.2 -> 43.6 us, 202 MB: 37.4 -> 33.4), below that a result
// may be there for what reads it next (134 MB: 22.2 -> 23.2).
inline bool passes_caches(size_t bytes) { return bytes >= ((size_t)192 << 20); }

/* ---------------- rotary positions over several axes ---------------- */

// What the kernels read of a call. freq: turns of a pair per position, in 64 bits: a position of 10^6 times a
// frequency of one radian is off by a tenth of a radian in 32 bits. Pairs behind the last axis have frequency 0.
// NP: pairs that fit (heads of up to 64 send a quarter of the frequencies, and half a microsecond less a launch).
constexpr int MAX_PAIRS = 128;
template <int NP>
struct RopeKernelArgs {
    const void *x;
    const int32_t *pos;
    void *y;
    int dt;
    unsigned rows, nh, hd, ldx, ldy, pos_rows, n_axes;
    unsigned start[4], dim[4];   // each axis' elements of a head
    unsigned total;              // elements of all axes
    int half_split;
    double freq[NP];
};

// pair p of a head: its axis and the positions of its two elements
template <int NP>
__device__ __forceinline__ void pair_at(const RopeKernelArgs<NP> &a, unsigned p, unsigned &axis, unsigned &e0, unsigned &e1) {
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

// Any width, stride and alignment (32768 rows of 32 heads of 64, f16: 109 us; whole chunks 44): a thread turns pair p of
// one row in every head, so its sine and cosine are taken once.
__global__ __launch_bounds__(256) void rope_axes_any_kernel(const RopeKernelArgs<MAX_PAIRS> a) {
    const unsigned np = a.hd / 2;
    const long long n = (long long)a.rows * np;
    for (long long id = (long long)blockIdx.x * 256 + threadIdx.x; id < n; id += (long long)gridDim.x * 256) {
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
}

// Whole chunks of VE elements (16 bytes; 8 or two elements where halves of axes do not divide into more): a workgroup takes
// rb rows, computes the cosines and sines of their pairs once (in LDS, for all heads) while its first chunks are under way,
// and turns them. An item is a chunk (neighbouring pairs) or the two
// chunks that hold a pair's halves; behind the axes a chunk is copied. per_head items a head, per_row a row;
// the magic numbers divide by them.
// Bound by memory: 32768 rows of 32 heads of 64, f16, 269 MB: 44.3 us, 6.05 TB/s (a large copy: 6.2); 4999 rows of 24
// heads of 128, bf16, 61 MB: 13.3 us, 4.6 TB/s, with the start of the launch in it; a few rows: 2.6 us, a launch.
struct RopeChunks {
    unsigned rb, per_head, per_row, head_magic, row_magic;
};
template <typename T, bool HALF, bool ONCE, int NP, int VE>
__global__ __launch_bounds__(256) void rope_axes_kernel(const RopeKernelArgs<NP> a, const RopeChunks c) {
    constexpr int UN = 4;   // items in flight a thread
    typedef T vec __attribute__((ext_vector_type(VE)));
    extern __shared__ float2 table[];   // [row of the workgroup][pair]
    const unsigned np = a.hd / 2, r0 = blockIdx.x * c.rb, rows = min(c.rb, a.rows - r0), items = rows * c.per_row;
    const T *x = (const T *)a.x + (long long)r0 * a.ldx;
    T *y = (T *)a.y + (long long)r0 * a.ldy;
    auto load = [](const T *p) { return ONCE ? __builtin_nontemporal_load((const vec *)p) : *(const vec *)p; };
    auto store = [](T *p, vec v) {
        if constexpr (ONCE) __builtin_nontemporal_store(v, (vec *)p);
        else *(vec *)p = v;
    };
    auto place = [&](unsigned i, unsigned &r, unsigned &h, unsigned &p, unsigned &e0, unsigned &e1) {   // item i: row, head, first pair, chunks
        r = __umulhi(i, c.row_magic);
        const unsigned in_row = i - r * c.per_row;
        h = __umulhi(in_row, c.head_magic);
        const unsigned k = (in_row - h * c.per_head) * VE;
        if constexpr (HALF) {
            unsigned axis;
            p = k;
            pair_at(a, p, axis, e0, e1);
            if (2 * p >= a.total) {   // copied
                p = MAX_PAIRS;
                e0 = e1 = k + a.total / 2;
            }
        } else {
            p = k / 2;
            e0 = e1 = k;
        }
    };
    auto fill = [&]() {
        for (unsigned i = threadIdx.x; i < rows * np; i += 256) {
            const unsigned r = i / np, p = i - r * np;
            unsigned axis, e0, e1;
            pair_at(a, p, axis, e0, e1);
            float cs, sn;
            turn(a.freq[p], a.pos[(long long)((r0 + r) % a.pos_rows) * a.n_axes + axis], cs, sn);
            table[i] = make_float2(cs, sn);
        }
        __syncthreads();
    };
    for (unsigned i0 = 0; i0 < items; i0 += 256 * UN) {
        vec v0[UN], v1[HALF ? UN : 1];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const unsigned i = i0 + u * 256 + threadIdx.x;
            if (i >= items) break;
            unsigned r, h, p, e0, e1;
            place(i, r, h, p, e0, e1);
            const T *row = x + (unsigned long long)r * a.ldx + h * a.hd;
            v0[u] = load(row + e0);
            if constexpr (HALF) v1[u] = load(row + e1);
        }
        if (i0 == 0) fill();
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const unsigned i = i0 + u * 256 + threadIdx.x;
            if (i >= items) break;
            unsigned r, h, p, e0, e1;
            place(i, r, h, p, e0, e1);
            T *row = y + (unsigned long long)r * a.ldy + h * a.hd;
            const float2 *t = table + r * np;
            if constexpr (HALF) {
                if (p < MAX_PAIRS) {
                    vec w0, w1;
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        const float2 cs = t[p + e];
                        const float f0 = (float)v0[u][e], f1 = (float)v1[u][e];
                        w0[e] = (T)(f0 * cs.x - f1 * cs.y);
                        w1[e] = (T)(f0 * cs.y + f1 * cs.x);
                    }
                    store(row + e0, w0);
                    store(row + e1, w1);
                } else {
                    store(row + e0, v0[u]);
                }
            } else {
                vec w = v0[u];
#pragma unroll
                for (int e = 0; e < VE; e += 2) {
                    if (e0 + e >= a.total) break;
                    const float2 cs = t[p + e / 2];
                    const float f0 = (float)v0[u][e], f1 = (float)v0[u][e + 1];
                    w[e] = (T)(f0 * cs.x - f1 * cs.y);
                    w[e + 1] = (T)(f0 * cs.y + f1 * cs.x);
                }
                store(row + e0, w);
            }
        }
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

// Rows that the kernel below does not hold in registers (over 8192 elements): a workgroup takes a row at a time, the row (f,
// then x_out) in LDS as f32 (6352 rows of 1024: 38 us; in registers 15.7).
__global__ __launch_bounds__(256) void gate_norm_any_kernel(const GateNormArgs a) {
    extern __shared__ float row[];
    __shared__ float red[4];
    const unsigned H = a.H;
    const int tid = threadIdx.x;
    const float n = (float)H;
    for (unsigned r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const long long xr = (long long)r * a.ldx, fr = (long long)r * a.ldf, orow = (long long)r * a.ldo, yr = (long long)r * a.ldy;
        const float *mod = a.mod ? a.mod + (long long)(r / a.mod_rows) * a.chunks * H : nullptr;
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
        if (!a.y) continue;
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
}

// W waves a row, NC chunks of eight elements a lane, the row in registers between one read and one write. A wave (a group of
// W) takes `per` rows one after the other and keeps what they share:
// y = n(x_out) * A + B with A = pre_w (1 + scale), B = pre_b (1 + scale) + shift, and z's G = f_scale gate post_w, D =
// f_scale gate post_b, made anew where a row of mod begins.
// Bound by memory: 32771 rows of 2048, bf16, each with its row of mod (1.34 GB): 229 us, 5.9 TB/s (a large copy: 6.2); 6352
// rows of 1024 with shared modulation, f32 and f16: 15.7 us, 5.0 TB/s; 8 rows: 3.5 us, a launch and a chain of four sums.
// ANY: rows of any alignment and width: a lane's elements are 64 W apart, loaded and stored one by one, so that a wave's
// access is of neighbours wherever a row begins (16-byte accesses at odd places: 20000 rows of 2501, bf16, each with its
// row of mod, 440 us; a row in LDS 380; so 185).
template <typename TX, typename TF, int W, int NC, bool ONCE, bool ANY>
__global__ __launch_bounds__(W > 1 ? 64 * W : 256, NC == 1 ? 4 : 2) void gate_norm_kernel(const GateNormArgs a, unsigned per) {
    constexpr int GROUPS = W > 1 ? 1 : 4;   // row groups of a workgroup
    __shared__ float red_all[GROUPS][W];
    // uniform where buffers are made (elsewhere it costs 1 to 2%)
    const int wave = ANY ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : threadIdx.x >> 6, lane = threadIdx.x & 63;
    float *red = red_all[wave / W];
    const unsigned H = a.H, chunks = H / 8, first = (wave % W) * 64 + lane;
    // chunk c of the lane: elements 8 k on, k = 64 W c + first, or (ANY) 64 W (8 c + e) + first, e = 0..7
    auto there = [&](int c) { return ANY || c * 64 * W + first < chunks; };
    auto place = [&](int c, int e) { return (8 * c + e) * 64 * W + first; };
    // ANY: a row as a buffer of its own, whose elements from H on read as zeros and are not written
    auto buffer = [&](auto *p) { return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, (int)(H * sizeof(*p)), 0x00020000); };
    auto load8 = [&](auto *p, int c) {
        typedef std::remove_cv_t<std::remove_pointer_t<decltype(p)>> T;
        typedef typename Eight<T>::type V;
        if constexpr (ANY) {
            const auto row = buffer(p);
            V v;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int lane_at = first * sizeof(T), at = (8 * c + e) * 64 * W * sizeof(T);
                if constexpr (sizeof(T) == 4) v[e] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(row, lane_at, at, 0));
                else v[e] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(row, lane_at, at, 0));
            }
            return v;
        } else {
            return *(const V *)(p + 8 * (c * 64 * W + first));
        }
    };
    auto put8 = [&](auto *p, int c, const floatx8 &v) {
        typedef std::remove_pointer_t<decltype(p)> T;
        if constexpr (ANY) {
            const auto row = buffer(p);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int lane_at = first * sizeof(T), at = (8 * c + e) * 64 * W * sizeof(T);
                if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint((float)v[e]), row, lane_at, at, 0);
                else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (T)v[e]), row, lane_at, at, 0);
            }
        } else {
            store8(p + 8 * (c * 64 * W + first), v, std::integral_constant<bool, ONCE>());
        }
    };
    // zeros where there is no element
    auto clear = [&](floatx8 &v, int c) {
        if constexpr (ANY) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (place(c, e) >= H) v[e] = 0.0f;
        } else {
            if (!there(c)) v = floatx8{};
        }
    };
    const unsigned group = blockIdx.x * GROUPS + wave / W;
    const unsigned r0 = group * per, r1 = min(r0 + per, a.rows);
    const float n = (float)H;
    floatx8 A[NC], B[NC], G[NC], D[NC];
    unsigned have = ~0u;
    // sum over the row's waves; every wave of a workgroup takes part the same number of times (W > 1: one group)
    auto row_sum = [&](float v) {
        v = wave_sum(v);
        if constexpr (W > 1) {
            __syncthreads();
            if (lane == 0) red[wave % W] = v;
            __syncthreads();
            v = red[0];
#pragma unroll
            for (int w = 1; w < W; ++w) v += red[w];
        }
        return v;
    };
    auto sum8 = [](const floatx8 &v) { return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])); };
    // centres x for an LN, and its 1 / sqrt(mean square + eps)
    auto norm = [&](floatx8 (&x)[NC], int kind, float eps) {
        if (kind == NORM_NONE) return 1.0f;
        float s = 0.0f;
        if (kind == NORM_LN) {
#pragma unroll
            for (int c = 0; c < NC; ++c) s += sum8(x[c]);
            const float mean = row_sum(s) / n;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                x[c] -= mean;
                clear(x[c], c);
            }
            s = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) s += sum8(x[c] * x[c]);
        return 1.0f / sqrtf(row_sum(s) / n + eps);
    };
    typename Eight<TF>::type rf[NC];
    typename Eight<TX>::type rx[NC];
    auto load = [&](unsigned r) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (there(c)) {
                rf[c] = load8((const TF *)a.f + (unsigned long long)r * a.ldf, c);
                rx[c] = load8((const TX *)a.x + (unsigned long long)r * a.ldx, c);
            } else {
                rf[c] = typename Eight<TF>::type{};
                rx[c] = typename Eight<TX>::type{};
            }
        }
    };
    if (r0 < r1) load(r0);
    for (unsigned r = r0; r < r1; ++r) {
        floatx8 f[NC], x[NC];
        const unsigned m = r / a.mod_rows;
        if (m != have) {
            have = m;
            const float *mod = a.mod ? a.mod + (unsigned long long)m * a.chunks * H : nullptr;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const floatx8 none{};
                auto vec = [&](const float *p, float other) {
                    return !p ? none + other : there(c) ? load8(p, c) : none;
                };
                const floatx8 g = vec(a.gate >= 0 ? mod + (unsigned long long)a.gate * H : nullptr, 1.0f) * a.f_scale;
                const floatx8 s = 1.0f + vec(a.scale >= 0 ? mod + (unsigned long long)a.scale * H : nullptr, 0.0f);
                G[c] = g * vec(a.post_w, 1.0f);
                D[c] = g * vec(a.post_b, 0.0f);
                A[c] = s * vec(a.pre_w, 1.0f);
                B[c] = s * vec(a.pre_b, 0.0f) + vec(a.shift >= 0 ? mod + (unsigned long long)a.shift * H : nullptr, 0.0f);
            }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            f[c] = __builtin_convertvector(rf[c], floatx8);
            x[c] = __builtin_convertvector(rx[c], floatx8) * a.x_scale;
        }
        if (r + 1 < r1) load(r + 1);   // under way while this row is worked on
        const float inv = norm(f, a.post, a.post_eps);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            x[c] += f[c] * inv * G[c] + D[c];
            if (there(c)) put8((TX *)a.x_out + (unsigned long long)r * a.ldo, c, x[c]);
            clear(x[c], c);
        }
        if (!a.y) continue;
        const float pinv = norm(x, a.pre, a.pre_eps);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if (!there(c)) break;
            const floatx8 y = x[c] * pinv * A[c] + B[c];
            const unsigned long long at = (unsigned long long)r * a.ldy;
            if (a.ydt == DT_F32) put8((float *)a.y + at, c, y);
            else if (a.ydt == DT_F16) put8((half_t *)a.y + at, c, y);
            else put8((bf16_t *)a.y + at, c, y);
        }
    }
}

template <typename TX, typename TF, int W, int NC, bool ANY>
int launch_gate_norm_rows(const GateNormArgs &a, hipStream_t st) {
    const GateNormCut cut = gate_norm_cut(a.rows, a.mod_rows, W, NC);
    const dim3 grid(cut.grid), block(cut.block);
    const unsigned per = cut.per;
    const bool once = passes_caches((size_t)a.rows * a.H * (2 * sizeof(TX) + sizeof(TF) + (a.y ? elem_bytes(a.ydt) : 0)));
    if constexpr (ANY) TSN_LAUNCH((gate_norm_kernel<TX, TF, W, NC, false, true>), grid, block, 0, st, a, per);
    else if (once) TSN_LAUNCH((gate_norm_kernel<TX, TF, W, NC, true, false>), grid, block, 0, st, a, per);
    else TSN_LAUNCH((gate_norm_kernel<TX, TF, W, NC, false, false>), grid, block, 0, st, a, per);
    TSN_HIP_CHECK(hipGetLastError());
    return TSN_OK;
}
template <typename TX, typename TF>
int launch_gate_norm_typed(const GateNormArgs &a, bool aligned, hipStream_t st) {
    if (!aligned) {
        if (a.H <= 512) return launch_gate_norm_rows<TX, TF, 1, 1, true>(a, st);
        if (a.H <= 1024) return launch_gate_norm_rows<TX, TF, 2, 1, true>(a, st);
        if (a.H <= 2048) return launch_gate_norm_rows<TX, TF, 4, 1, true>(a, st);
        if (a.H <= 4096) return launch_gate_norm_rows<TX, TF, 8, 1, true>(a, st);
        return launch_gate_norm_rows<TX, TF, 16, 1, true>(a, st);   // to 8192
    }
    if (a.H <= 512) return launch_gate_norm_rows<TX, TF, 1, 1, false>(a, st);
    if (a.H <= 1024) return launch_gate_norm_rows<TX, TF, 2, 1, false>(a, st);
    // two chunks a lane and half the waves: 20000 x 2504 with modulation a row 230 us, 178 as here; 6352 x 1536 23.2, 22.4
    if (a.H <= 2048) return launch_gate_norm_rows<TX, TF, 4, 1, false>(a, st);
    if (a.H <= 4096) return launch_gate_norm_rows<TX, TF, 8, 1, false>(a, st);
    // to 8192. Sixteen waves of one chunk, bf16, beside this (us): 6352 x 5120 with shared modulation 58.8, 56.7, with a row's
    // own 136, 157 (floors 42, 104); 6352 x 8192 88, 88 and 193, 200 (67, 167); f32 and f16 87.8, 89.3 and 160, 171 at 5120.
    return launch_gate_norm_rows<TX, TF, 8, 2, false>(a, st);
}
template <typename TX>
int launch_gate_norm_f(const GateNormArgs &a, bool aligned, hipStream_t st) {
    if (a.fdt == DT_F32) return launch_gate_norm_typed<TX, float>(a, aligned, st);
    return a.fdt == DT_F16 ? launch_gate_norm_typed<TX, half_t>(a, aligned, st) : launch_gate_norm_typed<TX, bf16_t>(a, aligned, st);
}

} // namespace

int rope_axes_check(RopeAxesArgs &a) {
    TSN_REQUIRE(a.x && a.pos && a.y, "rope_axes: null tensor");
    TSN_REQUIRE(is_elem(a.dt), "rope_axes: dtype f32, f16 or bf16");
    TSN_REQUIRE(a.rows > 0 && a.nh > 0 && a.hd > 0, "rope_axes: empty shape");
    TSN_REQUIRE(a.rows < (1u << 31), "rope_axes: 2^31 rows or more");
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
    TSN_REQUIRE(n < (1ULL << 31), "rope_axes: rows of 2^31 elements or more");
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

namespace {

// what the kernels read, but for the frequencies of pairs that NP does not hold
template <int NP>
RopeKernelArgs<NP> rope_kernel_args(const RopeAxesArgs &c) {
    RopeKernelArgs<NP> a{};
    a.x = c.x; a.pos = c.pos; a.y = c.y; a.dt = c.dt;
    a.rows = c.rows; a.nh = c.nh; a.hd = c.hd; a.ldx = c.ldx; a.ldy = c.ldy; a.pos_rows = c.pos_rows; a.n_axes = c.n_axes;
    a.half_split = c.half_split;
    for (unsigned i = 0; i < c.n_axes; ++i) {
        a.start[i] = a.total;
        a.dim[i] = c.dim[i];
        a.total += c.dim[i];
        const unsigned n = c.dim[i] / 2;
        if (n == 0) continue;
        // Pair by pair times base^(-1/n), in 64 bits of mantissa: n roundings are 2^-57 at most. The factor is that of pow
        // with one step of Newton's for factor^n base = 1. (A pow for each pair takes 1.5 us a call more, powl 0.7.)
        const double near = pow((double)c.base[i], -1.0 / n);
        long double q = c.base[i], power = near;
        for (unsigned e = n; e; e >>= 1, power *= power)
            if (e & 1) q *= power;
        const long double ratio = near + near * ((1.0L - q) / n);
        long double f = (c.inverse ? -1.0L : 1.0L) * c.fscale[i] / (2.0L * 3.14159265358979323846264338327950288L);
        for (unsigned p = 0; p < n; ++p, f *= ratio) a.freq[a.start[i] / 2 + p] = (double)f;
    }
    return a;
}

template <typename T, int NP, int VE>
int launch_rope_chunks(const RopeAxesArgs &c, const RopeChunks &k, hipStream_t st) {
    const RopeKernelArgs<NP> a = rope_kernel_args<NP>(c);
    const dim3 grid((c.rows + k.rb - 1) / k.rb);
    const size_t lds = (size_t)k.rb * (c.hd / 2) * sizeof(float2);
    const bool once = passes_caches((size_t)2 * c.rows * c.nh * c.hd * sizeof(T));
    if (c.half_split) {
        if (once) TSN_LAUNCH((rope_axes_kernel<T, true, true, NP, VE>), grid, dim3(256), lds, st, a, k);
        else TSN_LAUNCH((rope_axes_kernel<T, true, false, NP, VE>), grid, dim3(256), lds, st, a, k);
    } else if constexpr (VE * sizeof(T) == 16) {   // neighbours: whole chunks whatever the axes are
        if (once) TSN_LAUNCH((rope_axes_kernel<T, false, true, NP, VE>), grid, dim3(256), lds, st, a, k);
        else TSN_LAUNCH((rope_axes_kernel<T, false, false, NP, VE>), grid, dim3(256), lds, st, a, k);
    }
    TSN_HIP_CHECK(hipGetLastError());
    return TSN_OK;
}
template <typename T, int VE>
int launch_rope_typed(const RopeAxesArgs &c, const RopeChunks &k, hipStream_t st) {
    return c.hd <= 64 ? launch_rope_chunks<T, 32, VE>(c, k, st) : launch_rope_chunks<T, MAX_PAIRS, VE>(c, k, st);
}

} // namespace

int launch_rope_axes(const RopeAxesArgs &c, hipStream_t st) {
    unsigned total = 0, halves = 0;
    for (unsigned i = 0; i < c.n_axes; ++i) {
        total += c.dim[i];
        halves |= c.dim[i] / 2;
    }
    // whole chunks: aligned rows and heads, and for halves whole chunks of each half
    auto whole = [&](unsigned ve) {
        const unsigned at = (unsigned)((uintptr_t)c.x | (uintptr_t)c.y) / (unsigned)elem_bytes(c.dt);
        return ((at | c.ldx | c.ldy | c.hd | (c.half_split ? halves : 0)) & (ve - 1)) == 0;
    };
    unsigned ve = c.dt == DT_F32 ? 4 : 8;
    while (c.half_split && ve > 2 && !whole(ve)) ve /= 2;
    if (whole(ve)) {
        RopeChunks k{};
        k.per_head = c.half_split ? (total / 2 + (c.hd - total)) / ve : c.hd / ve;
        k.per_row = c.nh * k.per_head;
        // rows that give a workgroup's threads four items each, but no more than leave every CU eight workgroups
        const unsigned long long fill = c.rows / 2048 + 1;
        k.rb = (unsigned)std::max<unsigned long long>(1, std::min<unsigned long long>({1024 / k.per_row, fill, 16384 / c.hd}));
        k.rb = std::max(k.rb, c.rows >> 23);   // a launch has less than 2^32 threads
        // i / d = umulhi(i, magic) while i * d < 2^32
        auto magic = [](unsigned d) { return d == 1 ? 0u : (unsigned)((0x100000000ULL + d - 1) / d); };
        k.head_magic = magic(k.per_head);
        k.row_magic = magic(k.per_row);
        const unsigned long long most = (unsigned long long)k.rb * k.per_row;
        if (k.per_head > 1 && most * k.per_row < (1ULL << 32) && k.rb <= 16384 / c.hd) {
            if (c.dt == DT_F32) return ve == 4 ? launch_rope_typed<float, 4>(c, k, st) : launch_rope_typed<float, 2>(c, k, st);
            if (ve == 2) return c.dt == DT_F16 ? launch_rope_typed<half_t, 2>(c, k, st) : launch_rope_typed<bf16_t, 2>(c, k, st);
            if (ve == 4) return c.dt == DT_F16 ? launch_rope_typed<half_t, 4>(c, k, st) : launch_rope_typed<bf16_t, 4>(c, k, st);
            return c.dt == DT_F16 ? launch_rope_typed<half_t, 8>(c, k, st) : launch_rope_typed<bf16_t, 8>(c, k, st);
        }
    }
    const RopeKernelArgs<MAX_PAIRS> a = rope_kernel_args<MAX_PAIRS>(c);
    const unsigned long long n = (unsigned long long)c.rows * (c.hd / 2);
    TSN_LAUNCH(rope_axes_any_kernel, dim3((unsigned)std::min<unsigned long long>((n + 255) / 256, 1 << 20)), dim3(256), 0, st, a);
    TSN_HIP_CHECK(hipGetLastError());
    return TSN_OK;
}

// Rows that share a row of mod in turn, so that the waves fill the device once (16 or 8 a CU): 6352 rows of 1024 take
// 22.2 us a row a wave, 16.6 us four rows a wave, 15.7 us four rows two waves (5.0 TB/s). A row of mod of its own:
// a row a group, and many groups waiting for a place. A launch has less than 2^32 threads.
GateNormCut gate_norm_cut(uint32_t rows, uint32_t mod_rows, unsigned waves, unsigned chunks) {
    const unsigned long long at_once = chunks == 1 ? 4096 : 2048;
    const unsigned groups_of = waves > 1 ? 1 : 4;   // row groups of a workgroup
    GateNormCut c;
    c.block = waves > 1 ? 64 * waves : 256;
    const unsigned most = 0xFFFFFFFFu / c.block * groups_of;   // groups of a launch
    const unsigned long long turns = ((unsigned long long)rows * waves + at_once - 1) / at_once;
    c.per = std::max(mod_rows == 1 ? 1u : (unsigned)std::min(turns, 32ULL), rows / most + (rows % most != 0));
    const unsigned groups = rows / c.per + (rows % c.per != 0);
    c.grid = (groups + groups_of - 1) / groups_of;
    return c;
}

int gate_add_norm_check(GateNormArgs &a) {
    TSN_REQUIRE(a.x && a.f && a.x_out, "gate_add_norm: null tensor");
    TSN_REQUIRE(is_elem(a.xdt) && is_elem(a.fdt) && is_elem(a.ydt), "gate_add_norm: dtypes f32, f16 or bf16");
    TSN_REQUIRE(a.post >= NORM_NONE && a.post <= NORM_LN && a.pre >= NORM_NONE && a.pre <= NORM_LN, "gate_add_norm: norm kind");
    TSN_REQUIRE(a.rows > 0 && a.H > 0, "gate_add_norm: empty shape");
    TSN_REQUIRE(a.rows < (1u << 31), "gate_add_norm: 2^31 rows or more");
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
    const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.f | (uintptr_t)a.x_out | (uintptr_t)a.y | (uintptr_t)a.mod | (uintptr_t)a.post_w |
                         (uintptr_t)a.post_b | (uintptr_t)a.pre_w | (uintptr_t)a.pre_b;
    const bool aligned = a.H % 8 == 0 && ((a.ldx | a.ldf | a.ldo | a.ldy) & 7) == 0 && (at & 31) == 0;
    if (a.H <= 8192) {
        if (a.xdt == DT_F32) return launch_gate_norm_f<float>(a, aligned, st);
        return a.xdt == DT_F16 ? launch_gate_norm_f<half_t>(a, aligned, st) : launch_gate_norm_f<bf16_t>(a, aligned, st);
    }
    TSN_LAUNCH(gate_norm_any_kernel, dim3(std::min(a.rows, 1u << 20)), dim3(256), a.H * sizeof(float), st, a);
    TSN_HIP_CHECK(hipGetLastError());
    return TSN_OK;
}

} // namespace tsn
