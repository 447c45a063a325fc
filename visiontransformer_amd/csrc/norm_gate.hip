// The residual update between two sub-blocks with the norms on both sides of it, one pass forwards and one backwards:
//     p = post(u),   y = a x + s_b g * p,   h = pre(y)
// u the branch's output, post / pre a LayerNorm, an RMS norm or nothing, g a gate per channel or per sample, s_b the
// sample's branch scale (stochastic depth; a sample at 0 keeps y = a x and u is not read), a the residual scale.
// With uh = (u - mu) r the normalised branch the affine part folds into the gate: s g p = s (uh * gw + gb),
// gw = g * w_post, gb = g * b_post, so a row needs gw, gb and the parameters of pre, no more.
//
// Backward, per row:  t = dy + pre'(dh),  dx = a t,  du = post'(s t gw), and four column sums
//     A = sum s t uh,  B = sum s t,  C = sum dh yh,  E = sum dh
// from which every parameter gradient follows: dg = w_post A + b_post B, dw_post = g A, db_post = g B, dw_pre = C,
// db_pre = E.  uh and yh are formed again from x and u in 32 bits (the stored y is rounded), the four row statistics
// are kept by the forward pass.
//
// Bound by HBM (forward x, u -> y, h; backward dy, dh, x, u -> dx, du; 256 x 197 rows of 768 bf16, an eighth of the samples
// without a branch: 65 us forwards, 101 + 6 back, 4.6 TB/s; 4 x 4099 rows of 4096, fp32 stream with bf16 branches: 157 and
// 263 + 9).  A row lives in the registers of one wave up to 1024 elements, of 4 or 8 waves beyond, and is read once;
// parameters and column sums stay in registers while a wave walks its rows.  Column sums are added over the workgroup's rows, written once per workgroup and reduced in a
// fixed order by a second launch: no atomics, results are bitwise reproducible.
#include <algorithm>

#include "common.h"

namespace {

enum { NG_NONE = 0, NG_LAYER = 1, NG_RMS = 2 };

struct NgArgs {
    const void *x, *u;
    long long xs[2], us[2];            // batch and token strides of x and u
    void *y, *h;                       // dense [rows, D]
    const void* gate;
    int gate_f32;                      // gate stored as fp32 (else bf16)
    long long gate_stride;             // elements between samples; 0: one gate per channel
    const float *branch_scale, *post_w, *post_b, *pre_w, *pre_b;
    float* stats;                      // [4][rows]: mu_u, r_u, mu_y, r_y (NULL: not kept)
    // backward
    const void *dy, *dh;               // dense, may be NULL
    void *dx, *du;                     // dense, may be NULL
    float* partial;                    // [blocks][4][D]
    long long rows;
    int N, D, post, pre, chunks;       // chunks: row ranges per sample (gate per sample) or in all (gate per channel)
    float res_scale, eps;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) NVec {
    T v[V];
};

// sum over the 64 lanes of a wave, the same value in every lane: shifts within the rows of 16, two broadcasts between
// rows, all on the vector unit (a shuffle would go through LDS six times)
__device__ __forceinline__ float lanes_sum(float v) {
#define NG_STEP(ctrl, rows) \
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, rows, 0xf, true))
    NG_STEP(0x111, 0xf);   // row_shr 1, 2, 4, 8
    NG_STEP(0x112, 0xf);
    NG_STEP(0x114, 0xf);
    NG_STEP(0x118, 0xf);
    NG_STEP(0x142, 0xa);   // row_bcast 15, 31
    NG_STEP(0x143, 0xc);
#undef NG_STEP
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// pair sums over the WPR waves that share a row; `red` alternates between two halves so that one barrier a call is enough
template <int WPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red, int& flip) {
    a = lanes_sum(a);
    b = lanes_sum(b);
    if (WPR > 1) {
        float* r = red + flip * 2 * WPR;
        flip ^= 1;
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
            r[2 * w] = a;
            r[2 * w + 1] = b;
        }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < WPR; ++i) {
            a += r[2 * i];
            b += r[2 * i + 1];
        }
    }
}

template <int WPR>
__device__ __forceinline__ float row_sum(float a, float* red, int& flip) {
    if (WPR > 1) {
        float z = 0.f;
        row_sum2<WPR>(a, z, red, flip);
        return a;
    }
    return lanes_sum(a);
}

template <int V>
__device__ __forceinline__ void load_f32v(const float* p, float (&o)[V]) {
    const NVec<float, V> t = *reinterpret_cast<const NVec<float, V>*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = t.v[j];
}

// what a thread's columns need of the parameters: gw = gate * post_w, gb = gate * post_b
template <int V, int ITERS, int WPR>
__device__ __forceinline__ void load_gate(const NgArgs& a, int b, float (&gw)[ITERS][V], float (&gb)[ITERS][V]) {
    const int t = WPR > 1 ? (int)threadIdx.x : (int)(threadIdx.x & 63);
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        const int c = (it * 64 * WPR + t) * V;
        float g[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            g[j] = 1.f;
            gb[it][j] = 0.f;
        }
        if (c < a.D) {
            if (a.gate) {
                const long long o = (long long)b * a.gate_stride + c;
                if (a.gate_f32) {
                    load_f32v<V>((const float*)a.gate + o, g);
                } else {
                    const NVec<bf16_t, V> tv = *reinterpret_cast<const NVec<bf16_t, V>*>((const bf16_t*)a.gate + o);
#pragma unroll
                    for (int j = 0; j < V; ++j) g[j] = to_f32(tv.v[j]);
                }
            }
            if (a.post_b) {
                load_f32v<V>(a.post_b + c, gb[it]);
#pragma unroll
                for (int j = 0; j < V; ++j) gb[it][j] *= g[j];
            }
            if (a.post_w) {
                float w[V];
                load_f32v<V>(a.post_w + c, w);
#pragma unroll
                for (int j = 0; j < V; ++j) g[j] *= w[j];
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) gw[it][j] = g[j];
    }
}

template <int V, int ITERS, int WPR>
__device__ __forceinline__ void load_param(const float* p, int D, float fill, float (&o)[ITERS][V]) {
    const int t = WPR > 1 ? (int)threadIdx.x : (int)(threadIdx.x & 63);
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        const int c = (it * 64 * WPR + t) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) o[it][j] = fill;
        if (p && c < D) load_f32v<V>(p + c, o[it]);
    }
}

template <typename T, int V, int ITERS, int WPR>
__device__ __forceinline__ void fetch_row(const T* p, int D, NVec<T, V> (&o)[ITERS]) {
    const int t = WPR > 1 ? (int)threadIdx.x : (int)(threadIdx.x & 63);
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        const int c = (it * 64 * WPR + t) * V;
        if (p && c < D) {
            o[it] = *reinterpret_cast<const NVec<T, V>*>(p + c);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) o[it].v[j] = from_f32<T>(0.f);
        }
    }
}

// mean and 1/sqrt(var + eps) of a row held in registers: deviations are taken from the mean in a second sweep over the
// registers, so a large common offset costs no digits
template <int V, int ITERS, int WPR>
__device__ __forceinline__ void row_stats(const NgArgs& a, const float (&v)[ITERS][V], int kind, float& mu, float& r, float* red,
                                          int& flip) {
    const int t = WPR > 1 ? (int)threadIdx.x : (int)(threadIdx.x & 63);
    mu = 0.f;
    if (kind == NG_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int it = 0; it < ITERS; ++it)
#pragma unroll
            for (int j = 0; j < V; ++j) s += v[it][j];
        mu = row_sum<WPR>(s, red, flip) / (float)a.D;
    }
    float q = 0.f;
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
        if ((it * 64 * WPR + t) * V < a.D) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = v[it][j] - mu;
                q += d * d;
            }
        }
    }
    r = rsqrtf(row_sum<WPR>(q, red, flip) / (float)a.D + a.eps);
}

template <typename TX, typename TU, int V, int ITERS, int WPR>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void ngr_fwd_kernel(NgArgs a) {
    constexpr int RPB = WPR == 1 ? 4 : 1;          // rows a workgroup works on at a time
    __shared__ float red[4 * WPR];
    int flip = 0;
    const int t = WPR > 1 ? (int)threadIdx.x : (int)(threadIdx.x & 63);
    const int wave = WPR == 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : 0;
    float gw[ITERS][V], gb[ITERS][V], pw[ITERS][V], pb[ITERS][V];
    load_param<V, ITERS, WPR>(a.pre_w, a.D, 1.f, pw);
    load_param<V, ITERS, WPR>(a.pre_b, a.D, 0.f, pb);
    int gate_of = -1;
    const long long stride = (long long)gridDim.x * RPB;
    long long row = (long long)blockIdx.x * RPB + wave;
    if (row >= a.rows) return;
    NVec<TX, V> nx[ITERS];
    NVec<TU, V> nu[ITERS];
    float ns = 1.f;
    int nb = 0;
    auto fetch = [&](long long r) {
        const long long b = r / a.N, n = r - b * a.N;
        nb = (int)b;
        ns = a.branch_scale ? a.branch_scale[b] : 1.f;
        fetch_row<TX, V, ITERS, WPR>((const TX*)a.x + b * a.xs[0] + n * a.xs[1], a.D, nx);
        fetch_row<TU, V, ITERS, WPR>(ns != 0.f ? (const TU*)a.u + b * a.us[0] + n * a.us[1] : (const TU*)nullptr, a.D, nu);
    };
    fetch(row);
    for (; row < a.rows; row += stride) {
        float xv[ITERS][V], uv[ITERS][V];
#pragma unroll
        for (int it = 0; it < ITERS; ++it)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                xv[it][j] = to_f32(nx[it].v[j]);
                uv[it][j] = to_f32(nu[it].v[j]);
            }
        const float s = ns;
        const int b = nb;
        if (row + stride < a.rows) fetch(row + stride);
        if (gate_of < 0 || (a.gate_stride && b != gate_of)) {
            load_gate<V, ITERS, WPR>(a, b, gw, gb);
            gate_of = b;
        }
        float mu = 0.f, ru = 1.f, my = 0.f, ry = 1.f;
        if (s == 0.f)
            ru = 0.f;
        else if (a.post != NG_NONE)
            row_stats<V, ITERS, WPR>(a, uv, a.post, mu, ru, red, flip);
        TX* yr = (TX*)a.y + row * (long long)a.D;
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
            const int c = (it * 64 * WPR + t) * V;
            NVec<TX, V> o;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float p = fmaf((uv[it][j] - mu) * ru, gw[it][j], gb[it][j]);
                xv[it][j] = s == 0.f ? a.res_scale * xv[it][j] : fmaf(s, p, a.res_scale * xv[it][j]);
                if (c >= a.D) xv[it][j] = 0.f;
                o.v[j] = from_f32<TX>(xv[it][j]);
            }
            if (c < a.D) *reinterpret_cast<NVec<TX, V>*>(yr + c) = o;
        }
        if (a.pre != NG_NONE) {
            row_stats<V, ITERS, WPR>(a, xv, a.pre, my, ry, red, flip);
            TU* hr = (TU*)a.h + row * (long long)a.D;
#pragma unroll
            for (int it = 0; it < ITERS; ++it) {
                const int c = (it * 64 * WPR + t) * V;
                if (c < a.D) {
                    NVec<TU, V> o;
#pragma unroll
                    for (int j = 0; j < V; ++j) o.v[j] = from_f32<TU>(fmaf((xv[it][j] - my) * ry, pw[it][j], pb[it][j]));
                    *reinterpret_cast<NVec<TU, V>*>(hr + c) = o;
                }
            }
        }
        if (a.stats && t == 0) {
            a.stats[row] = mu;
            a.stats[a.rows + row] = ru;
            a.stats[2 * a.rows + row] = my;
            a.stats[3 * a.rows + row] = ry;
        }
    }
}

// one workgroup: rows [r0, r1) of one range; with a gate per sample a range lies within one sample
template <typename TX, typename TU, int V, int ITERS, int WPR>
__global__ __launch_bounds__(WPR == 1 ? 256 : 64 * WPR) void ngr_bwd_kernel(NgArgs a) {
    constexpr int RPB = WPR == 1 ? 4 : 1;
    __shared__ float red[4 * WPR];
    __shared__ float cols[WPR == 1 ? 3 * 64 * V : 1];
    int flip = 0;
    const int t = WPR > 1 ? (int)threadIdx.x : (int)(threadIdx.x & 63);
    const int wave = WPR == 1 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : 0;
    float gw[ITERS][V], gb[ITERS][V], pw[ITERS][V];
    float sA[ITERS][V], sB[ITERS][V], sC[ITERS][V], sE[ITERS][V];
    load_param<V, ITERS, WPR>(a.pre_w, a.D, 1.f, pw);
#pragma unroll
    for (int it = 0; it < ITERS; ++it)
#pragma unroll
        for (int j = 0; j < V; ++j) sA[it][j] = sB[it][j] = sC[it][j] = sE[it][j] = 0.f;
    const long long per = a.gate_stride ? a.N : a.rows;
    const int seg = blockIdx.x / a.chunks, chunk = blockIdx.x - seg * a.chunks;
    const long long r0 = seg * per + chunk * per / a.chunks, r1 = seg * per + (chunk + 1) * per / a.chunks;
    load_gate<V, ITERS, WPR>(a, seg, gw, gb);
    const float inv_d = 1.f / (float)a.D;
    const bool pre = a.pre != NG_NONE && a.dh;
    // the next row's loads are in flight behind a row's arithmetic where their registers (dy, x, dh, u as stored) leave room
    constexpr bool AHEAD = ITERS * V * (sizeof(TX) + sizeof(TU)) / 2 <= 48;
    NVec<TX, V> nx[ITERS], ndy[ITERS];
    NVec<TU, V> nu[ITERS], ndh[ITERS];
    float ns = 1.f, nmu = 0.f, nru = 0.f, nmy = 0.f, nry = 0.f;
    auto fetch = [&](long long row) {
        const long long b = row / a.N, n = row - b * a.N;
        ns = a.branch_scale ? a.branch_scale[b] : 1.f;
        fetch_row<TX, V, ITERS, WPR>(a.dy ? (const TX*)a.dy + row * a.D : (const TX*)nullptr, a.D, ndy);
        fetch_row<TU, V, ITERS, WPR>(pre ? (const TU*)a.dh + row * a.D : (const TU*)nullptr, a.D, ndh);
        fetch_row<TX, V, ITERS, WPR>(pre ? (const TX*)a.x + b * a.xs[0] + n * a.xs[1] : (const TX*)nullptr, a.D, nx);
        nmu = a.stats[row];
        nru = a.stats[a.rows + row];
        nmy = a.stats[2 * a.rows + row];
        nry = a.stats[3 * a.rows + row];
        fetch_row<TU, V, ITERS, WPR>(ns != 0.f ? (const TU*)a.u + b * a.us[0] + n * a.us[1] : (const TU*)nullptr, a.D, nu);
    };
    if (AHEAD && r0 + wave < r1) fetch(r0 + wave);
    for (long long row = r0 + wave; row < r1; row += RPB) {
        if (!AHEAD) fetch(row);
        const float s = ns, mu = nmu, ru = nru, my = nmy, ry = nry;
        const bool live = s != 0.f;
        float tv[ITERS][V], uh[ITERS][V], yh[ITERS][V];
        NVec<TU, V> dhv[ITERS];
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
            const bool in = (it * 64 * WPR + t) * V < a.D;
            dhv[it] = ndh[it];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                tv[it][j] = to_f32(ndy[it].v[j]);
                uh[it][j] = (to_f32(nu[it].v[j]) - mu) * ru;
                const float ax = a.res_scale * to_f32(nx[it].v[j]);
                const float yv = live ? fmaf(s, fmaf(uh[it][j], gw[it][j], gb[it][j]), ax) : ax;
                yh[it][j] = in ? (yv - my) * ry : 0.f;
            }
        }
        if (AHEAD && row + RPB < r1) fetch(row + RPB);
        if (pre) {
            float c1 = 0.f, c2 = 0.f;
#pragma unroll
            for (int it = 0; it < ITERS; ++it)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float dh = to_f32(dhv[it].v[j]);
                    sC[it][j] = fmaf(dh, yh[it][j], sC[it][j]);
                    sE[it][j] += dh;
                    const float g = dh * pw[it][j];
                    c1 += g;
                    c2 = fmaf(g, yh[it][j], c2);
                }
            row_sum2<WPR>(c1, c2, red, flip);
            c1 = a.pre == NG_LAYER ? c1 * inv_d : 0.f;
            c2 *= inv_d;
#pragma unroll
            for (int it = 0; it < ITERS; ++it)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    tv[it][j] = fmaf(ry, fmaf(to_f32(dhv[it].v[j]), pw[it][j], -c1) - yh[it][j] * c2, tv[it][j]);
        }
        if (a.dx) {
            TX* dr = (TX*)a.dx + row * a.D;
#pragma unroll
            for (int it = 0; it < ITERS; ++it) {
                const int c = (it * 64 * WPR + t) * V;
                if (c < a.D) {
                    NVec<TX, V> o;
#pragma unroll
                    for (int j = 0; j < V; ++j) o.v[j] = from_f32<TX>(a.res_scale * tv[it][j]);
                    *reinterpret_cast<NVec<TX, V>*>(dr + c) = o;
                }
            }
        }
        float d1 = 0.f, d2 = 0.f;
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
            const bool in = (it * 64 * WPR + t) * V < a.D;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float st = live && in ? s * tv[it][j] : 0.f;
                sA[it][j] = fmaf(st, uh[it][j], sA[it][j]);
                sB[it][j] += st;
                tv[it][j] = st * gw[it][j];
                d1 += tv[it][j];
                d2 = fmaf(tv[it][j], uh[it][j], d2);
            }
        }
        if (a.du) {
            if (a.post != NG_NONE) {
                row_sum2<WPR>(d1, d2, red, flip);
                d1 = a.post == NG_LAYER ? d1 * inv_d : 0.f;
                d2 *= inv_d;
#pragma unroll
                for (int it = 0; it < ITERS; ++it)
#pragma unroll
                    for (int j = 0; j < V; ++j) tv[it][j] = ru * ((tv[it][j] - d1) - uh[it][j] * d2);
            }
            TU* dr = (TU*)a.du + row * a.D;
#pragma unroll
            for (int it = 0; it < ITERS; ++it) {
                const int c = (it * 64 * WPR + t) * V;
                if (c < a.D) {
                    NVec<TU, V> o;
#pragma unroll
                    for (int j = 0; j < V; ++j) o.v[j] = from_f32<TU>(tv[it][j]);
                    *reinterpret_cast<NVec<TU, V>*>(dr + c) = o;
                }
            }
        }
    }
    if (!a.partial) return;
    float* out = a.partial + (long long)blockIdx.x * 4 * a.D;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
            const int c = (it * 64 * WPR + t) * V;
            float v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = q == 0 ? sA[it][j] : q == 1 ? sB[it][j] : q == 2 ? sC[it][j] : sE[it][j];
            if (WPR == 1) {                        // the four waves' sums meet in LDS, in wave order
                __syncthreads();
                if (wave > 0)
#pragma unroll
                    for (int j = 0; j < V; ++j) cols[((wave - 1) * V + j) * 64 + t] = v[j];
                __syncthreads();
                if (wave == 0)
#pragma unroll
                    for (int j = 0; j < V; ++j)
#pragma unroll
                        for (int w = 0; w < 3; ++w) v[j] += cols[(w * V + j) * 64 + t];
            }
            if (wave == 0 && c < a.D) {
                NVec<float, V> o;
#pragma unroll
                for (int j = 0; j < V; ++j) o.v[j] = v[j];
                *reinterpret_cast<NVec<float, V>*>(out + (long long)q * a.D + c) = o;
            }
        }
    }
}

struct NgFinal {
    const float* partial;          // [segs][chunks][4][D]
    const void* gate;
    int gate_f32;
    long long gate_stride;
    const float *post_w, *post_b;
    void* dgate;                   // [segs][D], of the gate's type
    float *dpost_w, *dpost_b, *dpre_w, *dpre_b;
    int segs, chunks, D;
};

__device__ __forceinline__ float gate_at(const NgFinal& f, int seg, int c) {
    if (!f.gate) return 1.f;
    const long long o = (long long)seg * f.gate_stride + c;
    return f.gate_f32 ? ((const float*)f.gate)[o] : to_f32(((const bf16_t*)f.gate)[o]);
}

// NF_COLS columns x NF_GROUPS row groups a workgroup; blockIdx.y = 0 reduces the pair (A, B), 1 the pair (C, E).  Partials
// are added in a fixed order.  Few columns a workgroup, because a row of 768 would otherwise occupy 12 of them.
constexpr int NF_COLS = 16, NF_GROUPS = 64;

__device__ __forceinline__ void final_pair(float& p, float& q, float (*red)[2][NF_COLS], int col, int grp) {
    for (int n = NF_GROUPS; n > 1; n >>= 3) {            // eight into one, twice
        if (grp < n) {
            red[grp][0][col] = p;
            red[grp][1][col] = q;
        }
        __syncthreads();
        p = q = 0.f;
        if (grp < n / 8)
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                p += red[grp * 8 + g][0][col];
                q += red[grp * 8 + g][1][col];
            }
        __syncthreads();
    }
}

__global__ __launch_bounds__(NF_COLS* NF_GROUPS) void ngr_final_kernel(NgFinal f) {
    const int col = threadIdx.x % NF_COLS, grp = threadIdx.x / NF_COLS;
    const int c = blockIdx.x * NF_COLS + col;
    const bool in = c < f.D, branch = blockIdx.y == 0;
    __shared__ float red[NF_GROUPS][2][NF_COLS];
    const float* part = f.partial + (branch ? 0 : 2ll * f.D) + c;
    auto add = [&](long long k, float& p, float& q) {
        p += part[k * 4 * f.D];
        q += part[k * 4 * f.D + f.D];
    };
    auto gate_grad = [&](int seg, float p, float q) {
        if (!f.dgate) return;
        const float d = (f.post_w ? f.post_w[c] : 1.f) * p + (f.post_b ? f.post_b[c] * q : 0.f);
        const long long o = (long long)seg * f.D + c;
        if (f.gate_f32) ((float*)f.dgate)[o] = d;
        else ((bf16_t*)f.dgate)[o] = (bf16_t)d;
    };
    float tp = 0.f, tq = 0.f;
    if (!branch || f.chunks >= NF_GROUPS) {
        // a sum over everything, or one segment after the other with the groups on its chunks
        const int segs = branch ? f.segs : 1;
        const long long n = branch ? f.chunks : (long long)f.segs * f.chunks;
        for (int seg = 0; seg < segs; ++seg) {
            float p = 0.f, q = 0.f;
            if (in)
                for (long long k = grp; k < n; k += NF_GROUPS) add(seg * n + k, p, q);
            final_pair(p, q, red, col, grp);
            if (grp == 0 && in) {
                if (branch) {
                    gate_grad(seg, p, q);
                    const float g = gate_at(f, seg, c);
                    p *= g;
                    q *= g;
                }
                tp += p;
                tq += q;
            }
        }
    } else {
        // many segments of few chunks: a group takes whole segments
        if (in)
            for (int seg = grp; seg < f.segs; seg += NF_GROUPS) {
                float p = 0.f, q = 0.f;
                for (int k = 0; k < f.chunks; ++k) add((long long)seg * f.chunks + k, p, q);
                gate_grad(seg, p, q);
                const float g = gate_at(f, seg, c);
                tp = fmaf(g, p, tp);
                tq = fmaf(g, q, tq);
            }
        final_pair(tp, tq, red, col, grp);
    }
    if (grp == 0 && in) {
        float *o0 = branch ? f.dpost_w : f.dpre_w, *o1 = branch ? f.dpost_b : f.dpre_b;
        if (o0) o0[c] = tp;
        if (o1) o1[c] = tq;
    }
}

struct NgPlan {
    int V, iters, wpr;
};

// A row goes to one wave while sixteen values a lane hold it, to four or eight while eight do, then to eight: 4096 columns by
// four waves of sixteen values took 189 us forwards and 303 back (4 x 4099 rows, fp32 stream), by eight of eight 151 and 256
bool ng_plan(int D, bool vec, NgPlan* p) {
    p->V = vec ? 4 : 1;
    const int values[4][2] = {{1, 16}, {4, 8}, {8, 8}, {8, 16}};      // waves, values per lane
    for (auto& v : values) {
        const int w = v[0], iters = ceil_div(D, 64 * w * p->V);
        if (iters * p->V <= v[1]) {
            p->wpr = w;
            p->iters = iters;
            return true;
        }
    }
    return false;
}

// partial-sum rows of the backward pass: two workgroups of four waves a compute unit (one of eight), spread over the samples
// where the gate is per sample
int ng_chunks(bool per_sample, int B, int N, int wpr) {
    const long long rows = (long long)B * N;
    const int rpb = wpr == 1 ? 4 : 1;
    const int target = wpr <= 4 ? 512 : 256;
    if (!per_sample) return (int)std::max<long long>(1, std::min<long long>(target, (rows + rpb - 1) / rpb));
    return std::max(1, std::min(target / std::max(1, B), ceil_div(N, rpb)));
}

template <typename TX, typename TU, int V, int ITERS, int WPR>
void ng_launch(const NgArgs& a, bool fwd, unsigned blocks, hipStream_t s) {
    constexpr int THREADS = WPR == 1 ? 256 : 64 * WPR;
    if (fwd)
        hipLaunchKernelGGL((ngr_fwd_kernel<TX, TU, V, ITERS, WPR>), dim3(blocks), dim3(THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((ngr_bwd_kernel<TX, TU, V, ITERS, WPR>), dim3(blocks), dim3(THREADS), 0, s, a);
}

template <typename TX, typename TU>
void ng_dispatch(const NgArgs& a, const NgPlan& p, bool fwd, unsigned blocks, hipStream_t s) {
    // the pairs of waves and vectors per lane that ng_plan gives: (1, 1..4), (4, 2), (8, 2..4) of four values, and single values
    // in sizes of 4, 8 and 16
#define NG(V, I, W) ng_launch<TX, TU, V, I, W>(a, fwd, blocks, s)
    if (p.V == 4) {
        if (p.wpr == 1) {
            if (p.iters <= 1) NG(4, 1, 1);
            else if (p.iters == 2) NG(4, 2, 1);
            else if (p.iters == 3) NG(4, 3, 1);
            else NG(4, 4, 1);
        } else if (p.wpr == 4) {
            NG(4, 2, 4);
        } else {
            if (p.iters <= 2) NG(4, 2, 8);
            else if (p.iters == 3) NG(4, 3, 8);
            else NG(4, 4, 8);
        }
    } else if (p.wpr == 1) {
        if (p.iters <= 4) NG(1, 4, 1);
        else NG(1, 16, 1);
    } else if (p.wpr == 4) {
        NG(1, 8, 4);
    } else {
        if (p.iters <= 8) NG(1, 8, 8);
        else NG(1, 16, 8);
    }
#undef NG
}

bool ng_types_ok(int dx, int du) {
    return (dx == VITMI_F32 && (du == VITMI_F32 || du == VITMI_BF16)) || (dx == VITMI_BF16 && du == VITMI_BF16);
}

int ng_check(const char* who, const vitmi_ngr_args* g) {
    VITMI_CHECK_ARG(g, "%s: null arguments", who);
    VITMI_CHECK_ARG(ng_types_ok(g->dt_x, g->dt_u), "%s: residual type %d with branch type %d (fp32 or bf16, the residual at least as wide)",
                    who, g->dt_x, g->dt_u);
    VITMI_CHECK_ARG(g->B >= 0 && g->N >= 0 && g->D > 0, "%s: bad shape B=%d N=%d D=%d", who, g->B, g->N, g->D);
    VITMI_CHECK_ARG(g->post >= 0 && g->post <= 2 && g->pre >= 0 && g->pre <= 2, "%s: bad norm kind %d / %d", who, g->post, g->pre);
    VITMI_CHECK_ARG(!g->gate || g->gate_dt == VITMI_F32 || g->gate_dt == VITMI_BF16, "%s: bad gate type %d", who, g->gate_dt);
    VITMI_CHECK_ARG(g->eps >= 0.f, "%s: eps must not be negative", who);
    if (g->D > 8192) {
        vitmi_set_error("%s: D=%d exceeds the supported row length 8192", who, g->D);
        return VITMI_ERR_UNSUPPORTED;
    }
    return VITMI_OK;
}

bool ng_vec(const vitmi_ngr_args* g) {
    if (g->D % 4) return false;
    const uintptr_t ex = g->dt_x == VITMI_F32 ? 16 : 8, eu = g->dt_u == VITMI_F32 ? 16 : 8, eg = g->gate_dt == VITMI_F32 ? 16 : 8;
    auto al = [](const void* p, uintptr_t m) { return (reinterpret_cast<uintptr_t>(p) & (m - 1)) == 0; };
    for (int i = 0; i < 2; ++i)
        if (g->xs[i] % 4 || g->us[i] % 4) return false;
    if (g->gate && (g->gate_stride % 4 || !al(g->gate, eg))) return false;
    return al(g->x, ex) && al(g->u, eu) && al(g->y, ex) && al(g->h, eu) && al(g->post_w, 16) && al(g->post_b, 16) &&
           al(g->pre_w, 16) && al(g->pre_b, 16) && al(g->dy, ex) && al(g->dh, eu) && al(g->dx, ex) && al(g->du, eu);
}

void ng_fill(const vitmi_ngr_args* g, NgArgs* a) {
    *a = NgArgs{};
    a->x = g->x; a->u = g->u; a->y = g->y; a->h = g->h;
    for (int i = 0; i < 2; ++i) {
        a->xs[i] = g->xs[i];
        a->us[i] = g->us[i];
    }
    a->gate = g->gate;
    a->gate_f32 = g->gate_dt == VITMI_F32;
    a->gate_stride = g->gate ? g->gate_stride : 0;
    a->branch_scale = g->branch_scale;
    a->post_w = g->post == NG_NONE ? nullptr : g->post_w;
    a->post_b = g->post == NG_NONE ? nullptr : g->post_b;
    a->pre_w = g->pre == NG_NONE ? nullptr : g->pre_w;
    a->pre_b = g->pre == NG_NONE ? nullptr : g->pre_b;
    a->stats = g->stats;
    a->dy = g->dy; a->dh = g->dh; a->dx = g->dx; a->du = g->du;
    a->rows = (long long)g->B * g->N;
    a->N = g->N; a->D = g->D; a->post = g->post; a->pre = g->pre;
    a->res_scale = g->res_scale;
    a->eps = g->eps;
}

}  // namespace

extern "C" int vitmi_norm_gate_residual_fwd(const vitmi_ngr_args* g, void* stream) {
    const char* who = "vitmi_norm_gate_residual_fwd";
    if (int rc = ng_check(who, g)) return rc;
    if (g->B == 0 || g->N == 0) return VITMI_OK;
    VITMI_CHECK_ARG(g->x && g->u && g->y && (g->pre == NG_NONE || g->h), "%s: null pointer", who);
    NgPlan p;
    if (!ng_plan(g->D, ng_vec(g), &p)) {
        vitmi_set_error("%s: no plan for D=%d", who, g->D);
        return VITMI_ERR_UNSUPPORTED;
    }
    NgArgs a;
    ng_fill(g, &a);
    hipStream_t s = as_stream(stream);
    const int ex = g->dt_x == VITMI_F32 ? 4 : 2, eu = g->dt_u == VITMI_F32 ? 4 : 2;
    ProfScope prof(VITMI_FAM_LAYERNORM, s, (double)a.rows * g->D * (2 * ex + eu * (g->pre ? 2 : 1)));
    const int rpb = p.wpr == 1 ? 4 : 1;
    // sixteen waves a compute unit walk the rows, each with its next row's loads outstanding
    const long long cap = p.wpr == 8 ? 512 : 1024;
    const unsigned blocks = (unsigned)std::min<long long>((a.rows + rpb - 1) / rpb, cap);
    if (g->dt_x == VITMI_BF16) ng_dispatch<bf16_t, bf16_t>(a, p, true, blocks, s);
    else if (g->dt_u == VITMI_BF16) ng_dispatch<float, bf16_t>(a, p, true, blocks, s);
    else ng_dispatch<float, float>(a, p, true, blocks, s);
    VITMI_LAUNCH_CHECK(who);
    return VITMI_OK;
}

extern "C" long long vitmi_norm_gate_residual_bwd_workspace_bytes(int B, int N, int D, int gate_per_sample) {
    if (B <= 0 || N <= 0 || D <= 0) return 0;
    // the plan depends on alignment: room for the most row ranges any plan makes
    const long long a = ng_chunks(gate_per_sample != 0, B, N, 1), b = ng_chunks(gate_per_sample != 0, B, N, 4);
    return std::max(a, b) * (gate_per_sample ? B : 1) * 4ll * D * (long long)sizeof(float);
}

extern "C" int vitmi_norm_gate_residual_bwd(const vitmi_ngr_args* g, void* workspace, void* stream) {
    const char* who = "vitmi_norm_gate_residual_bwd";
    if (int rc = ng_check(who, g)) return rc;
    const bool per_sample = g->gate && g->gate_stride != 0;
    const bool sums = g->dgate || g->dpost_w || g->dpost_b || g->dpre_w || g->dpre_b;
    VITMI_CHECK_ARG(g->B > 0 && g->N > 0, "%s: no rows", who);
    VITMI_CHECK_ARG(g->x && g->u && g->stats && (g->dy || g->dh) && (workspace || !sums), "%s: null pointer", who);
    VITMI_CHECK_ARG(!g->dgate || g->gate, "%s: gradient of an absent gate", who);
    VITMI_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "%s: the workspace must be aligned to 16 bytes", who);
    NgPlan p;
    if (!ng_plan(g->D, ng_vec(g), &p)) {
        vitmi_set_error("%s: no plan for D=%d", who, g->D);
        return VITMI_ERR_UNSUPPORTED;
    }
    VITMI_CHECK_ARG(!per_sample || g->B < (1 << 22), "%s: gates of %d samples are beyond one launch", who, g->B);
    NgArgs a;
    ng_fill(g, &a);
    a.chunks = ng_chunks(per_sample, g->B, g->N, p.wpr);
    a.partial = sums ? (float*)workspace : nullptr;
    const int segs = per_sample ? g->B : 1;
    hipStream_t s = as_stream(stream);
    const int ex = g->dt_x == VITMI_F32 ? 4 : 2, eu = g->dt_u == VITMI_F32 ? 4 : 2;
    ProfScope prof(VITMI_FAM_LAYERNORM, s, (double)a.rows * g->D * (3 * ex + 3 * eu));
    const unsigned blocks = (unsigned)(segs * a.chunks);
    if (g->dt_x == VITMI_BF16) ng_dispatch<bf16_t, bf16_t>(a, p, false, blocks, s);
    else if (g->dt_u == VITMI_BF16) ng_dispatch<float, bf16_t>(a, p, false, blocks, s);
    else ng_dispatch<float, float>(a, p, false, blocks, s);
    VITMI_LAUNCH_CHECK(who);
    if (sums) {
        NgFinal f = {a.partial, a.gate, a.gate_f32, a.gate_stride, a.post_w, a.post_b, g->dgate, g->dpost_w, g->dpost_b,
                     g->dpre_w, g->dpre_b, segs, a.chunks, g->D};
        hipLaunchKernelGGL(ngr_final_kernel, dim3(ceil_div(g->D, NF_COLS), 2), dim3(NF_COLS * NF_GROUPS), 0, s, f);
        VITMI_LAUNCH_CHECK(who);
    }
    return VITMI_OK;
}
