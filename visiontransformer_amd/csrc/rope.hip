// Rotary positions with several axes (time, height, width) on query / key rows [B, N, H, DH].
//
// Pair p of a head belongs to axis a and turns by theta = pos_a * base_a^(-j / s_a), j its index within the axis (or
// p / P over one ladder shared by the axes):
//     y1 = x1 cos(theta) - x2 sin(theta),   y2 = x2 cos(theta) + x1 sin(theta),
// the pair being dims (p, P + p) or (2p, 2p + 1); dims from 2P on pass through.  The backward pass is the same with -theta.
//
// Bound by HBM: every element is read once and written once, three operations each (256 x 197 tokens of 24 bf16 heads of 64:
// 62 us a pass, 5.0 TB/s; 2 x 21601 of 20 fp32 heads of 80: 103 us, 5.4 TB/s).  A workgroup takes a tile of
// tokens of one sample and ALL heads of both tensors, so that the angles of a token (the only expensive arithmetic) are
// formed once per tile and shared by the heads through LDS; its first row loads are on their way meanwhile.
// The angle is formed in turns in 64 bits and reduced to an eighth of a turn there -- a far position times a frequency
// keeps no fraction of a turn in 32 bits -- and only the reduced angle goes to the 32-bit sine and cosine.
#include <algorithm>

#include "common.h"

namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_MAX_PAIRS = 256;

struct RopeTensor {
    const void* x;
    void* y;
    long long xs[3], ys[3];   // batch, token, head strides
};
struct RopeArgs {
    RopeTensor t[2];
    const void* pos;
    long long ps[3];          // batch, token, axis strides
    double log2_base[4];
    int first_pair[5];        // first pair of each axis; [axes] = P
    int axes, pos_type, P, DH, N, tile, tiles;
    unsigned div_tok[2], div_head;
    int units_tok[2];         // units per token of each tensor
    int units_head, units_rot;
    int copy_rest;            // the pass-through dims are copied (not in place)
    int shared, inverse;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) RVec {
    T v[V];
};

// how a unit of V pairs lies in memory: two vectors of V elements P apart; one vector of 2V (interleaved); two single
// elements side by side (interleaved where no two-element vector fits: odd widths or strides)
enum { ROPE_HALVES = 0, ROPE_INTER = 1, ROPE_INTER_SCALAR = 2 };

template <typename T, int V, int MODE>
struct RopeUnit {
    RVec<T, MODE == ROPE_INTER ? 2 * V : V> a, b;
    T* y;                     // the unit's first vector in the output; NULL: no unit
    int cs;                   // where its angles start; < 0: a pass-through unit (vector a only)
};

// n / d for n, d < 2^16 with m = ceil(2^32 / d): a division would cost more than the rest of a unit's addressing
__device__ __forceinline__ int div16(int n, unsigned m) { return m ? (int)__umulhi((unsigned)n, m) : n; }

__device__ __forceinline__ double rope_pos(const RopeArgs& a, long long off) {
    if (a.pos_type == VITMI_POS_I64) return (double)((const long long*)a.pos)[off];
    if (a.pos_type == VITMI_POS_I32) return (double)((const int*)a.pos)[off];
    return (double)((const float*)a.pos)[off];
}

// cos and sin of 2 pi * turns, turns in 64 bits; the 32-bit functions see at most an eighth of a turn
__device__ __forceinline__ float2 rope_cos_sin(double turns) {
    const double t = turns - rint(turns), q = rint(4.0 * t);
    const float r = (float)(2.0 * (t - 0.25 * q));    // half turns in [-1/4, 1/4]
    float s, c;
    sincospif(r, &s, &c);
    const int k = (int)q & 3;
    const float c1 = (k & 1) ? -s : c, s1 = (k & 1) ? c : s;
    return (k & 2) ? make_float2(-c1, -s1) : make_float2(c1, s1);
}

// unit u of a tile of tensor W, whose first token's rows start at x and y
template <typename T, int V, int MODE, int W>
__device__ __forceinline__ void rope_fetch(const RopeArgs& a, RopeUnit<T, V, MODE>& r, int u, int total, const T* x, T* y) {
    r.y = nullptr;
    if (u >= total) return;
    const int tok = div16(u, a.div_tok[W]), rem = u - tok * a.units_tok[W];
    const int head = div16(rem, a.div_head), c = rem - head * a.units_head;
    constexpr int N = MODE == ROPE_INTER ? 2 * V : V;
    const bool rot = c < a.units_rot;
    const int d = rot ? c * (MODE == ROPE_HALVES ? V : 2 * V) : 2 * a.P + (c - a.units_rot) * N;
    x += tok * a.t[W].xs[1] + head * a.t[W].xs[2] + d;
    r.y = y + tok * a.t[W].ys[1] + head * a.t[W].ys[2] + d;
    r.cs = rot ? tok * a.P + c * V : -1;
    r.a = *reinterpret_cast<const RVec<T, N>*>(x);
    if (MODE != ROPE_INTER && rot) r.b = *reinterpret_cast<const RVec<T, N>*>(x + (MODE == ROPE_HALVES ? a.P : 1));
}

template <typename T, int V, int MODE>
__device__ __forceinline__ void rope_finish(const RopeArgs& a, RopeUnit<T, V, MODE>& r, const float2* cs) {
    if (!r.y) return;
    constexpr int N = MODE == ROPE_INTER ? 2 * V : V;
    if (r.cs >= 0) {
        const float2* w = cs + r.cs;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 t = w[j];
            T& e1 = MODE == ROPE_INTER ? r.a.v[2 * j] : r.a.v[j];
            T& e2 = MODE == ROPE_INTER ? r.a.v[2 * j + 1] : r.b.v[j];
            const float p = to_f32(e1), q = to_f32(e2);
            e1 = from_f32<T>(p * t.x - q * t.y);
            e2 = from_f32<T>(q * t.x + p * t.y);
        }
        if (MODE != ROPE_INTER) *reinterpret_cast<RVec<T, N>*>(r.y + (MODE == ROPE_HALVES ? a.P : 1)) = r.b;
    }
    *reinterpret_cast<RVec<T, N>*>(r.y) = r.a;
}

// units from `first` on of one sample's tile, K a thread in flight
template <typename T, int V, int MODE, int W, int K>
__device__ __forceinline__ void rope_walk(const RopeArgs& a, RopeUnit<T, V, MODE> (&r)[K], int first, int toks, int b, int n0, const float2* cs) {
    const RopeTensor& t = a.t[W];
    const int total = toks * a.units_tok[W];
    const T* x = (const T*)t.x + b * t.xs[0] + n0 * t.xs[1];
    T* y = (T*)t.y + b * t.ys[0] + n0 * t.ys[1];
    for (int u = first; u < total; u += K * ROPE_THREADS) {
#pragma unroll
        for (int i = 0; i < K; ++i) rope_fetch<T, V, MODE, W>(a, r[i], u + i * ROPE_THREADS, total, x, y);
#pragma unroll
        for (int i = 0; i < K; ++i) rope_finish<T, V, MODE>(a, r[i], cs);
    }
}

template <typename T, int V, int MODE>
__global__ __launch_bounds__(ROPE_THREADS) void rope_kernel(RopeArgs a) {
    extern __shared__ double rope_lds[];
    double* freq = rope_lds;                                   // [P] turns per position step
    float2* cs = reinterpret_cast<float2*>(rope_lds + a.P);     // [tile][P]
    const int b = blockIdx.x / a.tiles, n0 = (blockIdx.x - b * a.tiles) * a.tile;
    const int toks = min(a.tile, a.N - n0), t = threadIdx.x;
    constexpr int K = 3;
    RopeUnit<T, V, MODE> r[K];
    {
        const T* x = (const T*)a.t[0].x + b * a.t[0].xs[0] + n0 * a.t[0].xs[1];
        T* y = (T*)a.t[0].y + b * a.t[0].ys[0] + n0 * a.t[0].ys[1];
#pragma unroll
        for (int i = 0; i < K; ++i) rope_fetch<T, V, MODE, 0>(a, r[i], t + i * ROPE_THREADS, toks * a.units_tok[0], x, y);
    }
    if (t < a.P) {
        int ax = 0;
        while (t >= a.first_pair[ax + 1]) ++ax;
        const double e = a.shared ? (double)t / a.P
                                  : (double)(t - a.first_pair[ax]) / (a.first_pair[ax + 1] - a.first_pair[ax]);
        freq[t] = exp2(-e * a.log2_base[ax]) * 0.15915494309189533577;   // 1 / (2 pi)
    }
    __syncthreads();
    for (int i = t; i < toks * a.P; i += ROPE_THREADS) {
        const int tok = i / a.P, p = i - tok * a.P;
        int ax = 0;
        while (p >= a.first_pair[ax + 1]) ++ax;
        float2 w = rope_cos_sin(rope_pos(a, b * a.ps[0] + (n0 + tok) * a.ps[1] + ax * a.ps[2]) * freq[p]);
        if (a.inverse) w.y = -w.y;
        cs[i] = w;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i) rope_finish<T, V, MODE>(a, r[i], cs);
    rope_walk<T, V, MODE, 0, K>(a, r, t + K * ROPE_THREADS, toks, b, n0, cs);
    if (a.t[1].x) rope_walk<T, V, MODE, 1, K>(a, r, t, toks, b, n0, cs);
}

template <typename T>
void launch_rope(const RopeArgs& k, int mode, int V, unsigned blocks, size_t lds, hipStream_t s) {
#define ROPE_GO(v, m) hipLaunchKernelGGL((rope_kernel<T, v, m>), dim3(blocks), dim3(ROPE_THREADS), lds, s, k)
    if (mode == ROPE_INTER_SCALAR) ROPE_GO(1, ROPE_INTER_SCALAR);
    else if (mode == ROPE_INTER) {
        if (V == 1) ROPE_GO(1, ROPE_INTER);
        else if (V == 2) ROPE_GO(2, ROPE_INTER);
        else if constexpr (sizeof(T) == 2) ROPE_GO(4, ROPE_INTER);
    } else {
        if (V == 1) ROPE_GO(1, ROPE_HALVES);
        else if (V == 2) ROPE_GO(2, ROPE_HALVES);
        else if (V == 4) ROPE_GO(4, ROPE_HALVES);
        else if constexpr (sizeof(T) == 2) ROPE_GO(8, ROPE_HALVES);
    }
#undef ROPE_GO
}

}  // namespace

extern "C" int vitmi_rope_axes(const vitmi_rope_args* a, void* stream) {
    VITMI_CHECK_ARG(a, "vitmi_rope_axes: null arguments");
    VITMI_CHECK_ARG(a->dt == VITMI_F32 || a->dt == VITMI_BF16, "vitmi_rope_axes: bad dtype %d", a->dt);
    VITMI_CHECK_ARG(a->axes >= 1 && a->axes <= 4, "vitmi_rope_axes: %d axes, 1 to 4 are supported", a->axes);
    VITMI_CHECK_ARG(a->pos_type == VITMI_POS_I32 || a->pos_type == VITMI_POS_I64 || a->pos_type == VITMI_POS_F32,
                    "vitmi_rope_axes: bad position type %d", a->pos_type);
    VITMI_CHECK_ARG(a->B >= 0 && a->N >= 0 && a->DH > 0 && a->t[0].heads > 0, "vitmi_rope_axes: bad shape B=%d N=%d DH=%d H=%d",
                    a->B, a->N, a->DH, a->t[0].heads);
    RopeArgs k = {};
    int P = 0;
    for (int i = 0; i < a->axes; ++i) {
        VITMI_CHECK_ARG(a->sections[i] > 0 && a->sections[i] <= ROPE_MAX_PAIRS, "vitmi_rope_axes: section %d holds %d pairs", i,
                        a->sections[i]);
        VITMI_CHECK_ARG(a->log2_base[i] > 0, "vitmi_rope_axes: the base of axis %d must be above 1", i);
        k.first_pair[i] = P;
        k.log2_base[i] = a->log2_base[i];
        P += a->sections[i];
    }
    for (int i = a->axes; i < 5; ++i) k.first_pair[i] = P;
    VITMI_CHECK_ARG(P <= ROPE_MAX_PAIRS && 2 * P <= a->DH, "vitmi_rope_axes: %d pairs do not fit a head of %d (at most %d)", P,
                    a->DH, ROPE_MAX_PAIRS);
    if (a->B == 0 || a->N == 0) return VITMI_OK;
    VITMI_CHECK_ARG(a->pos && a->t[0].x && a->t[0].y, "vitmi_rope_axes: null pointer");
    VITMI_CHECK_ARG(!a->t[1].x || (a->t[1].y && a->t[1].heads > 0), "vitmi_rope_axes: second tensor without output or heads");

    const int esz = a->dt == VITMI_F32 ? 4 : 2;
    const int nt = a->t[1].x ? 2 : 1;
    // V pairs a unit: the widest vectors (16 bytes and below) that pairs, rest, strides and pointers are multiples of
    const bool inter = a->interleaved != 0;
    auto fits = [&](int pairs) {
        const int v = inter ? 2 * pairs : pairs;
        if (P % pairs || (a->DH - 2 * P) % v) return false;
        for (int i = 0; i < nt; ++i) {
            const vitmi_rope_tensor& t = a->t[i];
            if ((reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.y)) % (v * esz)) return false;
            for (int d = 0; d < 3; ++d)
                if (t.xs[d] % v || t.ys[d] % v) return false;
        }
        return true;
    };
    int V = inter ? 8 / esz : 16 / esz;
    while (V > 1 && !fits(V)) V >>= 1;
    const int mode = !inter ? ROPE_HALVES : V == 1 && !fits(1) ? ROPE_INTER_SCALAR : ROPE_INTER;
    long long heads = 0;
    bool in_place = true;
    for (int i = 0; i < nt; ++i) {
        const vitmi_rope_tensor& t = a->t[i];
        k.t[i].x = t.x;
        k.t[i].y = t.y;
        for (int d = 0; d < 3; ++d) {
            k.t[i].xs[d] = t.xs[d];
            k.t[i].ys[d] = t.ys[d];
            in_place = in_place && t.xs[d] == t.ys[d];
        }
        in_place = in_place && t.x == t.y;
        heads += t.heads;
    }
    k.pos = a->pos;
    for (int d = 0; d < 3; ++d) k.ps[d] = a->pos_stride[d];
    k.axes = a->axes;
    k.pos_type = a->pos_type;
    k.P = P;
    k.DH = a->DH;
    k.N = a->N;
    k.shared = a->shared_ladder;
    k.inverse = a->inverse;
    k.units_rot = P / V;
    const int rest = (a->DH - 2 * P) / (mode == ROPE_INTER ? 2 * V : V);
    k.units_head = k.units_rot + (in_place ? 0 : rest);
    auto magic = [](int d) { return d == 1 ? 0u : (unsigned)(((1ull << 32) + d - 1) / d); };
    long long ut = 1;                 // the larger tensor's units per token
    for (int i = 0; i < nt; ++i) {
        const long long n = (long long)a->t[i].heads * k.units_head;
        VITMI_CHECK_ARG(n < 65536, "vitmi_rope_axes: %d heads of %d are beyond one call", a->t[i].heads, a->DH);
        k.units_tok[i] = (int)n;
        k.div_tok[i] = magic((int)n);
        ut = std::max(ut, n);
    }
    k.div_head = magic(k.units_head);
    // tokens per workgroup: as many as 24 KB of rows share one round of angles (256 x 197 tokens of 24 bf16 heads of 64: 62 us
    // with 8 tokens, 67 with 4, 66 with 16; 2 x 21601 of 20 fp32 heads of 80: 103 with 2, 107 with 4, 117 with 8), fewer while
    // that leaves compute units without work
    int tile = 16;
    while (tile > 1 && ((long long)a->B * ceil_div(a->N, tile) < 1024 || tile * ut >= 65536 || tile * heads * a->DH * esz > 24 * 1024)) tile >>= 1;
    k.tile = tile;
    k.tiles = ceil_div(a->N, tile);
    const long long blocks = (long long)a->B * k.tiles;
    VITMI_CHECK_ARG(blocks < (1ll << 32) / ROPE_THREADS, "vitmi_rope_axes: %lld tiles are beyond one launch", blocks);
    hipStream_t s = as_stream(stream);
    ProfScope prof(VITMI_FAM_OTHER, s, 2.0 * a->B * a->N * heads * a->DH * esz);
    const size_t lds = (size_t)P * 8 * (1 + tile);
    if (a->dt == VITMI_F32) launch_rope<float>(k, mode, V, (unsigned)blocks, lds, s);
    else launch_rope<bf16_t>(k, mode, V, (unsigned)blocks, lds, s);
    VITMI_LAUNCH_CHECK("vitmi_rope_axes");
    return VITMI_OK;
}
