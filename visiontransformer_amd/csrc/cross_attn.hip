// Attention of query rows over the states of another sequence, q [B, Nq, Hq, D] over k, v [B, Nk, Hk, D]: lengths of
// their own, query heads that share a key head (group G = Hq / Hk), a key length per sample or a key mask.
//     s = scale q.k over the allowed keys,  p = softmax(s),  o = p v;   a sample without an allowed key gives o = 0
//     delta = sum_d dO o,  dp = dO.v,  ds = scale p (dp - delta),  dq = ds k,  dk = ds^T q,  dv = p^T dO (summed over the group)
// One (sample, key head) is one problem of R = G * Nq query rows (row r: head r / Nq of the group, position r % Nq) and Nk
// keys, so the heads of a group share the staged keys.
//
// All kernels work on 32 x 32 tiles of the matrix instructions with the index that a softmax or a sum runs along in a
// lane's REGISTERS and the other on the lane: S^T = K Q^T holds one query per lane, so that the row statistics are
// register work with a rare exchange between the two half waves, and the registers of P are the B operand of the next
// product as they are.  For bf16 the key rows of the first product are fed in a permuted order (key_of) so that these
// registers hold eight consecutive keys; the other operand (V^T, K^T, Q^T, dO^T) comes out of a row-major LDS image by
// transposing reads.  The fp32 form runs the same code over the fp32 matrix instruction.
//   forward      four waves of 32 rows share double-buffered tiles of 64 keys (fp32: 32); the running maximum is moved only
//                when a row outgrows it by 2^8, so the rescale of the accumulators almost never runs.
//   few rows     (up to 64 a problem: generation, pooling; small fp32 launches) the four waves share 32 rows and walk key
//                tiles of their own without a barrier; their results are joined in LDS.
//   short keys   (bf16, up to 256 keys) the whole backward pass in one launch, every probability formed once.
//   dq           four waves of 32 rows over all key tiles (S, dP, dq);  dk / dv: four waves of 32 keys over all row tiles
//                of all heads of the group (S, dP, dv, dk).  Seven products where five would do.
// No atomics: every sum runs in a fixed order, results are bitwise reproducible.  Where the tiles of a launch leave compute
// units idle, the inner loop is split over workgroups (dk / dv: equal shares of all tiles) that leave fp32 partial results
// in the workspace, joined by a second launch.
// Staging: 16-byte loads that land in LDS without a register between; they cost their issue and nothing else, and the next
// tile's are on their way during a tile's products.
// Rounding: in bf16, probabilities and dS are rounded to bf16 before the second product of each pair (the matrix instruction's
// operands; sums and statistics are 32-bit), which leaves results up to 1.5 times as far from the exact ones as rounding the
// exact result alone.  Two terms of P in the row form cost 19 % at 197 keys, 7 % at 77 and 32 % in the long shape below.  The
// few-row form, which waits for memory, and the one-launch backward pass of up to 32 keys have them.  delta is formed from the
// rounded output elsewhere: gradients of few ALLOWED keys there, where dP and delta nearly cancel, are up to 2.3 times as far off
// (0.0038 with two, 0.0027 with eight, 0.0025 with 32; rounding alone 0.0017).  One-term row sums add the rounded
// probabilities, so the weights sum to one.
// Measured (kernel alone; the chip holds about 1.9 GHz under these products):
//   2 x 4096 rows, 16 heads over 4 of 128, 4609 and 3457 keys, bf16: forward 316 us (857 TFLOP/s), dq 415, dk / dv 632 + 24 for
//   the join.  Matrix instructions run 48 % (forward), 49 % (dk / dv) and 56 % (dq) of the busy time: with two waves a SIMD the
//   exponentials, conversions and staging between the products are not covered in full.
//   32 x 12 heads of 64, 576 rows, 197 keys: forward 31 us, backward 73 + 7; 16 x 8 of 80, 1025 rows, 77 keys: 21, 39 + 7.
//   8 x 1 row, 32 heads over 8 of 128, about 12800 keys: 85 + 5 us, 5.0 TB/s of keys and values.
//   fp32, 8 x 6 heads of 64, 333 rows, 257 keys: 33, dq 43, dk / dv 48 + 8: 144 workgroups for 256 compute units, and matrix
//   instructions run 44 to 55 % of the busy time of those, one wave a SIMD with nothing to cover its waits.
//   Heads off the vector size (8 bf16 or 4 fp32 elements) and operands off a 16-byte border take element loads and the width of
//   128 throughout: 32 x 12 heads, 576 rows, 197 keys in bf16, forward 178 us with heads of 66, 157 of 36, 185 of 64 off a
//   border; backward 770, 641, 755.
// Masked keys: their K and V rows are staged as zeros whatever they hold, their scores are -inf.
#include <algorithm>
#include <atomic>

#include "common.h"
#include "shares.h"

namespace {

constexpr float XA_LOG2E = 1.4426950408889634f;
constexpr int XA_THREADS = 256;
constexpr float XA_SLACK = 8.f;     // log2 of how far a row may outgrow its running maximum before it is moved

struct XaArgs {
    const void *q, *k, *v;
    void* o;                              // dense [B, Nq, Hq, D]
    long long qs[3], ks[3], vs[3];        // batch, row, head strides
    const void* kv_len;                   // [B] int32 / int64 or NULL
    const unsigned char* key_mask;        // [B, Nk] or NULL
    long long mask_stride;
    int len64;
    float* lse;                           // [B, Hk, R], log2 domain; +inf: nothing to attend to
    float *part_o, *part_ml;              // [splits][B, Nq, Hq, D], [splits][B, Hk, R][2]
    int Nq, Nk, Hq, Hk, G, R, D, splits, tiles, whole;
    float c;                              // scale * log2(e)
    float scale;
    // backward
    const void* dout;
    long long dos[3];
    float* delta;                         // [B, Hk, R]
    void *dq, *dk, *dv;                   // dense, or NULL
    float *part_dq;
    float* part_kv;                       // [workgroups][first, last share][dk, dv][128][D]
    int B;
    long long n_q;                        // elements of q
};

template <typename T> struct Mx;
template <> struct Mx<bf16_t> {
    typedef bf16x8 frag;
    static constexpr int FE = 8, KD = 16;   // elements of a fragment per lane, contraction depth of a fragment
    static constexpr int KT = 64;           // sequence rows of a staged tile
};
template <> struct Mx<float> {
    typedef f32x4 frag;
    static constexpr int FE = 4, KD = 8;
    static constexpr int KT = 32;
};

__device__ __forceinline__ void mma(f32x16& acc, const bf16x8& a, const bf16x8& b) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& acc, const f32x4& a, const f32x4& b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], acc, 0, 0, 0);
}

// sequence index (0..31) fed as row m of a 32-row A operand, and the index that accumulator register e of half wave h
// then holds (the hardware's row of that register is 8 (e / 4) + 4 h + e % 4)
template <typename T> __device__ __forceinline__ int key_of_row(int m);
template <> __device__ __forceinline__ int key_of_row<bf16_t>(int m) {
    const int g = m >> 3;
    return 16 * (g >> 1) + 8 * ((m >> 2) & 1) + 4 * (g & 1) + (m & 3);
}
template <> __device__ __forceinline__ int key_of_row<float>(int m) { return (m & 24) + 2 * (m & 3) + ((m >> 2) & 1); }
template <typename T> __device__ __forceinline__ int key_of(int e, int h);
template <> __device__ __forceinline__ int key_of<bf16_t>(int e, int h) {
    const int g = e >> 2;
    return 16 * (g >> 1) + 8 * h + 4 * (g & 1) + (e & 3);
}
template <> __device__ __forceinline__ int key_of<float>(int e, int h) { return 8 * (e >> 2) + 2 * (e & 3) + h; }

// registers of a 32 x 32 accumulator as B operand: group n of KD consecutive sequence indices
__device__ __forceinline__ bf16x8 acc_frag(const f32x16& p, int n, bf16_t) {
    union {
        bf16x2 h[4];
        bf16x8 v;
    } u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u.h[i] = __builtin_convertvector(f32x2{p[8 * n + 2 * i], p[8 * n + 2 * i + 1]}, bf16x2);
    return u.v;
}
__device__ __forceinline__ f32x4 acc_frag(const f32x16& p, int n, float) {
    return f32x4{p[4 * n], p[4 * n + 1], p[4 * n + 2], p[4 * n + 3]};
}

// what the rounding to `hi` = acc_frag(p, n) left over, rounded in turn
__device__ __forceinline__ bf16x8 rest_frag(const f32x16& p, int n, const bf16x8& hi) {
    bf16x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (bf16_t)(p[8 * n + j] - (float)hi[j]);
    return r;
}

// l plus the sum of a fragment of probabilities: the rounded ones that the output is summed of, two an instruction; fp32 adds its
// own as they are formed
__device__ __forceinline__ float add_frag(const bf16x8& p, float l) {
    union {
        bf16x8 v;
        bf16x2 h[4];
    } u;
    u.v = p;
    const bf16x2 one = {(bf16_t)1.f, (bf16_t)1.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) l = __builtin_amdgcn_fdot2_f32_bf16(u.h[i], one, l, false);
    return l;
}
__device__ __forceinline__ float add_frag(const f32x4&, float l) { return l; }

template <typename T> __device__ __forceinline__ typename Mx<T>::frag zero_frag() {
    typename Mx<T>::frag z;
#pragma unroll
    for (int j = 0; j < Mx<T>::FE; ++j) z[j] = (T)0.f;
    return z;
}

// LDS image of KT sequence rows: planes of 32 dims, [DP / 32][KT][32].  A row of a plane is CP 16-byte chunks, chunk c of
// row r stored at c ^ swz(r).  With rows of 64 (bf16) or 128 bytes (fp32) both kinds of read then touch every bank once:
// 16 rows of one chunk (the rows of a row read), and for bf16 4 rows of all chunks (a transposing read), for fp32 two
// adjacent rows (a column read) -- and every address is a lane constant plus an immediate.
template <typename T> constexpr int cp_of() { return 32 * (int)sizeof(T) / 16; }
template <typename T> __device__ __forceinline__ int swz(int row) { return sizeof(T) == 2 ? (row >> 2) & 3 : (row >> 1) & 7; }
template <typename T> __device__ __forceinline__ int img_off(int row, int chunk) { return row * 32 + ((chunk ^ swz<T>(row)) * Mx<T>::FE); }

template <typename T, int KT>
__device__ __forceinline__ typename Mx<T>::frag row_frag(const T* img, int row, int c, int h) {
    constexpr int PER = 32 / Mx<T>::KD;      // fragments a plane
    return *reinterpret_cast<const typename Mx<T>::frag*>(img + (c / PER) * KT * 32 + img_off<T>(row, (c % PER) * 2 + h));
}
// A operand [32 dims of plane db as rows][KD sequence rows seq0..]: lane l holds dim l % 32 of the sequence rows that
// accumulator registers of half wave l / 32 hold (key_of)
template <int KT>
__device__ __forceinline__ bf16x8 col_frag(const bf16_t* img, int seq0, int db, int lane) {
    const int g = lane >> 4, q = (lane >> 2) & 3, p = lane & 3, row = 8 * (g >> 1) + q, chunk = 2 * (g & 1) + (p >> 1);
    const bf16_t* plane = img + db * KT * 32 + seq0 * 32 + 4 * (p & 1);
    typedef __attribute__((address_space(3))) s16x4* lp;
    union {
        s16x4 h[2];
        bf16x8 v;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(plane + img_off<bf16_t>(row, chunk)));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(plane + img_off<bf16_t>(row + 4, chunk)));
    return u.v;
}
template <int KT>
__device__ __forceinline__ f32x4 col_frag(const float* img, int seq0, int db, int lane) {
    const float* plane = img + db * KT * 32;
    const int d = lane & 31;
    f32x4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = plane[img_off<float>(seq0 + 2 * j + (lane >> 5), d >> 2) + (d & 3)];
    return r;
}

// FE elements of a row in global memory from dim d on; dims beyond D read as zero
template <typename T, bool VEC>
__device__ __forceinline__ typename Mx<T>::frag global_piece(const T* row, int d, int D) {
    typename Mx<T>::frag f = zero_frag<T>();
    if (VEC) {
        if (d < D) f = *reinterpret_cast<const typename Mx<T>::frag*>(row + d);
    } else {
#pragma unroll
        for (int j = 0; j < Mx<T>::FE; ++j)
            if (d + j < D) f[j] = row[d + j];
    }
    return f;
}

__device__ __forceinline__ int keys_of(const XaArgs& a, int b) {
    if (!a.kv_len) return a.Nk;
    const long long n = a.len64 ? ((const long long*)a.kv_len)[b] : (long long)((const int*)a.kv_len)[b];
    return (int)(n < 0 ? 0 : (n > a.Nk ? a.Nk : n));
}
// the same for a sample that the whole wave works on, in a scalar register
__device__ __forceinline__ int keys_of_wave(const XaArgs& a, int b) { return __builtin_amdgcn_readfirstlane(keys_of(a, b)); }
template <int KT> constexpr unsigned long long full_mask() { return ~0ull >> (64 - KT); }

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

__device__ __attribute__((aligned(16))) unsigned int xa_zero16[4] = {0u, 0u, 0u, 0u};

// Starts a load of 16 bytes a lane straight into LDS, lane i's at byte `to` + 16 i (`to` the same in the whole wave).  Inline
// assembly, because the compiler would hold every transposing LDS read back until such a load is complete, whichever
// image it fills; wait_loads() and a barrier stand between a load and the reads of its image.
__device__ __forceinline__ void load_to_lds(const void* from, unsigned to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"(to) : "memory", "m0");
}
// the same from a wave-uniform address plus a lane's byte offset: no vector arithmetic per load
__device__ __forceinline__ void load_to_lds(const void* base, unsigned offset, unsigned to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(to) : "memory", "m0");
}
__device__ __forceinline__ long long uniform(long long v) {       // a wave-uniform value into scalar registers
    const unsigned lo = __builtin_amdgcn_readfirstlane((int)(unsigned)v), hi = __builtin_amdgcn_readfirstlane((int)(unsigned)((unsigned long long)v >> 32));
    return (long long)(((unsigned long long)hi << 32) | lo);
}
template <typename P> __device__ __forceinline__ P* uniform(P* p) { return reinterpret_cast<P*>(uniform((long long)p)); }
__device__ __forceinline__ unsigned lds_addr(const void* p) {
    return (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)p);
}

// query row r of a group is position m of head g; without shared heads there is nothing to divide
__device__ __forceinline__ void split_row(int Nq, int R, int r, int& g, int& m) {
    g = 0;
    if (Nq != R) g = r / Nq;
    m = r - g * Nq;
}
__device__ __forceinline__ void split_row(const XaArgs& a, int r, int& g, int& m) { split_row(a.Nq, a.R, r, g, m); }

// A tile of KT rows of two matrices into their LDS images.  DMA: 16-byte loads that land in LDS without a register between
// (fetch starts them, they are complete after the next wait on vector memory), 64 lanes filling 1 KB of an image in
// its own order: a load instruction of 256 threads is PPI planes, so that a thread keeps one row.  Otherwise: through
// registers, fetched row by row, stored by store().  Rows whose mask bit is off and dims from D on are zeros.
template <typename T, int DP, bool VEC, int KT, int TH, bool DMA>
struct Stage {
    static constexpr int CP = cp_of<T>(), NP = DP / 32, PPI = TH / (KT * CP) > 0 ? TH / (KT * CP) : 1;
    static constexpr int CPR = NP * CP, IT = DMA ? 1 : KT * CPR / TH;
    static_assert(DMA ? PPI * KT * CP == TH && NP % PPI == 0 && VEC : KT * CPR % TH == 0, "a tile is a whole number of pieces per thread");
    typename Mx<T>::frag x[IT], y[IT];
    unsigned ox, oy;      // DMA: byte offsets of the thread's piece of plane 0 from a tile's first row
    int tail;             // DMA: dims from here on are beyond D in the thread's chunk of a plane that ends there
    bool near;            // a tile spans less than 4 GB of either matrix
    __device__ __forceinline__ void init(long long lx, long long ly, int D, int t) {
        if (!DMA) return;
        const int r = row_of(0, t), d = 32 * (t / (KT * CP)) + ((t % CP) ^ swz<T>(r)) * Mx<T>::FE;
        ox = (unsigned)((r * lx + d) * sizeof(T));
        oy = (unsigned)((r * ly + d) * sizeof(T));
        tail = D - d;
        near = uniform((lx > ly ? lx : ly) * KT * (long long)sizeof(T)) < (1ll << 32) - 4096;
    }
    // a whole tile whose first rows start at bx / by: only lanes beyond D have nothing to load, and their place in LDS holds the
    // zeros that the general form left there
    __device__ __forceinline__ void whole(const T* bx, const T* by, T* ix, T* iy, int D, int t) {
        bx = uniform(bx);
        by = uniform(by);
        const unsigned lx = lds_addr(ix + (t & ~63) * Mx<T>::FE), ly = lds_addr(iy + (t & ~63) * Mx<T>::FE);
#pragma unroll
        for (int p = 0; p < NP; p += PPI)
            if (32 * (p + PPI) <= D || 32 * p < tail) {
                load_to_lds(bx + 32 * p, ox, lx + p * KT * 32 * (unsigned)sizeof(T));
                load_to_lds(by + 32 * p, oy, ly + p * KT * 32 * (unsigned)sizeof(T));
            }
    }
    // the thread's row of a tile (DMA), or row of piece i
    __device__ __forceinline__ static int row_of(int i, int t) { return DMA ? t % (KT * CP) / CP : (t + i * TH) / CPR; }
    // px / py: start of the row that row_of names, valid where ok
    __device__ __forceinline__ void piece(int i, const T* px, const T* py, bool ok, T* ix, T* iy, int D, int t) {
        if (DMA) {
            const int r = row_of(0, t), chunk = (t % CP) ^ swz<T>(r);
#pragma unroll
            for (int p = 0; p < NP; p += PPI) {
                const int d = 32 * (p + t / (KT * CP)) + chunk * Mx<T>::FE;
                const bool on = ok && d < D;
                const void* sx = on ? (const void*)(px + d) : (const void*)xa_zero16;
                const void* sy = on ? (const void*)(py + d) : (const void*)xa_zero16;
                const int o = p * KT * 32 + (t & ~63) * Mx<T>::FE;
                load_to_lds(sx, lds_addr(ix + o));
                load_to_lds(sy, lds_addr(iy + o));
            }
        } else {
            const int d = ((t + i * TH) % CPR) * Mx<T>::FE;
            x[i] = y[i] = zero_frag<T>();
            if (ok) {
                x[i] = global_piece<T, VEC>(px, d, D);
                y[i] = global_piece<T, VEC>(py, d, D);
            }
        }
    }
    // key rows row0 + r with row strides lx, ly; `clean`: the images' places beyond D hold zeros already
    __device__ __forceinline__ void fetch(const T* px, long long lx, const T* py, long long ly, int row0, unsigned long long mask, T* ix,
                                          T* iy, int D, int t, bool clean) {
        if (DMA && mask == full_mask<KT>() && near && (clean || D == DP)) {
            whole(px + row0 * lx, py + row0 * ly, ix, iy, D, t);
            return;
        }
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int r = row_of(i, t);
            piece(i, px + (long long)(row0 + r) * lx, py + (long long)(row0 + r) * ly, (mask >> r) & 1, ix, iy, D, t);
        }
    }
    // query rows: row r of the flattened group is position r % Nq of head r / Nq
    __device__ __forceinline__ void fetch_rows(const T* px, const long long* sx, const T* py, const long long* sy, int row0, int R, int Nq, T* ix,
                                               T* iy, int D, int t, bool clean) {
        if (DMA && near && (clean || D == DP)) {
            int g0, n0;
            split_row(Nq, R, row0, g0, n0);
            if (n0 + KT <= Nq) {                          // all of one head
                whole(px + n0 * sx[1] + g0 * sx[2], py + n0 * sy[1] + g0 * sy[2], ix, iy, D, t);
                return;
            }
        }
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int r = row0 + row_of(i, t);
            int g, n;
            split_row(Nq, R, r, g, n);
            piece(i, px + n * sx[1] + g * sx[2], py + n * sy[1] + g * sy[2], r < R, ix, iy, D, t);
        }
    }
    __device__ __forceinline__ void store(T* ix, T* iy, int t) {
        if (DMA) return;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = t + i * TH, r = c / CPR, ch = c % CPR, o = (ch / CP) * KT * 32 + img_off<T>(r, ch % CP);
            *reinterpret_cast<typename Mx<T>::frag*>(ix + o) = x[i];
            *reinterpret_cast<typename Mx<T>::frag*>(iy + o) = y[i];
        }
    }
};

// The key mask of tiles t0, t0 + step, ..: cur is the running tile's, next the following one's; the mask bytes of the tile after
// that are already on their way
template <int KT>
struct MaskWalk {
    unsigned long long cur, next;
    int byte, n, step, b;
    __device__ __forceinline__ int load(const XaArgs& a, int tile, int lane) const {
        const int key = tile * KT + lane;
        return a.key_mask && lane < KT && key < n ? a.key_mask[b * a.mask_stride + key] : 0;
    }
    __device__ __forceinline__ unsigned long long bits(const XaArgs& a, int tile, int v) const {
        const long long left = (long long)n - (long long)tile * KT;
        if (left <= 0) return 0;
        const unsigned long long m = left >= 64 ? ~0ull : (1ull << left) - 1;
        return (a.key_mask ? __ballot(v != 0) : m) & m & full_mask<KT>();
    }
    __device__ __forceinline__ void start(const XaArgs& a, int b_, int n_, int t0, int step_, int lane) {
        b = b_;
        n = n_;
        step = step_;
        const int v0 = load(a, t0, lane), v1 = load(a, t0 + step, lane);
        byte = load(a, t0 + 2 * step, lane);
        cur = bits(a, t0, v0);
        next = bits(a, t0 + step, v1);
    }
    __device__ __forceinline__ void advance(const XaArgs& a, int tile, int lane) {     // from tile to tile + step
        cur = next;
        next = bits(a, tile + 2 * step, byte);
        byte = load(a, tile + 3 * step, lane);
    }
};

// every vector-memory load of the wave has landed, the LDS-bound ones among them; the builtin (vmcnt 0, the other counters
// free), so that the compiler knows it of its own loads too
__device__ __forceinline__ void wait_loads() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0F70);
    asm volatile("" ::: "memory");
}

// Workgroups are dealt to the 8 XCDs round-robin.  This cuts the launch into 16 contiguous pieces, two an XCD: neighbours in
// a piece read the same keys, which the XCD's L2 then fetches once, and the second piece comes from the other half of the
// batch, so that long and short samples even out over the XCDs.
__device__ __forceinline__ int xa_block() {
    const int n = gridDim.x, x = blockIdx.x & 7, slot = blockIdx.x >> 3;
    const int q = n >> 4, rem = n & 15;                        // pieces of q or q + 1
    const int first = q + (x < rem);                           // XCD x's first piece is piece x, its second x + 8
    const int p = slot < first ? x : x + 8, off = slot < first ? slot : slot - first;
    return p * q + (p < rem ? p : rem) + off;
}

// scores of one 32-key block against the lane's query
template <typename T, int DP, int KT>
__device__ __forceinline__ void scores(f32x16& s, const T* img, int key0, const typename Mx<T>::frag (&f)[DP / Mx<T>::KD], int lane) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
    const int row = key0 + key_of_row<T>(lane & 31);
#pragma unroll
    for (int c = 0; c < DP / Mx<T>::KD; ++c) mma(s, row_frag<T, KT>(img, row, c, lane >> 5), f[c]);
}

template <typename T>
__device__ __forceinline__ void mask_scores(f32x16& s, unsigned m, int h) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
        if (!((m >> key_of<T>(e, h)) & 1)) s[e] = -INFINITY;
}

// 32 staged keys (their images' rows from kimg, vimg on) against the lane's query: running softmax and o^T += V^T P^T.  TWO: P as a
// rounding and its rest, and its own sum in 32 bits, so that nothing but the result is rounded.
template <typename T, int DP, int KT, bool TWO = false>
__device__ __forceinline__ void attend(const T* kimg, const T* vimg, const typename Mx<T>::frag (&qf)[DP / Mx<T>::KD], unsigned mask, float c,
                                       f32x16 (&o)[DP / 32], float& m, float& l, int lane) {
    f32x16 s;
    scores<T, DP, KT>(s, kimg, 0, qf, lane);
    if (mask != ~0u) mask_scores<T>(s, mask, lane >> 5);
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx *= c;
    if (__any(mx > m + XA_SLACK)) {
        const float mn = fmaxf(m, fmaxf(mx, other_half(mx)));
        const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] *= f;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], c, -m));
        if (sizeof(T) == 4 || TWO) l += s[e];
    }
#pragma unroll
    for (int n = 0; n < 32 / Mx<T>::KD; ++n) {
        const typename Mx<T>::frag pf = acc_frag(s, n, T());
        if constexpr (TWO) {
            const typename Mx<T>::frag pr = rest_frag(s, n, pf);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) {
                const typename Mx<T>::frag vf = col_frag<KT>(vimg, n * Mx<T>::KD, d, lane);
                mma(o[d], vf, pf);
                mma(o[d], vf, pr);
            }
        } else {
            l = add_frag(pf, l);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) mma(o[d], col_frag<KT>(vimg, n * Mx<T>::KD, d, lane), pf);
        }
    }
}

// four consecutive dims (8 g + 4 h ..) of an accumulator block to a dense row
template <typename T, bool VEC>
__device__ __forceinline__ void store4(T* row, int d, int D, float v0, float v1, float v2, float v3) {
    if (VEC) {
        if (d < D) {
            T p[4] = {from_f32<T>(v0), from_f32<T>(v1), from_f32<T>(v2), from_f32<T>(v3)};
            struct alignas(4 * sizeof(T)) Q {
                T v[4];
            };
            *reinterpret_cast<Q*>(row + d) = *reinterpret_cast<Q*>(p);
        }
    } else {
        const float v[4] = {v0, v1, v2, v3};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (d + j < D) row[d + j] = from_f32<T>(v[j]);
    }
}
// a 32-dim block of an accumulator to dims d0.. of a dense row.  bf16: the half waves hold four dims of every eight each and
// swap one group of a pair, so that a lane stores 16 bytes and a row 32 together.
template <typename T, bool VEC>
__device__ __forceinline__ void store_block(T* row, int d0, const f32x16& o, float f, int h, int D) {
    if constexpr (VEC && sizeof(T) == 2) {
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
            union {
                bf16x2 v[2];
                unsigned w[2];
            } x, y;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                x.v[i] = __builtin_convertvector(f32x2{o[4 * g + 2 * i] * f, o[4 * g + 2 * i + 1] * f}, bf16x2);
                y.v[i] = __builtin_convertvector(f32x2{o[4 * g + 4 + 2 * i] * f, o[4 * g + 5 + 2 * i] * f}, bf16x2);
            }
            u32x4 out;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const auto r = __builtin_amdgcn_permlane32_swap(x.w[i], y.w[i], false, false);
                out[i] = r[0];
                out[2 + i] = r[1];
            }
            const int d = d0 + 8 * (g + h);
            if (row && d < D) *reinterpret_cast<u32x4*>(row + d) = out;
        }
    } else if (row) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
            store4<T, VEC>(row, d0 + 8 * g + 4 * h, D, o[4 * g] * f, o[4 * g + 1] * f, o[4 * g + 2] * f, o[4 * g + 3] * f);
    }
}
// a NULL row is not stored, but its lane takes part in the exchange
template <typename T, bool VEC, int DP>
__device__ __forceinline__ void store_acc(T* row, const f32x16 (&o)[DP / 32], float f, int h, int D) {
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) store_block<T, VEC>(row, 32 * db, o[db], f, h, D);
}

// element offset of query row r of problem (b, hk) in a dense [B, Nq, Hq, D]
__device__ __forceinline__ long long dense_row(const XaArgs& a, int b, int hk, int r) {
    int g, n;
    split_row(a, r, g, n);
    return (((long long)b * a.Nq + n) * a.Hq + hk * a.G + g) * a.D;
}

// result rows of a forward kernel: normalised output and lse, or (splits) unnormalised partials
template <typename T, int DP, bool VEC>
__device__ __forceinline__ void finish_rows(const XaArgs& a, int b, int hk, int r, int split, const f32x16 (&o)[DP / 32], float m, float l,
                                            int h) {
    const bool in = r < a.R;
    const long long row = in ? dense_row(a, b, hk, r) : 0, st = ((long long)b * a.Hk + hk) * a.R + r;
    if (a.splits == 1) {
        store_acc<T, VEC, DP>(in ? (T*)a.o + row : nullptr, o, l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l), h, a.D);
        if (in && a.lse && h == 0) a.lse[st] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
    } else {
        store_acc<float, VEC, DP>(in ? a.part_o + split * a.n_q + row : nullptr, o, 1.f, h, a.D);
        if (in && h == 0) {
            float2* ml = reinterpret_cast<float2*>(a.part_ml) + (long long)split * (a.n_q / a.D) + st;
            *ml = make_float2(m, l);
        }
    }
}

// this workgroup's share [t0, t1) of `tiles` tiles
__device__ __forceinline__ void split_range(int tiles, int splits, int split, int& t0, int& t1) {
    t0 = (int)((long long)tiles * split / splits);
    t1 = (int)((long long)tiles * (split + 1) / splits);
}

template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(XA_THREADS, sizeof(T) == 4 ? 1 : 2) void xattn_fwd_kernel(XaArgs a) {
    constexpr int KT = Mx<T>::KT, IMG = KT * DP;
    extern __shared__ __align__(16) char xa_lds[];
    T* const lds = reinterpret_cast<T*>(xa_lds);        // K, V, K, V
    const int t = threadIdx.x, lane = t & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    int idx = xa_block();
    const int rt = idx % a.tiles;
    idx /= a.tiles;
    const int split = idx % a.splits;
    idx /= a.splits;
    const int hk = idx % a.Hk, b = idx / a.Hk;
    const int r = rt * 128 + wave * 32 + (lane & 31);
    const bool busy = rt * 128 + wave * 32 < a.R;         // the wave has a row; without one it only helps staging
    typename Mx<T>::frag qf[DP / Mx<T>::KD];
    {
        int g, n;
        split_row(a, r, g, n);
        const T* qp = (const T*)a.q + b * a.qs[0] + n * a.qs[1] + (hk * a.G + g) * a.qs[2];
#pragma unroll
        for (int c = 0; c < DP / Mx<T>::KD; ++c)
            qf[c] = r < a.R ? global_piece<T, VEC>(qp, c * Mx<T>::KD + h * Mx<T>::FE, a.D) : zero_frag<T>();
    }
    f32x16 o[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    const int n = keys_of_wave(a, b);
    const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
    const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
    int t0, t1;
    split_range((n + KT - 1) / KT, a.splits, split, t0, t1);
    Stage<T, DP, VEC, KT, XA_THREADS, VEC> st;
    MaskWalk<KT> mw;
    st.init(a.ks[1], a.vs[1], a.D, t);
    if (t0 < t1) {
        mw.start(a, b, n, t0, 1, lane);
        T* img = lds + (t0 & 1) * 2 * IMG;
        st.fetch(kp, a.ks[1], vp, a.vs[1], t0 * KT, mw.cur, img, img + IMG, a.D, t, false);
    }
    for (int kt = t0; kt < t1; ++kt) {
        T* img = lds + (kt & 1) * 2 * IMG;
        const unsigned long long mk = mw.cur;
        st.store(img, img + IMG, t);
        wait_loads();
        __syncthreads();
        if (kt + 1 < t1) {
            T* nxt = lds + ((kt + 1) & 1) * 2 * IMG;
            st.fetch(kp, a.ks[1], vp, a.vs[1], (kt + 1) * KT, mw.next, nxt, nxt + IMG, a.D, t, kt > t0);
            mw.advance(a, kt, lane);
        }
        if (busy && mk) {
#pragma unroll
            for (int kb = 0; kb < KT / 32; ++kb)          // blocks of 32 keys without an allowed one are left out
                if ((unsigned)(mk >> (32 * kb))) attend<T, DP, KT>(img + kb * 1024, img + IMG + kb * 1024, qf, (unsigned)(mk >> (32 * kb)), a.c, o, m, l, lane);
        }
    }
    l += other_half(l);
    finish_rows<T, DP, VEC>(a, b, hk, r, split, o, m, l, h);
}

// one wave's LDS image is written and read by that wave alone: its LDS operations run in order, only the compiler is held
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Few rows: every wave walks 32-key tiles of its own for the same 32 rows.  Bound by the bytes of K and V, which go
// through registers: a wave waits for its own loads alone, four of them a SIMD cover for each other (5.0 TB/s at 8 x 8 key heads of
// 128).  P enters its product as two bf16 terms, which costs nothing beside the loads (82 us either way).
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(XA_THREADS) void xattn_few_kernel(XaArgs a) {
    constexpr int KT = 32, IMG = KT * DP;
    extern __shared__ __align__(16) char xa_lds[];
    const int t = threadIdx.x, lane = t & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    T* const img = reinterpret_cast<T*>(xa_lds) + wave * 2 * IMG;
    int idx = xa_block();
    const int rt = idx % a.tiles;
    idx /= a.tiles;
    const int split = idx % a.splits;
    idx /= a.splits;
    const int hk = idx % a.Hk, b = idx / a.Hk;
    const int r = rt * 32 + (lane & 31);
    const int n = keys_of_wave(a, b);
    const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
    const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
    int t0, t1;
    split_range((n + KT - 1) / KT, a.splits, split, t0, t1);
    Stage<T, DP, VEC, KT, 64, false> st;
    MaskWalk<KT> mw;
    if (t0 + wave < t1) {
        mw.start(a, b, n, t0 + wave, 4, lane);
        st.fetch(kp, a.ks[1], vp, a.vs[1], (t0 + wave) * KT, mw.cur, nullptr, nullptr, a.D, lane, false);
    }
    typename Mx<T>::frag qf[DP / Mx<T>::KD];
    {
        int g, nn;
        split_row(a, r, g, nn);
        const T* qp = (const T*)a.q + b * a.qs[0] + nn * a.qs[1] + (hk * a.G + g) * a.qs[2];
#pragma unroll
        for (int c = 0; c < DP / Mx<T>::KD; ++c)
            qf[c] = r < a.R ? global_piece<T, VEC>(qp, c * Mx<T>::KD + h * Mx<T>::FE, a.D) : zero_frag<T>();
    }
    f32x16 o[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    for (int kt = t0 + wave; kt < t1; kt += 4) {
        const unsigned long long mk = mw.cur;
        st.store(img, img + IMG, lane);
        wave_fence();
        if (kt + 4 < t1) {
            st.fetch(kp, a.ks[1], vp, a.vs[1], (kt + 4) * KT, mw.next, nullptr, nullptr, a.D, lane, false);
            mw.advance(a, kt, lane);
        }
        if (mk) attend<T, DP, KT, sizeof(T) == 2>(img, img + IMG, qf, (unsigned)mk, a.c, o, m, l, lane);
        wave_fence();
    }
    l += other_half(l);
    // join the four waves in wave order: running maxima first, then the rescaled sums and outputs
    float* const xo = reinterpret_cast<float*>(xa_lds);                    // [4][DP][32] after the barrier
    float* const xm = xo + 4 * DP * 32;                                   // [4][32][2]
    __syncthreads();
    if (h == 0) {
        xm[(wave * 32 + (lane & 31)) * 2] = m;
        xm[(wave * 32 + (lane & 31)) * 2 + 1] = l;
    }
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) xo[(wave * DP + 32 * d + 8 * (e >> 2) + 4 * h + (e & 3)) * 32 + (lane & 31)] = o[d][e];
    __syncthreads();
    float mm = -INFINITY, w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) mm = fmaxf(mm, xm[(i * 32 + (lane & 31)) * 2]);
    l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float mi = xm[(i * 32 + (lane & 31)) * 2], li = xm[(i * 32 + (lane & 31)) * 2 + 1];
        w[i] = mi == -INFINITY ? (li == 0.f ? 0.f : li) : __builtin_amdgcn_exp2f(mi - mm);
        l += mi == -INFINITY ? li : li * w[i];
    }
    m = mm;
    if (r >= a.R) return;
    const float f = a.splits == 1 ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;
    const long long row = dense_row(a, b, hk, r), sti = ((long long)b * a.Hk + hk) * a.R + r;
    // the waves share the dims of the output: 8 consecutive ones a thread and step
    for (int d = 8 * (2 * wave + h); d < DP; d += 64) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float oi = xo[(i * DP + d + j) * 32 + (lane & 31)];
                v[j] = w[i] == 0.f ? v[j] : fmaf(oi, w[i], v[j]);
            }
            v[j] *= f;
        }
        if (a.splits == 1) {
            store4<T, VEC>((T*)a.o + row, d, a.D, v[0], v[1], v[2], v[3]);
            store4<T, VEC>((T*)a.o + row, d + 4, a.D, v[4], v[5], v[6], v[7]);
        } else {
            store4<float, VEC>(a.part_o + split * a.n_q + row, d, a.D, v[0], v[1], v[2], v[3]);
            store4<float, VEC>(a.part_o + split * a.n_q + row, d + 4, a.D, v[4], v[5], v[6], v[7]);
        }
    }
    if (wave == 0 && h == 0) {
        if (a.splits == 1) {
            if (a.lse) a.lse[sti] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
        } else {
            reinterpret_cast<float2*>(a.part_ml)[(long long)split * (a.n_q / a.D) + sti] = make_float2(m, l);
        }
    }
}

// Joins the key splits (at most 64) of a forward launch, one wave a row: lane s holds split s's maximum and sum, the partial rows
// are then added in split order, eight loads in flight
template <typename T>
__global__ __launch_bounds__(256) void xattn_join_kernel(XaArgs a, long long rows) {
    const int lane = threadIdx.x & 63;
    const long long st = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (st >= rows) return;
    const int r = (int)(st % a.R);
    const long long bh = st / a.R;
    const int hk = (int)(bh % a.Hk), b = (int)(bh / a.Hk);
    float2 p = make_float2(-INFINITY, 0.f);
    if (lane < a.splits) p = reinterpret_cast<const float2*>(a.part_ml)[lane * rows + st];
    const float m = wave_max(p.x);
    // a share without an allowed key counts for nothing, whatever its partial row holds
    const float w = p.y == 0.f ? 0.f : (p.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(p.x - m));
    const float l = wave_sum(p.y == 0.f ? 0.f : p.y * w);
    const long long row = dense_row(a, b, hk, r);
    const bool in0 = lane < a.D, in1 = lane + 64 < a.D;
    float o0 = 0.f, o1 = 0.f;
    for (int s0 = 0; s0 < a.splits; s0 += 8) {
        float x0[8], x1[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float* po = a.part_o + (s0 + i) * a.n_q + row + lane;
            const bool on = s0 + i < a.splits;
            x0[i] = on && in0 ? po[0] : 0.f;
            x1[i] = on && in1 ? po[64] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float wi = __shfl(w, (s0 + i) & 63, 64);
            if (s0 + i < a.splits && wi != 0.f) {
                o0 = fmaf(x0[i], wi, o0);
                o1 = fmaf(x1[i], wi, o1);
            }
        }
    }
    const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    T* op = (T*)a.o + row;
    if (in0) op[lane] = from_f32<T>(o0 * f);
    if (in1) op[lane + 64] = from_f32<T>(o1 * f);
    if (a.lse && lane == 0) a.lse[st] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// dq (and delta, which the dk / dv launch reads): four waves of 32 rows over the key tiles, two products of 32 x 32 scores
// and one that turns them into dq; 415 us at the long shape above, 977 TFLOP/s of its own three products
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(XA_THREADS, sizeof(T) == 4 || !VEC ? 1 : 2) void xattn_dq_kernel(XaArgs a) {
    constexpr int KT = Mx<T>::KT, IMG = KT * DP, NF = DP / Mx<T>::KD;
    extern __shared__ __align__(16) char xa_lds[];
    T* const lds = reinterpret_cast<T*>(xa_lds);
    const int t = threadIdx.x, lane = t & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    int idx = xa_block();
    const int rt = idx % a.tiles;
    idx /= a.tiles;
    const int split = idx % a.splits;
    idx /= a.splits;
    const int hk = idx % a.Hk, b = idx / a.Hk;
    const int r = rt * 128 + wave * 32 + (lane & 31);
    const bool in = r < a.R;
    const long long row = in ? dense_row(a, b, hk, r) : 0, sti = ((long long)b * a.Hk + hk) * a.R + r;
    typename Mx<T>::frag qf[NF], gf[NF];
    float lse = INFINITY, delta = 0.f;
    {
        int g, n;
        split_row(a, r, g, n);
        const T* qp = (const T*)a.q + b * a.qs[0] + n * a.qs[1] + (hk * a.G + g) * a.qs[2];
        const T* gp = (const T*)a.dout + b * a.dos[0] + n * a.dos[1] + (hk * a.G + g) * a.dos[2];
        const T* op = (const T*)a.o + row;
#pragma unroll
        for (int c = 0; c < NF; ++c) {
            const int d = c * Mx<T>::KD + h * Mx<T>::FE;
            qf[c] = in ? global_piece<T, VEC>(qp, d, a.D) : zero_frag<T>();
            gf[c] = in ? global_piece<T, VEC>(gp, d, a.D) : zero_frag<T>();
            const typename Mx<T>::frag of = in ? global_piece<T, VEC>(op, d, a.D) : zero_frag<T>();
#pragma unroll
            for (int j = 0; j < Mx<T>::FE; ++j) delta = fmaf(to_f32(gf[c][j]), to_f32(of[j]), delta);
        }
        if (in) lse = a.lse[sti];
    }
    delta += other_half(delta);
    if (in && h == 0 && split == 0) a.delta[sti] = delta;
    f32x16 acc[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
    const int n = keys_of_wave(a, b);
    const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
    const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
    int t0, t1;
    split_range(a.dq ? (n + KT - 1) / KT : 0, a.splits, split, t0, t1);      // without dq only delta is wanted
    Stage<T, DP, VEC, KT, XA_THREADS, VEC> st;
    MaskWalk<KT> mw;
    st.init(a.ks[1], a.vs[1], a.D, t);
    if (t0 < t1) {
        mw.start(a, b, n, t0, 1, lane);
        T* img = lds + (t0 & 1) * 2 * IMG;
        st.fetch(kp, a.ks[1], vp, a.vs[1], t0 * KT, mw.cur, img, img + IMG, a.D, t, false);
    }
    for (int kt = t0; kt < t1; ++kt) {
        T* img = lds + (kt & 1) * 2 * IMG;
        const unsigned long long mk = mw.cur;
        st.store(img, img + IMG, t);
        wait_loads();
        __syncthreads();
        if (kt + 1 < t1) {
            T* nxt = lds + ((kt + 1) & 1) * 2 * IMG;
            st.fetch(kp, a.ks[1], vp, a.vs[1], (kt + 1) * KT, mw.next, nxt, nxt + IMG, a.D, t, kt > t0);
            mw.advance(a, kt, lane);
        }
        if (mk && rt * 128 + wave * 32 < a.R) {
#pragma unroll
            for (int kb = 0; kb < KT / 32; ++kb) {
                if (!(unsigned)(mk >> (32 * kb))) continue;
                f32x16 s, dp;
                scores<T, DP, KT>(s, img, 32 * kb, qf, lane);
                scores<T, DP, KT>(dp, img + IMG, 32 * kb, gf, lane);
                if (mk != full_mask<KT>()) mask_scores<T>(s, (unsigned)(mk >> (32 * kb)), h);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.c, -lse)) * (dp[e] - delta);
#pragma unroll
                for (int g = 0; g < 32 / Mx<T>::KD; ++g) {
                    const typename Mx<T>::frag f = acc_frag(s, g, T());
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) mma(acc[d], col_frag<KT>(img, 32 * kb + g * Mx<T>::KD, d, lane), f);
                }
            }
        }
    }
    if (!a.dq) return;
    if (a.splits == 1)
        store_acc<T, VEC, DP>(in ? (T*)a.dq + row : nullptr, acc, a.scale, h, a.D);
    else
        store_acc<float, VEC, DP>(in ? a.part_dq + split * a.n_q + row : nullptr, acc, 1.f, h, a.D);
}

// sum over the 32 lanes of a half wave, the same value in each of them, in a fixed order: shifts within the rows of 16, one exchange
__device__ __forceinline__ float half_wave_sum(float v) {
#define XA_STEP(ctrl) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, 0xf, 0xf, true))
    XA_STEP(0xb1);    // quad_perm 1 0 3 2
    XA_STEP(0x4e);    // quad_perm 2 3 0 1
    XA_STEP(0x141);   // row_half_mirror
    XA_STEP(0x140);   // row_mirror
#undef XA_STEP
    return v + __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401f));    // lane ^ 16
}

// dq, dk and dv of up to 32 NW keys in one launch (bf16): all keys of a problem fit the registers of one workgroup, wave w
// owning keys 32 w .. with their K and V fragments and their dk and dv, and an image of K in LDS.  The workgroup walks
// tiles of 32 SUB query rows; S, dP and dS of a tile are formed once (the two-launch form pays for the exponentials twice, and
// at heads of 64 they take longer than the products) and feed dk and dv as in xattn_dkv_kernel.  Every wave also leaves its dS
// as [key][row] in LDS -- the packed fragments as they are, two 16-byte writes a lane -- from where the tile's dq^T =
// K^T dS^T is formed over all keys, in pieces of 32 dims that the waves take in turns, a tile behind (NOW: a piece a wave, at
// once, which needs one dS image in place of two).  delta is formed from dO and O on the way in.
// Up to 32 keys (ONE) are all of one wave.  Few keys do not average roundings out, that of O, through delta, among them: with 7 keys
// gradients would be 0.0030 off, with 77 0.0024, where rounding the exact ones leaves 0.0017.  So delta = sum_k p dp is summed
// from the scores there, and P and dS enter the products as two bf16 terms each, a rounding and its rest: 0.0018 with 7 keys.
// The products are a small part of so few keys' work.
template <int DP, int NW, int SUB, bool ONE>
__global__ __launch_bounds__(64 * NW, 2) void xattn_bwd_short_kernel(XaArgs a) {
    typedef bf16_t T;
    constexpr int TH = 64 * NW, NK = 32 * NW, QT = 32 * SUB, NP = DP / 32, NF = DP / 16, IMG = QT * DP, DS = NK * QT;
    constexpr bool NOW = NP * SUB == NW;
    constexpr int TPR = TH / QT, NPC = (DP / 8 + TPR - 1) / TPR;
    extern __shared__ __align__(16) char xa_lds[];
    T* const kimg = reinterpret_cast<T*>(xa_lds);
    T* const lds = kimg + NK * DP;                        // Q, dO, Q, dO
    T* const dsi = lds + 4 * IMG;
    float* const rows = reinterpret_cast<float*>(dsi + (NOW ? 1 : 2) * DS);     // [2][lse, delta][QT]
    const int t = threadIdx.x, lane = t & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // the first a.whole problems have a workgroup each, the others share their rows among a.splits
    const int idx = xa_block();
    const bool shared = idx >= a.whole;
    const int sh = shared ? (idx - a.whole) / a.splits : 0, split = shared ? (idx - a.whole) - sh * a.splits : 0;
    const int bh = shared ? a.whole + sh : idx, b = bh / a.Hk, hk = bh - b * a.Hk;
    const int n = keys_of_wave(a, b), RT = (a.R + QT - 1) / QT;
    int t0, t1;
    split_range(RT, shared ? a.splits : 1, split, t0, t1);
    const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
    const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
    const T* qp = (const T*)a.q + b * a.qs[0] + (long long)hk * a.G * a.qs[2];
    const T* gp = (const T*)a.dout + b * a.dos[0] + (long long)hk * a.G * a.dos[2];
    const long long sti = ((long long)b * a.Hk + hk) * a.R;
    auto allowed = [&](int key) { return key < n && (!a.key_mask || a.key_mask[b * a.mask_stride + key] != 0); };

    // 1 KB of an image (16 rows of one plane) a load instruction; a wave keeps 16 of a tile's rows
    const int lrow = lane >> 2;
    auto piece = [&](const T* row, bool ok, int plane, int r, T* img, int rows_img, int r0) {
        const int d = 32 * plane + ((lane & 3) ^ swz<T>(r)) * 8;
        load_to_lds(ok && d < a.D ? (const void*)(row + d) : (const void*)xa_zero16, lds_addr(img + plane * rows_img * 32 + r0 * 32));
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r0 = 16 * (2 * wave + i), r = r0 + lrow;
        const bool ok = allowed(r);
#pragma unroll
        for (int p = 0; p < NP; ++p) piece(kp + r * a.ks[1], ok, p, r, kimg, NK, r0);
    }
    bf16x8 dof[NPC], of[NPC];
    float lse = INFINITY;
    auto issue = [&](int tile, int pair) {
        T* img = lds + pair * 2 * IMG;
        {
            const int r0 = 16 * (wave % (2 * SUB)), lr = r0 + lrow, r = tile * QT + lr;
            int g, m;
            split_row(a, r, g, m);
            const T *q = qp + m * a.qs[1] + g * a.qs[2], *d = gp + m * a.dos[1] + g * a.dos[2];
#pragma unroll
            for (int u = wave / (2 * SUB); u < 2 * NP; u += NW / (2 * SUB)) {
                if (u < NP) piece(q, r < a.R, u, lr, img, QT, r0);
                else piece(d, r < a.R, u - NP, lr, img + IMG, QT, r0);
            }
        }
        const int r = tile * QT + t / TPR;
        int g, m;
        split_row(a, r, g, m);
        const T* d = gp + m * a.dos[1] + g * a.dos[2];
        const T* o = (const T*)a.o + (((long long)b * a.Nq + m) * a.Hq + hk * a.G + g) * a.D;
        lse = INFINITY;
#pragma unroll
        for (int i = 0; i < NPC; ++i) {
            const int c = (t % TPR + TPR * i) * 8;
            dof[i] = of[i] = zero_frag<T>();
            if (!ONE && r < a.R && c < a.D) {
                dof[i] = *reinterpret_cast<const bf16x8*>(d + c);
                of[i] = *reinterpret_cast<const bf16x8*>(o + c);
            }
        }
        if (r < a.R && t % TPR == 0) lse = a.lse[sti + r];
    };
    auto leave_stats = [&](int pair) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NPC; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) s = fmaf(to_f32(dof[i][j]), to_f32(of[i][j]), s);
#pragma unroll
        for (int o = 1; o < TPR; o <<= 1) s += __shfl_xor(s, o, 64);
        if (t % TPR == 0) {
            rows[pair * 2 * QT + t / TPR] = lse;
            rows[pair * 2 * QT + QT + t / TPR] = s;
        }
    };
    if (t0 < t1) issue(t0, t0 & 1);

    const int key = wave * 32 + (lane & 31);
    const bool on = allowed(key);
    const bool all_on = __all(on), any_on = __any(on);
    constexpr bool KL = DP == 128;                        // K fragments out of the image: registers for them run out
    bf16x8 kf[KL ? 1 : NF], vf[NF];
#pragma unroll
    for (int c = 0; c < NF; ++c) {
        if (!KL) kf[KL ? 0 : c] = on ? global_piece<T, true>(kp + key * a.ks[1], c * 16 + h * 8, a.D) : zero_frag<T>();
        vf[c] = on ? global_piece<T, true>(vp + key * a.vs[1], c * 16 + h * 8, a.D) : zero_frag<T>();
    }
    f32x16 dk[NP], dv[NP];
#pragma unroll
    for (int d = 0; d < NP; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[d][e] = dv[d][e] = 0.f;
    auto ds_at = [&](int pair, int sub, int c) { return reinterpret_cast<bf16x8*>(dsi + (NOW ? 0 : pair * DS) + sub * NK * 32 + img_off<T>(key, c)); };
    if (!any_on) {                                        // a wave without a key leaves no dS: zeros stand in for it
#pragma unroll
        for (int p = 0; p < (NOW ? 1 : 2) * SUB; ++p) *ds_at(p / SUB, p % SUB, 2 * h) = *ds_at(p / SUB, p % SUB, 2 * h + 1) = zero_frag<T>();
    }
    const int blocks = (n + 31) >> 5;
    auto dq_piece = [&](int tile, int sub, int j) {
        const T* di = dsi + (NOW ? 0 : (tile & 1) * DS) + sub * NK * 32;
        f32x16 acc, alt;                                  // two chains: one would wait for itself
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] = alt[e] = 0.f;
#pragma unroll 2
        for (int kb = 0; kb < blocks; ++kb) {
            mma(acc, col_frag<NK>(kimg + kb * 1024, 0, j, lane), col_frag<NK>(di + kb * 1024, 0, 0, lane));
            mma(alt, col_frag<NK>(kimg + kb * 1024, 16, j, lane), col_frag<NK>(di + kb * 1024, 16, 0, lane));
            if (ONE) {                                    // the rests lie where a second wave's dS would
                mma(acc, col_frag<NK>(kimg, 0, j, lane), col_frag<NK>(di + 1024, 0, 0, lane));
                mma(alt, col_frag<NK>(kimg, 16, j, lane), col_frag<NK>(di + 1024, 16, 0, lane));
            }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] += alt[e];
        const int r = tile * QT + 32 * sub + (lane & 31);
        store_block<T, true>(r < a.R ? (T*)a.dq + dense_row(a, b, hk, r) : nullptr, 32 * j, acc, a.scale, h, a.D);
    };
    // the pieces of a tile's dq go round the waves (left to the waves without a key alone they hold the others up: 104 us for 75
    // at 32 x 12 heads, 576 rows, 197 keys)
    auto dq_tile = [&](int tile) {
        if (a.dq)
            for (int j = 0; j < NP * SUB; ++j)
                if ((tile * NP * SUB + j) % NW == wave && 32 * (j % NP) < a.D) dq_piece(tile, j / NP, j % NP);
    };
    for (int qt = t0; qt < t1; ++qt) {
        const int pair = qt & 1;
        T* img = lds + pair * 2 * IMG;
        const float* rs = rows + pair * 2 * QT;
        leave_stats(pair);
        wait_loads();
        __syncthreads();
        if (qt + 1 < t1) issue(qt + 1, pair ^ 1);
        if (!NOW && qt > t0) dq_tile(qt - 1);
        if (any_on) {
            // the sub-tiles' products take turns, so that one's chain runs while the other's waits
            f32x16 s[SUB], dp[SUB];
#pragma unroll
            for (int sub = 0; sub < SUB; ++sub)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[sub][e] = dp[sub][e] = 0.f;
#pragma unroll
            for (int c = 0; c < NF; ++c) {
                const bf16x8 k = KL ? row_frag<T, NK>(kimg, key, c, h) : kf[KL ? 0 : c];
#pragma unroll
                for (int sub = 0; sub < SUB; ++sub) {
                    mma(s[sub], row_frag<T, QT>(img, 32 * sub + key_of_row<T>(lane & 31), c, h), k);
                    mma(dp[sub], row_frag<T, QT>(img + IMG, 32 * sub + key_of_row<T>(lane & 31), c, h), vf[c]);
                }
            }
#pragma unroll
            for (int sub = 0; sub < SUB; ++sub) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int q = 32 * sub + key_of<T>(e, h);
                    s[sub][e] = __builtin_amdgcn_exp2f(fmaf(s[sub][e], a.c, -rs[q]));
                    dp[sub][e] = dp[sub][e] - rs[QT + q];             // (ONE: delta follows, a zero stands there)
                }
                if (!all_on) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[sub][e] = on ? s[sub][e] : 0.f;
                }
                if (ONE) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) dp[sub][e] -= half_wave_sum(s[sub][e] * dp[sub][e]);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) dp[sub][e] *= s[sub][e];
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const bf16x8 pf = acc_frag(s[sub], g, T()), df = acc_frag(dp[sub], g, T());
                    *ds_at(pair, sub, 2 * g + h) = df;
#pragma unroll
                    for (int d = 0; d < NP; ++d) {
                        mma(dv[d], col_frag<QT>(img + IMG, 32 * sub + 16 * g, d, lane), pf);
                        mma(dk[d], col_frag<QT>(img, 32 * sub + 16 * g, d, lane), df);
                    }
                    if (ONE) {
                        const bf16x8 pr = rest_frag(s[sub], g, pf), dr = rest_frag(dp[sub], g, df);
                        ds_at(pair, sub, 2 * g + h)[32 * 32 / 8] = dr;
#pragma unroll
                        for (int d = 0; d < NP; ++d) {
                            mma(dv[d], col_frag<QT>(img + IMG, 32 * sub + 16 * g, d, lane), pr);
                            mma(dk[d], col_frag<QT>(img, 32 * sub + 16 * g, d, lane), dr);
                        }
                    }
                }
            }
        }
        if (NOW) {
            __syncthreads();
            dq_tile(qt);
        }
    }
    if (!NOW && t0 < t1) {
        __syncthreads();
        dq_tile(t1 - 1);
    }
    if (!a.dk) return;
    const bool in = key < a.Nk;
    if (!on) {                                            // a masked key's lane worked on zeros: its gradients are zero
#pragma unroll
        for (int d = 0; d < NP; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) dk[d][e] = dv[d][e] = 0.f;
    }
    const long long row = (((long long)b * a.Nk + key) * a.Hk + hk) * a.D;
    if (!shared || a.splits == 1) {
        store_acc<T, true, DP>(in ? (T*)a.dk + row : nullptr, dk, a.scale, h, a.D);
        store_acc<T, true, DP>(in ? (T*)a.dv + row : nullptr, dv, 1.f, h, a.D);
    } else {                                              // [problem][split][dk, dv][Nk][D]
        float* slot = a.part_kv + ((((long long)sh * a.splits + split) * 2) * a.Nk + key) * a.D;
        store_acc<float, true, DP>(in ? slot : nullptr, dk, 1.f, h, a.D);
        store_acc<float, true, DP>(in ? slot + (long long)a.Nk * a.D : nullptr, dv, 1.f, h, a.D);
    }
}

// adds the shares of the problems from a.whole on, in order: a workgroup takes 4096 elements of one problem's dk and dv
template <typename T>
__global__ __launch_bounds__(256) void xattn_short_join_kernel(XaArgs a, int per) {
    const int sh = blockIdx.x / per, piece = blockIdx.x - sh * per, bh = a.whole + sh, b = bh / a.Hk, hk = bh - b * a.Hk;
    const long long n = 2ll * a.Nk * a.D;
    const float* p = a.part_kv + (long long)sh * a.splits * n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long e = piece * 4096ll + (i * 256 + threadIdx.x) * 4;      // D is a multiple of 8: four elements of a row
        if (e >= n) break;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < a.splits; k0 += 4) {
            f32x4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (k0 + k < a.splits) v[k] = *reinterpret_cast<const f32x4*>(p + (k0 + k) * n + e);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int q = 0; q < 4; ++q) s[q] += v[k][q];
        }
        const bool second = e >= n / 2;
        const int r = (int)(second ? e - n / 2 : e), key = r / a.D, d = r - key * a.D;
        const float f = second ? 1.f : a.scale;
        store4<T, true>((T*)(second ? a.dv : a.dk) + (((long long)b * a.Nk + key) * a.Hk + hk) * a.D, d, a.D, s[0] * f, s[1] * f, s[2] * f,
                        s[3] * f);
    }
}


// How the dk / dv launch cuts its work: a unit is one row tile against one live tile of 128 keys.  Streamed, every workgroup
// takes an equal share of the units in a row (shares.h), because whole key tiles, of which there may be a few more than the
// chip holds at once, would leave it idle for up to half the time.  Lengths per sample are only known here, so each wave
// counts the live tiles itself (64 samples a step).
__device__ __forceinline__ int lanes_scan(int v, int lane) {     // inclusive sums over the lanes
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    return v;
}
__device__ __forceinline__ int live_tiles(const XaArgs& a, int b) { return (keys_of(a, b) + 127) >> 7; }
__device__ __forceinline__ Shares stream_of(const XaArgs& a, int grid, int row_tiles, int lane) {
    long long tiles = 0;
    if (!a.kv_len) {
        tiles = (long long)a.B * a.tiles;
    } else {
        for (int b0 = 0; b0 < a.B; b0 += 64)
            tiles += __shfl(lanes_scan(b0 + lane < a.B ? live_tiles(a, b0 + lane) : 0, lane), 63, 64);
    }
    return shares_of(uniform(tiles * a.Hk), grid, row_tiles);
}
// sample, key head and key tile of live tile tau (samples in order, then heads, then tiles)
__device__ __forceinline__ void stream_tile(const XaArgs& a, long long tau, int lane, int& b, int& hk, int& kt) {
    if (!a.kv_len) {
        kt = (int)(tau % a.tiles);
        hk = (int)(tau / a.tiles % a.Hk);
        b = (int)(tau / a.tiles / a.Hk);
        return;
    }
    long long base = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int v = b0 + lane < a.B ? live_tiles(a, b0 + lane) : 0;
        const int inc = lanes_scan(v, lane);
        const long long tot = __shfl(inc, 63, 64);
        if (tau < (base + tot) * a.Hk) {
            // the first sample whose tiles reach beyond tau
            const int l = __ffsll(__ballot((base + inc) * a.Hk > tau)) - 1;
            const int vt = __shfl(v, l, 64);
            const int rest = (int)(tau - (base + __shfl(inc, l, 64) - vt) * a.Hk);
            b = b0 + l;
            hk = rest / vt;
            kt = rest - hk * vt;
            return;
        }
        base += tot;
    }
    b = hk = kt = 0;
}
// first live tile of (b, hk)
__device__ __forceinline__ long long stream_first(const XaArgs& a, int b, int hk, int lane) {
    if (!a.kv_len) return ((long long)b * a.Hk + hk) * a.tiles;
    long long base = 0;
    for (int b0 = 0; b0 <= b; b0 += 64)
        base += __shfl(lanes_scan(b0 + lane < b ? live_tiles(a, b0 + lane) : 0, lane), 63, 64);
    return base * a.Hk + (long long)hk * live_tiles(a, b);
}

// dk and dv: four waves of 32 keys over the row tiles of the whole group.  At bf16 heads beyond 96 the accumulators and both
// operands would take more than the 256 registers that two waves a SIMD have: V then stays in LDS and the row tiles are
// half as long (the long shape above: 636 us, 655 with part of it in scratch memory).
template <typename T, int DP, bool VEC> constexpr bool v_in_lds() { return sizeof(T) == 2 && DP == 128 && VEC; }
template <typename T, int DP, bool VEC> constexpr int row_tile() { return v_in_lds<T, DP, VEC>() ? 32 : Mx<T>::KT; }
template <typename T, int DP, bool VEC, bool STREAM>
__global__ __launch_bounds__(XA_THREADS, sizeof(T) == 4 || !VEC ? 1 : 2) void xattn_dkv_kernel(XaArgs a) {
    constexpr int QT = row_tile<T, DP, VEC>(), IMG = QT * DP, NF = DP / Mx<T>::KD;
    constexpr bool VL = v_in_lds<T, DP, VEC>();
    extern __shared__ __align__(16) char xa_lds[];
    T* const lds = reinterpret_cast<T*>(xa_lds);                           // Q, dO, Q, dO
    T* const vimg = lds + 4 * IMG;
    float* const rows = reinterpret_cast<float*>(vimg + (VL ? 128 * DP : 0));   // [2][lse, delta][QT]
    const int t = threadIdx.x, lane = t & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int blk = xa_block(), RT = (a.R + QT - 1) / QT;
    long long u = 0, u1 = 1;                              // not streamed: one key tile a workgroup
    Shares str = {};
    if (STREAM) {
        str = stream_of(a, gridDim.x, RT, lane);
        if (blk >= str.nb) return;
        u = str.begin(blk);
        u1 = str.begin(blk + 1);
    }
    int turn = 0;                                         // which of the two image pairs is next
    for (int part = 0; u < u1; ++part) {
        int b, hk, kt, t0 = 0, t1 = RT;
        if (STREAM) {
            const Share now = str.piece(u, u1);
            t0 = now.t0;
            t1 = now.t1;
            u += t1 - t0;
            stream_tile(a, now.tile, lane, b, hk, kt);
            b = __builtin_amdgcn_readfirstlane(b);
            hk = __builtin_amdgcn_readfirstlane(hk);
            kt = __builtin_amdgcn_readfirstlane(kt);
        } else {
            kt = blk % a.tiles;
            hk = blk / a.tiles % a.Hk;
            b = blk / a.tiles / a.Hk;
            u = u1;
        }
        const int key = kt * 128 + wave * 32 + (lane & 31);
        const int n = keys_of_wave(a, b);
        const bool on = key < n && (!a.key_mask || a.key_mask[b * a.mask_stride + key] != 0);
        typename Mx<T>::frag kf[NF], vf[VL ? 1 : NF];
        {
            const T* kp = (const T*)a.k + b * a.ks[0] + key * a.ks[1] + hk * a.ks[2];
            const T* vp = (const T*)a.v + b * a.vs[0] + key * a.vs[1] + hk * a.vs[2];
#pragma unroll
            for (int c = 0; c < NF; ++c) {
                const int d = c * Mx<T>::KD + h * Mx<T>::FE;
                kf[c] = on ? global_piece<T, VEC>(kp, d, a.D) : zero_frag<T>();
                if (!VL) vf[VL ? 0 : c] = on ? global_piece<T, VEC>(vp, d, a.D) : zero_frag<T>();
            }
        }
        f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) dk[d][e] = dv[d][e] = 0.f;
        const T* qp = (const T*)a.q + b * a.qs[0] + (long long)hk * a.G * a.qs[2];
        const T* gp = (const T*)a.dout + b * a.dos[0] + (long long)hk * a.G * a.dos[2];
        const long long sti = ((long long)b * a.Hk + hk) * a.R;
        Stage<T, DP, VEC, QT, XA_THREADS, VEC> st;
        st.init(a.qs[1], a.dos[1], a.D, t);
        float stat = 0.f;                                 // threads 0..QT-1: lse, QT..2QT-1: delta
        auto fetch = [&](int tile, int pair) {
            T* img = lds + pair * 2 * IMG;
            st.fetch_rows(qp, a.qs, gp, a.dos, tile * QT, a.R, a.Nq, img, img + IMG, a.D, t, tile > t0 + 1);
            if (t < 2 * QT) {
                const int r = tile * QT + (t < QT ? t : t - QT);
                stat = t < QT ? INFINITY : 0.f;
                if (r < a.R) stat = t < QT ? a.lse[sti + r] : a.delta[sti + r];
            }
        };
        const bool work = __syncthreads_or(on);           // also: every wave has left the images of the part before
        if (work) {
            if (VL) {                                     // a wave loads the rows that it reads itself
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int vr = wave * 32 + 16 * i + (lane >> 2), vk = kt * 128 + vr;
                    const bool ok = vk < n && (!a.key_mask || a.key_mask[b * a.mask_stride + vk] != 0);
                    const T* vp = (const T*)a.v + b * a.vs[0] + vk * a.vs[1] + hk * a.vs[2];
#pragma unroll
                    for (int p = 0; p < DP / 32; ++p) {
                        const int d = 32 * p + ((lane & 3) ^ swz<T>(vr)) * Mx<T>::FE;
                        load_to_lds(ok && d < a.D ? (const void*)(vp + d) : (const void*)xa_zero16, lds_addr(vimg + (p * 128 + wave * 32 + 16 * i) * 32));
                    }
                }
            }
            fetch(t0, turn);
            for (int qt = t0; qt < t1; ++qt, turn ^= 1) {
                T* img = lds + turn * 2 * IMG;
                float* rs = rows + turn * 2 * QT;
                st.store(img, img + IMG, t);
                if (t < 2 * QT) rs[t] = stat;
                wait_loads();
                __syncthreads();
                if (qt + 1 < t1) fetch(qt + 1, turn ^ 1);
#pragma unroll
                for (int qb = 0; qb < QT / 32; ++qb) {
                    if (qb > 0 && qt * QT + 32 * qb >= a.R) continue;
                    f32x16 s, dp;
                    scores<T, DP, QT>(s, img, 32 * qb, kf, lane);
                    if constexpr (VL) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) dp[e] = 0.f;
#pragma unroll
                        for (int c = 0; c < NF; ++c)
                            mma(dp, row_frag<T, QT>(img + IMG, 32 * qb + key_of_row<T>(lane & 31), c, h),
                                row_frag<T, 128>(vimg, wave * 32 + (lane & 31), c, h));
                    } else {
                        scores<T, DP, QT>(dp, img + IMG, 32 * qb, vf, lane);
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int q = 32 * qb + key_of<T>(e, h);
                        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.c, -rs[q]));
                        dp[e] = s[e] * (dp[e] - rs[QT + q]);
                    }
#pragma unroll
                    for (int g = 0; g < 32 / Mx<T>::KD; ++g) {
                        const typename Mx<T>::frag pf = acc_frag(s, g, T()), df = acc_frag(dp, g, T());
#pragma unroll
                        for (int d = 0; d < DP / 32; ++d) {
                            mma(dv[d], col_frag<QT>(img + IMG, 32 * qb + g * Mx<T>::KD, d, lane), pf);
                            mma(dk[d], col_frag<QT>(img, 32 * qb + g * Mx<T>::KD, d, lane), df);
                        }
                    }
                }
            }
        }
        const bool in = key < a.Nk;
        if (!on) {                                        // a masked key's lane worked on zeros: its gradients are zero
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) dk[d][e] = dv[d][e] = 0.f;
        }
        if (!STREAM || (t0 == 0 && t1 == RT)) {
            const long long row = (((long long)b * a.Nk + key) * a.Hk + hk) * a.D;
            store_acc<T, VEC, DP>(in ? (T*)a.dk + row : nullptr, dk, a.scale, h, a.D);
            store_acc<T, VEC, DP>(in ? (T*)a.dv + row : nullptr, dv, 1.f, h, a.D);
        } else {                                          // a workgroup's first and its last part may be shares of a tile
            float* slot = a.part_kv + (Shares::slot(blk, part) * 2 * 128 + wave * 32 + (lane & 31)) * a.D;
            store_acc<float, VEC, DP>(in ? slot : nullptr, dk, 1.f, h, a.D);
            store_acc<float, VEC, DP>(in ? slot + 128ll * a.D : nullptr, dv, 1.f, h, a.D);
        }
    }
}

// adds the shares of the key tiles that several workgroups of a streamed dk / dv launch worked on, in workgroup order, and clears
// the rows of tiles without a live key; 8 keys a workgroup, four shares' loads in flight
template <typename T>
__global__ __launch_bounds__(256) void xattn_dkv_join_kernel(XaArgs a, int grid, int row_tiles) {
    const int lane = threadIdx.x & 63;
    int idx = blockIdx.x >> 4;
    const int kt = idx % a.tiles;
    idx /= a.tiles;
    const int hk = idx % a.Hk, b = idx / a.Hk;
    const int k0 = kt * 128 + (blockIdx.x & 15) * 8;
    if (k0 >= a.Nk) return;
    const int keys = a.Nk - k0 < 8 ? a.Nk - k0 : 8;
    const bool live = kt < live_tiles(a, b);
    int i0 = 0, i1 = -1, part0 = 0;
    if (live) {
        const Shares str = stream_of(a, grid, row_tiles, lane);
        const long long x0 = (stream_first(a, b, hk, lane) + kt) * row_tiles;
        i0 = str.owner(x0);
        i1 = str.owner(x0 + row_tiles - 1);
        if (i0 == i1) return;                             // written in full by one workgroup
        part0 = str.part_of(i0, x0);
    }
    const bool v4 = a.D % 4 == 0;
    const int w = v4 ? 4 : 1, per = a.D / w;
    for (int j = threadIdx.x; j < 2 * keys * per; j += 256) {
        const int m = j / (keys * per), e = j - m * keys * per, key = e / per, d = (e - key * per) * w;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        for (int i = i0; i <= i1; i += 4) {
            float v[4][4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float* p = a.part_kv + ((Shares::slot(i + c, i + c == i0 ? part0 : 0) * 2 + m) * 128 + (blockIdx.x & 15) * 8 + key) * a.D + d;
#pragma unroll
                for (int q = 0; q < 4; ++q) v[c][q] = 0.f;
                if (i + c <= i1) {
                    if (v4) *reinterpret_cast<f32x4*>(v[c]) = *reinterpret_cast<const f32x4*>(p);
                    else v[c][0] = p[0];
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int q = 0; q < 4; ++q) s[q] += v[c][q];
        }
        const float f = m == 0 ? a.scale : 1.f;
        T* o = (T*)(m == 0 ? a.dk : a.dv) + (((long long)b * a.Nk + k0 + key) * a.Hk + hk) * a.D + d;
        for (int q = 0; q < w; ++q) o[q] = from_f32<T>(s[q] * f);
    }
}

// o[i] = f * sum over the splits, in split order
template <typename T>
__global__ __launch_bounds__(256) void xattn_sum_kernel(const float* p, T* o, float f, long long n, int splits) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float s = 0.f;
        for (int k0 = 0; k0 < splits; k0 += 8) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k0 + k < splits ? p[(k0 + k) * n + i] : 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) s += v[k];
        }
        o[i] = from_f32<T>(s * f);
    }
}

// ---------------------------------------------------------------------------------------------- host
constexpr int XA_MAX_D = 128;
constexpr long long XA_MAX_ROWS = (1ll << 31) - 256, XA_MAX_KEYS = (1ll << 31) - 4096;   // row and key indices are ints, up to 12 key tiles ahead

int xa_check(const char* who, const vitmi_xattn_args* g) {
    VITMI_CHECK_ARG(g, "%s: null arguments", who);
    VITMI_CHECK_ARG(g->dt == VITMI_F32 || g->dt == VITMI_BF16, "%s: bad dtype %d", who, g->dt);
    VITMI_CHECK_ARG(g->B >= 0 && g->Nq >= 0 && g->Nk >= 0 && g->Hq > 0 && g->Hk > 0 && g->D > 0,
                    "%s: bad shape B=%d Nq=%d Nk=%d Hq=%d Hk=%d D=%d", who, g->B, g->Nq, g->Nk, g->Hq, g->Hk, g->D);
    VITMI_CHECK_ARG(g->Hq % g->Hk == 0, "%s: %d query heads do not share %d key heads evenly", who, g->Hq, g->Hk);
    VITMI_CHECK_ARG(g->scale > 0.f && g->scale < INFINITY, "%s: the scale must be positive and finite", who);
    VITMI_CHECK_ARG(!(g->kv_len && g->key_mask), "%s: key lengths and a key mask exclude each other", who);
    if (g->D > XA_MAX_D) {
        vitmi_set_error("%s: heads of %d exceed the supported width %d", who, g->D, XA_MAX_D);
        return VITMI_ERR_UNSUPPORTED;
    }
    VITMI_CHECK_ARG((long long)(g->Hq / g->Hk) * g->Nq < XA_MAX_ROWS && (long long)g->Nk < XA_MAX_KEYS, "%s: lengths beyond one call", who);
    for (int i = 0; i < 3; ++i)
        VITMI_CHECK_ARG(g->qs[i] >= 0 && g->ks[i] >= 0 && g->vs[i] >= 0 && (!g->dout || g->dos[i] >= 0), "%s: negative strides", who);
    return VITMI_OK;
}

bool xa_vec(const vitmi_xattn_args* g) {
    const int fe = g->dt == VITMI_F32 ? 4 : 8;
    if (g->D % fe) return false;
    for (const void* p : {g->q, g->k, g->v, (const void*)g->o, g->dout, (const void*)g->dq, (const void*)g->dk, (const void*)g->dv})
        if (reinterpret_cast<uintptr_t>(p) & 15) return false;
    for (int i = 0; i < 3; ++i)
        if (g->qs[i] % fe || g->ks[i] % fe || g->vs[i] % fe || (g->dout && g->dos[i] % fe)) return false;
    return true;
}

int xa_width(int D, bool vec) { return !vec ? 128 : D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

struct XaPlan {
    bool few;
    int fwd_tiles, fwd_splits, dq_tiles, dq_splits, dkv_tiles, dkv_rt, dkv_grid, short_splits, short_whole;
};

int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }

// Splits of the key loop of the few-row kernel, `steps` tiles of 32 keys, which only memory bounds: none while the launch fills
// the chip twice over, else enough for that, each with eight tiles or more
int xa_few_splits(long long blocks, int steps) {
    if (blocks >= 512 || steps < 16) return 1;
    return (int)std::max<long long>(1, std::min<long long>({(512 + blocks - 1) / blocks, steps / 8, 64}));
}

// Splits of the key loop of the row kernels: the number with the shortest estimated time, in microseconds -- rounds of
// workgroups (two a compute unit share it in bf16, fp32 products leave nothing over beside one) times tiles a split, and
// for more than one split the joining launch with the partial rows' way to memory and back.  8 x 6 heads of 64 fp32, 333 rows,
// 257 keys: one split takes 32 us, two with their join 42.
int xa_splits(int dt, long long blocks, int steps, long long rows, int D) {
    const double tile = dt == VITMI_F32 ? D / 32.0 : 0.5 + D / 160.0, slots = dt == VITMI_F32 ? 256 : 512;
    if (blocks >= 4 * slots) return 1;
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 64 && (s == 1 || steps / s >= 2); ++s) {
        const double rounds = (double)(long long)((blocks * s + slots - 1) / slots);
        const double t = rounds * tile * (cdiv(steps, s) + 2) + (s > 1 ? 4 + s * (double)rows * D * 8 / 3e6 : 0);
        if (t < least) {
            least = t;
            best = s;
        }
    }
    return best;
}

XaPlan xa_plan(int dt, int B, int Nq, int Nk, int Hq, int Hk, int D, bool vec) {
    XaPlan p;
    const int R = Hq / Hk * Nq, KT = dt == VITMI_F32 ? 32 : 64;
    const long long bh = (long long)B * Hk;
    // also fp32 launches that would leave most matrix pipes without a wave, while all their tiles of 32 rows are at work at once: two
    // workgroups of this form fit a compute unit at heads up to 64, one at wider ones (LDS).  By tiles of 32 rows / of 128, us:
    // heads of 64, 257 keys, 128 tiles 15 / 18, 384 21 / 29, 512 21 / 29, 520 33 / 29; 100 keys, 512 tiles 12 / 16; 480 keys, 260 tiles
    // 28 / 27, 512 30 / 37; 512 keys (two splits) 384 tiles 36 / 35.  Heads of 128, 257 keys, 256 tiles 26 / 30, 260 48 / 31; 384
    // keys, 64 tiles 25 / 21, 256 27 / 30; 480 keys, 64 tiles 30 / 25.
    p.few = R <= 64 || (dt == VITMI_F32 && (D <= 64 ? bh * cdiv(R, 32) <= 512 && Nk <= 480 : bh * cdiv(R, 32) <= 256 && Nk <= 384));
    p.fwd_tiles = cdiv(R, p.few ? 32 : 128);
    const long long rows = bh * R;
    p.fwd_splits = p.few ? xa_few_splits(bh * p.fwd_tiles, cdiv(Nk, 32)) : xa_splits(dt, bh * p.fwd_tiles, cdiv(Nk, KT), rows, D);
    // all keys in one workgroup (bf16; two of four waves a compute unit, one of eight): the problems of a last round that would
    // leave half of the chip or more idle share their rows, eight tiles of 32 each
    p.short_splits = p.short_whole = 0;
    if (dt == VITMI_BF16 && vec && Nk <= 256) {
        const long long slots = Nk > 128 ? 256 : 512, rest = bh % slots;
        p.short_splits = rest == 0 ? 1 : (int)std::max<long long>(1, std::min<long long>({slots / rest, cdiv(R, 32) / 8, 64}));
        p.short_whole = (int)(p.short_splits > 1 ? bh - rest : bh);
    }
    p.dq_tiles = cdiv(R, 128);
    p.dq_splits = xa_splits(dt, bh * p.dq_tiles, cdiv(Nk, KT), rows, D);
    // dk / dv: a workgroup a key tile where that keeps nine tenths of the chip busy to the end (registers allow three a compute
    // unit in bf16 with heads up to 64, else two; fp32 products leave nothing over beside one), otherwise equal shares, of four row tiles or more
    p.dkv_tiles = cdiv(Nk, 128);
    p.dkv_rt = cdiv(R, dt == VITMI_BF16 && D > 96 && vec ? row_tile<bf16_t, 128, true>() : KT);
    const long long tiles = bh * p.dkv_tiles, slots = 256 * (dt == VITMI_F32 ? 1 : D <= 64 ? 3 : 2);
    const bool even = 10 * tiles >= 9 * slots * ((tiles + slots - 1) / slots);
    const long long grid = std::min<long long>(dt == VITMI_F32 ? slots : 512, tiles * p.dkv_rt / 4);
    p.dkv_grid = even || p.dkv_rt < 8 || grid <= tiles / 2 ? 0 : (int)grid;
    return p;
}

long long up256(long long x) { return (x + 255) & ~255ll; }

void xa_fill(const vitmi_xattn_args* g, XaArgs* a) {
    *a = XaArgs{};
    a->q = g->q; a->k = g->k; a->v = g->v; a->o = g->o;
    for (int i = 0; i < 3; ++i) {
        a->qs[i] = g->qs[i];
        a->ks[i] = g->ks[i];
        a->vs[i] = g->vs[i];
        a->dos[i] = g->dos[i];
    }
    a->kv_len = g->kv_len;
    a->len64 = g->kv_len_i64;
    a->key_mask = (const unsigned char*)g->key_mask;
    a->mask_stride = g->mask_stride;
    a->lse = g->lse;
    a->Nq = g->Nq; a->Nk = g->Nk; a->Hq = g->Hq; a->Hk = g->Hk; a->D = g->D;
    a->G = g->Hq / g->Hk;
    a->R = a->G * g->Nq;
    a->scale = g->scale;
    a->c = g->scale * XA_LOG2E;
    a->dout = g->dout;
    a->dq = g->dq; a->dk = g->dk; a->dv = g->dv;
    a->n_q = (long long)g->B * g->Nq * g->Hq * g->D;
    a->B = g->B;
}

// more than 64 KB of LDS a workgroup is asked for once per kernel and device (a bit of *done each)
int xa_need_lds(const void* fn, size_t lds, std::atomic<unsigned long long>* done) {
    if (lds <= 64 * 1024) return VITMI_OK;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (e == hipSuccess && (dev > 63 || !(done->load() & bit))) {
        e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e == hipSuccess && dev <= 63) done->fetch_or(bit);
    }
    return e == hipSuccess ? VITMI_OK : vitmi_hip_fail(e, "vitmi_cross_attn: LDS size");
}

enum { XK_FWD, XK_FEW, XK_DQ, XK_DKV, XK_DKV_STREAM };

template <typename T, int DP, bool VEC>
int xa_launch(int kind, const XaArgs& a, long long blocks, hipStream_t s) {
    constexpr size_t tile4 = 4ull * Mx<T>::KT * DP * sizeof(T);
    constexpr size_t few = std::max<size_t>(8ull * 32 * DP * sizeof(T), (4ull * DP * 32 + 256) * sizeof(float));
    constexpr size_t dkv = (4ull * row_tile<T, DP, VEC>() + (v_in_lds<T, DP, VEC>() ? 128 : 0)) * DP * sizeof(T) + 4ull * row_tile<T, DP, VEC>() * sizeof(float);
    const size_t lds = kind == XK_FEW ? few : kind >= XK_DKV ? dkv : tile4;
    const void* fn = kind == XK_FWD   ? (const void*)&xattn_fwd_kernel<T, DP, VEC>
                     : kind == XK_FEW ? (const void*)&xattn_few_kernel<T, DP, VEC>
                     : kind == XK_DQ  ? (const void*)&xattn_dq_kernel<T, DP, VEC>
                     : kind == XK_DKV ? (const void*)&xattn_dkv_kernel<T, DP, VEC, false>
                                      : (const void*)&xattn_dkv_kernel<T, DP, VEC, true>;
    static std::atomic<unsigned long long> done[XK_DKV_STREAM + 1];
    if (int rc = xa_need_lds(fn, lds, &done[kind])) return rc;
    VITMI_CHECK_ARG(blocks < (1ll << 32) / XA_THREADS, "vitmi_cross_attn: %lld tiles are beyond one launch", blocks);
    const dim3 grid((unsigned)blocks), block(XA_THREADS);
    if (kind == XK_FWD) hipLaunchKernelGGL((xattn_fwd_kernel<T, DP, VEC>), grid, block, lds, s, a);
    else if (kind == XK_FEW) hipLaunchKernelGGL((xattn_few_kernel<T, DP, VEC>), grid, block, lds, s, a);
    else if (kind == XK_DQ) hipLaunchKernelGGL((xattn_dq_kernel<T, DP, VEC>), grid, block, lds, s, a);
    else if (kind == XK_DKV) hipLaunchKernelGGL((xattn_dkv_kernel<T, DP, VEC, false>), grid, block, lds, s, a);
    else hipLaunchKernelGGL((xattn_dkv_kernel<T, DP, VEC, true>), grid, block, lds, s, a);
    VITMI_LAUNCH_CHECK("vitmi_cross_attn");
    return VITMI_OK;
}

template <typename T>
int xa_dispatch(int kind, const XaArgs& a, bool vec, long long blocks, hipStream_t s) {
    if (!vec) return xa_launch<T, 128, false>(kind, a, blocks, s);
    switch (xa_width(a.D, true)) {
        case 32: return xa_launch<T, 32, true>(kind, a, blocks, s);
        case 64: return xa_launch<T, 64, true>(kind, a, blocks, s);
        case 96: return xa_launch<T, 96, true>(kind, a, blocks, s);
        default: return xa_launch<T, 128, true>(kind, a, blocks, s);
    }
}

int xa_run(int kind, int dt, const XaArgs& a, bool vec, long long blocks, hipStream_t s) {
    return dt == VITMI_F32 ? xa_dispatch<float>(kind, a, vec, blocks, s) : xa_dispatch<bf16_t>(kind, a, vec, blocks, s);
}

int xa_sum(int dt, const float* p, void* o, float f, long long n, int splits, hipStream_t s) {
    const dim3 grid((unsigned)std::min<long long>(4096, (n + 255) / 256));
    if (dt == VITMI_F32)
        hipLaunchKernelGGL((xattn_sum_kernel<float>), grid, dim3(256), 0, s, p, (float*)o, f, n, splits);
    else
        hipLaunchKernelGGL((xattn_sum_kernel<bf16_t>), grid, dim3(256), 0, s, p, (bf16_t*)o, f, n, splits);
    VITMI_LAUNCH_CHECK("vitmi_cross_attn(sum)");
    return VITMI_OK;
}

template <int DP, int NW, bool ONE = false>
int xa_launch_short(const XaArgs& a, long long blocks, hipStream_t s) {
    // 64 rows a tile where LDS holds them (128 KB beside eight waves of heads up to 64): half the barriers
    constexpr int SUB = NW == 8 && DP <= 64 ? 2 : 1, QT = 32 * SUB;
    constexpr size_t lds = (32ull * NW * DP + 4ull * QT * DP + (DP / 32 * SUB == NW ? 1 : 2) * 32ull * NW * QT) * 2 + 4 * QT * sizeof(float);
    const void* fn = (const void*)&xattn_bwd_short_kernel<DP, NW, SUB, ONE>;
    static std::atomic<unsigned long long> done;
    if (int rc = xa_need_lds(fn, lds, &done)) return rc;
    VITMI_CHECK_ARG(blocks < (1ll << 32) / (64 * NW), "vitmi_cross_attn: %lld problems are beyond one launch", blocks);
    hipLaunchKernelGGL((xattn_bwd_short_kernel<DP, NW, SUB, ONE>), dim3((unsigned)blocks), dim3(64 * NW), lds, s, a);
    VITMI_LAUNCH_CHECK("vitmi_cross_attn(short)");
    return VITMI_OK;
}
int xa_run_short(const XaArgs& a, long long blocks, hipStream_t s) {
    const int w = xa_width(a.D, true);
    if (a.Nk <= 32) {
        if (w == 32) return xa_launch_short<32, 4, true>(a, blocks, s);
        if (w == 64) return xa_launch_short<64, 4, true>(a, blocks, s);
        if (w == 96) return xa_launch_short<96, 4, true>(a, blocks, s);
        return xa_launch_short<128, 4, true>(a, blocks, s);
    }
    if (a.Nk <= 128) {
        if (w == 32) return xa_launch_short<32, 4>(a, blocks, s);
        if (w == 64) return xa_launch_short<64, 4>(a, blocks, s);
        if (w == 96) return xa_launch_short<96, 4>(a, blocks, s);
        return xa_launch_short<128, 4>(a, blocks, s);
    }
    if (w == 32) return xa_launch_short<32, 8>(a, blocks, s);
    if (w == 64) return xa_launch_short<64, 8>(a, blocks, s);
    if (w == 96) return xa_launch_short<96, 8>(a, blocks, s);
    return xa_launch_short<128, 8>(a, blocks, s);
}

}  // namespace

extern "C" long long vitmi_cross_attn_fwd_workspace_bytes(int dt, int B, int Nq, int Nk, int Hq, int Hk, int D) {
    if (B <= 0 || Nq <= 0 || Nk <= 0 || Hk <= 0 || Hq <= 0 || D <= 0 || Hq % Hk) return 0;
    if ((long long)(Hq / Hk) * Nq >= XA_MAX_ROWS) return 0;
    const int s = xa_plan(dt, B, Nq, Nk, Hq, Hk, D, true).fwd_splits;
    if (s == 1) return 0;
    const long long rows = (long long)B * Nq * Hq;
    return up256(s * rows * D * 4) + up256(s * rows * 8);
}

extern "C" int vitmi_cross_attn_fwd(const vitmi_xattn_args* g, void* workspace, void* stream) {
    const char* who = "vitmi_cross_attn_fwd";
    if (int rc = xa_check(who, g)) return rc;
    if (g->B == 0 || g->Nq == 0) return VITMI_OK;
    VITMI_CHECK_ARG(g->q && g->o && (g->Nk == 0 || (g->k && g->v)), "%s: null pointer", who);
    const bool vec = xa_vec(g);
    const XaPlan p = xa_plan(g->dt, g->B, g->Nq, g->Nk, g->Hq, g->Hk, g->D, vec);
    VITMI_CHECK_ARG(p.fwd_splits == 1 || workspace, "%s: this shape needs a workspace", who);
    VITMI_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "%s: the workspace must be aligned to 16 bytes", who);
    XaArgs a;
    xa_fill(g, &a);
    const long long rows = (long long)g->B * g->Nq * g->Hq;
    a.tiles = p.fwd_tiles;
    a.splits = p.fwd_splits;
    a.part_o = (float*)workspace;
    a.part_ml = (float*)((char*)workspace + up256((long long)a.splits * rows * g->D * 4));
    hipStream_t s = as_stream(stream);
    ProfScope prof(VITMI_FAM_ATTN_FWD, s, 4.0 * rows * g->Nk * g->D);
    const long long blocks = (long long)g->B * g->Hk * a.tiles * a.splits;
    if (int rc = xa_run(p.few ? XK_FEW : XK_FWD, g->dt, a, vec, blocks, s)) return rc;
    if (a.splits > 1) {
        const dim3 grid((unsigned)((rows + 3) / 4));
        if (g->dt == VITMI_F32)
            hipLaunchKernelGGL((xattn_join_kernel<float>), grid, dim3(256), 0, s, a, rows);
        else
            hipLaunchKernelGGL((xattn_join_kernel<bf16_t>), grid, dim3(256), 0, s, a, rows);
        VITMI_LAUNCH_CHECK(who);
    }
    return VITMI_OK;
}

extern "C" long long vitmi_cross_attn_bwd_workspace_bytes(int dt, int B, int Nq, int Nk, int Hq, int Hk, int D) {
    if (B <= 0 || Nq <= 0 || Nk <= 0 || Hk <= 0 || Hq <= 0 || D <= 0 || Hq % Hk) return 0;
    if ((long long)(Hq / Hk) * Nq >= XA_MAX_ROWS) return 0;
    const long long rows = (long long)B * Nq * Hq;
    long long most = 0;
    for (bool vec : {false, true}) {                      // room for either alignment of the operands
        const XaPlan p = xa_plan(dt, B, Nq, Nk, Hq, Hk, D, vec);
        const long long n = vec && p.short_splits
                                ? ((long long)B * Hk - p.short_whole) * p.short_splits * 2 * Nk * D * 4
                                : up256(rows * 4) + (p.dq_splits > 1 ? up256(p.dq_splits * rows * D * 4) : 0) + (long long)p.dkv_grid * 4 * 128 * D * 4;
        most = std::max(most, n);
    }
    return std::max(most, 256ll);
}

extern "C" int vitmi_cross_attn_bwd(const vitmi_xattn_args* g, void* workspace, void* stream) {
    const char* who = "vitmi_cross_attn_bwd";
    if (int rc = xa_check(who, g)) return rc;
    VITMI_CHECK_ARG(g->B > 0 && g->Nq > 0 && g->Nk > 0, "%s: nothing to differentiate", who);
    VITMI_CHECK_ARG(g->q && g->k && g->v && g->o && g->dout && g->lse && workspace, "%s: null pointer", who);
    VITMI_CHECK_ARG((g->dk == nullptr) == (g->dv == nullptr), "%s: dk and dv come together", who);
    VITMI_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "%s: the workspace must be aligned to 16 bytes", who);
    const bool vec = xa_vec(g);
    const XaPlan p = xa_plan(g->dt, g->B, g->Nq, g->Nk, g->Hq, g->Hk, g->D, vec);
    XaArgs a;
    xa_fill(g, &a);
    const long long rows = (long long)g->B * g->Nq * g->Hq;
    hipStream_t s = as_stream(stream);
    ProfScope prof(VITMI_FAM_ATTN_BWD, s, 10.0 * rows * g->Nk * g->D);
    if (p.short_splits) {
        a.splits = p.short_splits;
        a.whole = p.short_whole;
        a.part_kv = (float*)workspace;
        const long long shared = (long long)g->B * g->Hk - a.whole;
        if (int rc = xa_run_short(a, a.whole + shared * a.splits, s)) return rc;
        if (g->dk && shared > 0) {
            const int per = cdiv(2ll * g->Nk * g->D, 4096);
            hipLaunchKernelGGL((xattn_short_join_kernel<bf16_t>), dim3((unsigned)(shared * per)), dim3(256), 0, s, a, per);
            VITMI_LAUNCH_CHECK(who);
        }
        return VITMI_OK;
    }
    char* w = (char*)workspace;
    a.delta = (float*)w;
    w += up256(rows * 4);
    a.tiles = p.dq_tiles;
    a.splits = g->dq ? p.dq_splits : 1;                   // without dq the launch forms delta alone
    if (a.splits > 1) {
        a.part_dq = (float*)w;
        w += up256(a.splits * a.n_q * 4);
    }
    a.part_kv = (float*)w;
    if (int rc = xa_run(XK_DQ, g->dt, a, vec, (long long)g->B * g->Hk * a.tiles * a.splits, s)) return rc;
    if (g->dq && a.splits > 1)
        if (int rc = xa_sum(g->dt, a.part_dq, g->dq, g->scale, a.n_q, a.splits, s)) return rc;
    if (g->dk) {
        a.tiles = p.dkv_tiles;
        const long long tiles = (long long)g->B * g->Hk * a.tiles;
        if (int rc = xa_run(p.dkv_grid ? XK_DKV_STREAM : XK_DKV, g->dt, a, vec, p.dkv_grid ? p.dkv_grid : tiles, s)) return rc;
        if (p.dkv_grid) {
            const dim3 grid((unsigned)(16 * tiles));
            if (g->dt == VITMI_F32)
                hipLaunchKernelGGL((xattn_dkv_join_kernel<float>), grid, dim3(256), 0, s, a, p.dkv_grid, p.dkv_rt);
            else
                hipLaunchKernelGGL((xattn_dkv_join_kernel<bf16_t>), grid, dim3(256), 0, s, a, p.dkv_grid, p.dkv_rt);
            VITMI_LAUNCH_CHECK(who);
        }
    }
    return VITMI_OK;
}
