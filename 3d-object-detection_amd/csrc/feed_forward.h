// Matrix products of the feed-forward operators (dense, gated) on the gfx950 matrix cores: one tiled kernel for
// fp32, bf16 and fp16 operands in every storage order that the forward and the backward products meet, with the
// operators' epilogues (bias, activation, gate product, residual) on the fp32 accumulators.
//
//   c[m][n] = epilogue( sum over k of a(m,k) b(k,n) )
//
// "a" is the operand whose index m counts output rows, "b" the one whose index n counts output columns.  Each is
// stored either with k contiguous (kInner: a row of memory is one m or n, columns run over k) or with m / n
// contiguous (kOuter: a row of memory is one k).  Forward: a = x (kInner), b = w (kOuter, or kInner where the
// weights are held (out,in)).  dx = dpre w^T: the same two with the weights' order the other way round.
// dw = x^T dpre: both kOuter, k = the rows of the batch.
//
// A workgroup of four waves owns a BM x BN tile; each wave a grid of 32 x 32 MFMA tiles.  The MFMA's A operand is the
// b side (lane = output column), its B operand the a side (lane = output row), so a lane's accumulators run along
// an output ROW, and a pass through LDS turns them into runs of eight columns of consecutive rows: bias, residual and
// result move as 16-byte vectors.
#pragma once
#include <algorithm>
#include <cstdint>

#include "fpn_common.h"

namespace fpn {
namespace ff {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
// 16 bytes at an element's alignment: rows of odd widths start anywhere (global memory takes such accesses whole)
typedef unsigned uintx4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef float floatx4_u __attribute__((ext_vector_type(4), aligned(4)));

enum { kInner = 0, kOuter = 1 };

struct Args {
    long m;                     // output rows
    int n;                      // output columns (of each half where GATED)
    long k;                     // length of one k segment
    int segs;                   // 1, or 2: the sum runs over (a[0],b[0]) and then (a[1],b[1])
    int batch;                  // 1, or 2: separate products a[0] b[i] -> c[i]
    long load_m;                // what may be read of kOuter operands' rows: m and n, or more where rows are padded
    int load_n;
    const void *a[2], *b[2];    // b: [segment], [batch member], or gate and up where GATED
    long lda[2], ldb[2];        // elements between two rows of memory
    const void *bias[2];
    int act;
    const void *residual;
    long ldr;
    void *c[2];
    long ldc;
    bool c_float;               // c is fp32 whatever the operands' type
    float *pre[2];              // pre-activations, for the backward pass (or null)
    long ldp;
    // the gated block's backward epilogue (or null): the sums are dh, from which dg = dh up act'(gate) and du = dh act(gate)
    // go to c[0] and c[1]; `sums` (or null): their column sums, one row of (2, n) per 32 TM output rows
    const float *gate, *up;
    float *sums;
    float *partial;             // split k: (batch, splits, 1 or 2, m, n) sums, joined by join_kernel
    int splits;
    long tiles_per_split;       // k tiles
    long mt;                    // output tiles along m and n
    int nt;
};

template <class T> struct Type;
template <> struct Type<float> {
    static constexpr int kE = 4;            // elements of a 16-byte chunk
    static constexpr int kCode = FPN_F32;
};
template <> struct Type<__bf16> {
    static constexpr int kE = 8;
    static constexpr int kCode = FPN_BF16;
};
template <> struct Type<_Float16> {
    static constexpr int kE = 8;
    static constexpr int kCode = FPN_F16;
};

// ---- activations, on fp32 values -------------------------------------------------------------------------------

// The normal distribution's Phi(v) and, as a by-product, exp(-v^2 / 2), for 16-bit results.  With z = |v| / sqrt 2 and
// t = 1 / (1 + 0.51 z), erfc(z) exp(z^2) is t times a polynomial in t; its seven coefficients were fitted to the
// smallest relative error on 0 <= z <= 10 (1.1e-6 in fp32, a 200th of fp16's half step), so the tail towards
// Phi -> 0 keeps its digits.  A third of the instructions of the library's erfcf, which fp32 results take.
__device__ inline float normal_cdf(float v, float &gauss)
{
    const float z = fabsf(v) * 0.70710678f;
    const float t = __builtin_amdgcn_rcpf(1.f + 0.51f * z);
    const float q = t * (0.287917584f + t * (0.284151107f + t * (0.279072791f + t * (0.0550344735f +
                    t * (0.358472407f + t * (-0.359154463f + t * 0.0945056677f))))));
    gauss = __expf(-z * z);
    const float tail = 0.5f * q * gauss;
    return v < 0.f ? tail : 1.f - tail;
}

template <bool EXACT> __device__ inline float sigmoid(float v)
{
    if (EXACT) return 1.f / (1.f + expf(-v));
    return __builtin_amdgcn_rcpf(1.f + __expf(-v));
}

constexpr float kGeluC = 1.5957691216057308f;      // 2 sqrt(2 / pi): (1 + tanh(z / 2)) / 2 = sigmoid(z)
constexpr float kGeluA = 0.044715f;
constexpr float kRsqrt2 = 0.70710678118654752f, kRsqrt2Pi = 0.39894228040143268f;

// act(v); ACT is a compile-time constant, EXACT the accuracy of an fp32 result
template <int ACT, bool EXACT> __device__ inline float activate(float v)
{
    if (ACT == FPN_ACT_RELU) return v < 0.f ? 0.f : v;                    // (a NaN stays one)
    if (ACT == FPN_ACT_SIGMOID) return sigmoid<EXACT>(v);
    if (ACT == FPN_ACT_SILU) return v * sigmoid<EXACT>(v);
    if (ACT == FPN_ACT_GELU) {
        if (EXACT) return 0.5f * v * erfcf(-v * kRsqrt2);
        float gauss;
        return v * normal_cdf(v, gauss);
    }
    if (ACT == FPN_ACT_GELU_TANH) return v * sigmoid<EXACT>(kGeluC * (v + kGeluA * v * v * v));
    return v;
}

// act(v) and act'(v).  1 - sigmoid(z) is taken as sigmoid(-z) (no cancellation); GELU's products that would be
// 0 * infinity in the far tails are cut off where the derivative is 0 or 1 to all bits.  (SiLU is finite wherever v is; at an
// infinity it is NaN, as its formula.)
template <int ACT, bool EXACT> __device__ inline float activate_grad(float v, float &value)
{
    if (ACT == FPN_ACT_RELU) {
        value = v < 0.f ? 0.f : v;
        return v > 0.f ? 1.f : (v <= 0.f ? 0.f : v);
    }
    if (ACT == FPN_ACT_SIGMOID) {
        value = sigmoid<EXACT>(v);
        return value * sigmoid<EXACT>(-v);
    }
    if (ACT == FPN_ACT_SILU) {
        const float s = sigmoid<EXACT>(v);
        value = v * s;
        return s * (1.f + v * sigmoid<EXACT>(-v));
    }
    if (ACT == FPN_ACT_GELU) {
        const float w = fminf(fabsf(v), 1e4f);                            // (the density is 0 there)
        float gauss, cdf;
        if (EXACT) {
            cdf = 0.5f * erfcf(-v * kRsqrt2);
            gauss = expf(-0.5f * w * w);
        } else {
            cdf = normal_cdf(v, gauss);
        }
        value = v * cdf;
        return cdf + copysignf(w, v) * kRsqrt2Pi * gauss;
    }
    if (ACT == FPN_ACT_GELU_TANH) {
        const float w = fminf(fmaxf(v, -1e4f), 1e4f);                     // (z' grows as v^2; sigmoid(+-z) is 0 there)
        const float z = kGeluC * (w + kGeluA * w * w * w);
        const float s = sigmoid<EXACT>(z);
        value = v * s;
        const float d = s + w * s * sigmoid<EXACT>(-z) * kGeluC * (1.f + 3.f * kGeluA * w * w);
        return v == v ? d : v;
    }
    value = v;
    return 1.f;
}

// f(integral_constant<ACT>) for the run-time activation (a wave-uniform branch around a whole vector's work)
template <int V> struct ActTag { static constexpr int value = V; };
template <class F> __device__ inline void for_activation(int act, F f)
{
    switch (act) {
    case FPN_ACT_RELU: f(ActTag<FPN_ACT_RELU>()); break;
    case FPN_ACT_SIGMOID: f(ActTag<FPN_ACT_SIGMOID>()); break;
    case FPN_ACT_SILU: f(ActTag<FPN_ACT_SILU>()); break;
    case FPN_ACT_GELU: f(ActTag<FPN_ACT_GELU>()); break;
    case FPN_ACT_GELU_TANH: f(ActTag<FPN_ACT_GELU_TANH>()); break;
    default: f(ActTag<FPN_ACT_NONE>()); break;
    }
}

// ---- eight consecutive elements of a row ------------------------------------------------------------------------

// v[i] = p[i] for i < count (<= 8), the rest 0; count >= 8 reads whole vectors
template <class T> __device__ inline void load8(const T *p, long count, float (&v)[8])
{
    if (count >= 8) {
        if constexpr (sizeof(T) == 4) {
            const floatx4_u lo = *reinterpret_cast<const floatx4_u *>(p), hi = *reinterpret_cast<const floatx4_u *>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = lo[i]; v[4 + i] = hi[i]; }
        } else {
            typedef T vec __attribute__((ext_vector_type(8)));
            const uintx4 raw = *reinterpret_cast<const uintx4_u *>(p);
            const vec x = __builtin_bit_cast(vec, raw);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < count ? (float)p[i] : 0.f;
    }
}

// load8 in two steps: the bytes, and what they are
template <class T> struct Raw8 {
    uintx4 v[sizeof(T) / 2];

    __device__ void load(const T *p, long count)
    {
        if (count >= 8) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = *reinterpret_cast<const uintx4_u *>(p + i * (16 / sizeof(T)));
        } else {
            typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
            constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
                vec e;
#pragma unroll
                for (int j = 0; j < E; ++j) e[j] = i * E + j < count ? p[i * E + j] : (T)0.f;
                v[i] = __builtin_bit_cast(uintx4, e);
            }
        }
    }

    __device__ void add_to(float (&sum)[8]) const
    {
        typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const uintx4 raw = v[i];
            const vec e = __builtin_bit_cast(vec, raw);
#pragma unroll
            for (int j = 0; j < E; ++j) sum[i * E + j] += (float)e[j];
        }
    }
};

template <class T> __device__ inline void store8(T *p, long count, const float (&v)[8])
{
    if (count >= 8) {
        if constexpr (sizeof(T) == 4) {
            floatx4_u lo, hi;
#pragma unroll
            for (int i = 0; i < 4; ++i) { lo[i] = v[i]; hi[i] = v[4 + i]; }
            *reinterpret_cast<floatx4_u *>(p) = lo;
            *reinterpret_cast<floatx4_u *>(p + 4) = hi;
        } else {
            typedef T vec __attribute__((ext_vector_type(8)));
            vec x;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (T)v[i];
            *reinterpret_cast<uintx4_u *>(p) = __builtin_bit_cast(uintx4, x);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < count) p[i] = (T)v[i];
    }
}

// The epilogue of eight columns of one output row: v = sums (v2: the up half where GATED)
template <class T, bool GATED>
__device__ inline void finish8(const Args &p, int member, long m, int n, float (&v)[8], float (&v2)[8])
{
    constexpr bool EXACT = sizeof(T) == 4;
    const long left = p.n - n;
    float w[8];
    if (p.bias[GATED ? 0 : member]) {
        load8(reinterpret_cast<const T *>(p.bias[GATED ? 0 : member]) + n, left, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += w[i];
    }
    if (GATED && p.bias[1]) {
        load8(reinterpret_cast<const T *>(p.bias[1]) + n, left, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v2[i] += w[i];
    }
    if (p.pre[0]) {
        // kept in fp32: rounded to 16 bits, gate and up would double the error of dx and dw
        store8(p.pre[0] + m * p.ldp + n, left, v);
        if (GATED) store8(p.pre[1] + m * p.ldp + n, left, v2);
    }
    if (p.act != FPN_ACT_NONE)
        for_activation(p.act, [&](auto tag) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = activate<decltype(tag)::value, EXACT>(v[i]);
        });
    if (GATED) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= v2[i];
    }
    if (p.residual) {
        load8(reinterpret_cast<const T *>(p.residual) + m * p.ldr + n, left, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += w[i];
    }
    if (p.c_float) store8(reinterpret_cast<float *>(p.c[member]) + m * p.ldc + n, left, v);
    else store8(reinterpret_cast<T *>(p.c[member]) + m * p.ldc + n, left, v);
}

// ---- tiles ------------------------------------------------------------------------------------------------------

constexpr int kThreads = 256;
constexpr int kTileBytes = 128;          // of k in one LDS tile: 64 sixteen-bit elements or 32 floats

__device__ inline uintx4 shift_right(uintx4 v, int bits)       // the 128-bit number v >> bits, zeros from the top
{
    unsigned long long lo = (unsigned long long)v[1] << 32 | v[0], hi = (unsigned long long)v[3] << 32 | v[2];
    if (bits >= 128) { lo = 0; hi = 0; }
    else if (bits >= 64) { lo = hi >> (bits - 64); hi = 0; }
    else if (bits > 0) { lo = lo >> bits | hi << (64 - bits); hi >>= bits; }
    uintx4 r;
    r[0] = (unsigned)lo; r[1] = (unsigned)(lo >> 32); r[2] = (unsigned)hi; r[3] = (unsigned)(hi >> 32);
    return r;
}

// One operand's tile: R rows (m or n) x kTileBytes of k.  Memory -> registers (`load`) -> LDS (`put`) -> MFMA
// operands (`frag`).
//
// LDS image, kInner: row r at 128 r, its eight 16-byte chunks permuted by (r ^ r >> 3 & 1) & 7, so that the sixteen
// rows that a ds_read_b128 touches at once fall on different banks.  kOuter: row k at k R sizeof(T); 16-bit elements
// in 32-byte units permuted by 2 (k & 1) ^ 5 (k >> 1 & 1), so that the four k rows and two units that
// ds_read_b64_tr_b16 gathers fall on different banks; floats with 128-byte units exchanged by k >> 2 & 1, since a
// wave's halves read rows k and k + 4.
//
// Ends: rows beyond the last repeat it (their results are never stored).  Along the contiguous direction a chunk
// that would pass the end is read from the last 16 bytes inside and shifted into place, which also puts zeros
// behind the end: no access leaves the operand, whatever its width and alignment.  Operands under one chunk wide are read
// element by element.
template <class T, int ORDER, int R> struct Tile {
    static constexpr int E = Type<T>::kE;
    static constexpr int BK = kTileBytes / (int)sizeof(T);
    static constexpr int kChunks = R * 8 / kThreads;
    static constexpr int kPerRow = R / E;                     // kOuter: chunks of a memory row
    static constexpr int kRowBytes = R * (int)sizeof(T);      // kOuter

    const char *base;        // uniform: the tile's first element of the current k tile
    long ld;
    long k;                  // of the segment
    long outer;              // rows or columns from this tile's first to the operand's end
    bool narrow;             // the operand is under one chunk wide
    unsigned off[kChunks];   // byte offsets of this thread's chunks in an inner k tile
    unsigned put_at[kChunks];
    int pos;                 // kInner: first k of this thread's chunks; kOuter: its first m / n
    int shift;               // elements that the last loaded tile's chunks move by
    unsigned zero;           // bit i: chunk i of the last loaded tile lies behind the last k
    uintx4 reg[kChunks];

    __device__ void init(long outer_left, long all, long k_, int tid)
    {
        outer = outer_left;
        narrow = (ORDER == kInner ? k_ : all) < E;
        shift = 0;
        zero = 0;
        if (ORDER == kInner) {
            pos = (tid & 7) * E;
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int r = (tid >> 3) + i * (kThreads / 8);
                put_at[i] = r * 128 + ((((tid & 7) ^ swizzle(r)) & 7) << 4);
            }
        } else {
            pos = (tid % kPerRow) * E;
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int kk = tid / kPerRow + i * (kThreads / kPerRow);
                put_at[i] = outer_at(kk, pos);
            }
        }
    }

    // (kInner: of row r) (kOuter: of row k)
    __device__ static int swizzle(int r) { return (r ^ (r >> 3 & 1)) & 7; }
    __device__ static unsigned outer_at(int kk, int n)
    {
        if (sizeof(T) == 2) {
            const int g = (((kk & 1) << 1) ^ ((kk >> 1 & 1) * 5)) & (R / 16 - 1);
            return kk * kRowBytes + (((n >> 4) ^ g) << 5) + (n & 15) * 2;
        }
        return kk * kRowBytes + ((n ^ (R > 32 ? (kk >> 2 & 1) << 5 : 0)) << 2);
    }

    // a new segment: where its memory is, and this thread's offsets
    __device__ void segment(const void *p, long ld_, long first, long k_, int tid)
    {
        ld = ld_;
        k = k_;
        base = reinterpret_cast<const char *>(p) + (ORDER == kInner ? first * ld : first) * (long)sizeof(T);
        if (ORDER == kInner) {
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const long r = min((long)((tid >> 3) + i * (kThreads / 8)), outer - 1);
                off[i] = (unsigned)(r * ld * (long)sizeof(T)) + (tid & 7) * 16;
            }
        } else {
            // (a tile that keeps less than a chunk starts reading that much before its own first column)
            const long before = narrow ? 0 : max(E - outer, 0l), n = min((long)pos, max(outer - E, -before));
            shift = (int)(pos - n);
            base -= before * (long)sizeof(T);
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
                off[i] = (unsigned)(((tid / kPerRow + i * (kThreads / kPerRow)) * ld + n + before) * (long)sizeof(T));
        }
    }

    // requests k tile kt of the segment
    __device__ void load(long kt, int tid)
    {
        const long k0 = kt * BK;
        const char *at = base + (ORDER == kInner ? k0 : k0 * ld) * (long)sizeof(T);
        const bool tail = k0 + BK > k;
        if (narrow) {
            load_elements(at, k - k0, tid);
            return;
        }
        if (ORDER == kInner) {
            int back = 0;
            shift = 0;
            if (tail) {
                back = (int)(k0 + pos - min(k0 + pos, k - E));
                shift = back;
            }
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
                reg[i] = *reinterpret_cast<const uintx4_u *>(at + ((long)off[i] - back * (int)sizeof(T)));
        } else {
            zero = 0;
            if (!tail) {
#pragma unroll
                for (int i = 0; i < kChunks; ++i) reg[i] = *reinterpret_cast<const uintx4_u *>(at + off[i]);
            } else {
                const int last = (int)(k - k0) - 1;
#pragma unroll
                for (int i = 0; i < kChunks; ++i) {
                    const int kk = tid / kPerRow + i * (kThreads / kPerRow);
                    if (kk > last) zero |= 1u << i;
                    reg[i] = *reinterpret_cast<const uintx4_u *>(at + (long)off[i] - (long)max(kk - last, 0) * ld * (long)sizeof(T));
                }
            }
        }
    }

    __device__ void load_elements(const char *at, long kleft, int tid)
    {
        shift = 0;
        zero = 0;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            typedef T vec __attribute__((ext_vector_type(E)));
            vec e;
            const long row = ORDER == kInner ? min((long)((tid >> 3) + i * (kThreads / 8)), outer - 1)
                                             : min((long)(tid / kPerRow + i * (kThreads / kPerRow)), kleft - 1);
            const bool row_in = ORDER == kInner || tid / kPerRow + i * (kThreads / kPerRow) < kleft;
            const long inside = ORDER == kInner ? kleft : outer;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const T got = reinterpret_cast<const T *>(at)[row * ld + min((long)pos + j, inside - 1)];
                e[j] = row_in && pos + j < inside ? got : (T)0.f;
            }
            reg[i] = __builtin_bit_cast(uintx4, e);
        }
    }

    __device__ void put(char *lds)
    {
        if (ORDER == kInner ? __builtin_amdgcn_ballot_w64(shift != 0) != 0
                            : (outer < R || __builtin_amdgcn_ballot_w64(zero != 0) != 0)) {
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                reg[i] = shift_right(reg[i], shift * 8 * (int)sizeof(T));
                if (ORDER == kOuter && (zero >> i & 1)) reg[i] = uintx4{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int i = 0; i < kChunks; ++i) *reinterpret_cast<uintx4 *>(lds + put_at[i]) = reg[i];
    }
};

// Where a lane finds its operands of the 32 rows from r0 on, in the four k steps of a tile
template <class T, int ORDER, int R, int TILES> struct Reader {
    static constexpr int kRowBytes = R * (int)sizeof(T);
    unsigned at[ORDER == kInner ? 4 : TILES];

    __device__ void init(const int (&first)[TILES], int lane)
    {
        const int l31 = lane & 31, h = lane >> 5;
        if (ORDER == kInner) {
#pragma unroll
            for (int s = 0; s < 4; ++s)
                at[s] = l31 * 128 + (((2 * s + h) ^ Tile<T, ORDER, R>::swizzle(l31)) << 4);
        } else if (sizeof(T) == 2) {
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                at[t] = Tile<T, ORDER, R>::outer_at(8 * h + (lane >> 2 & 3), first[t] + (lane & 16) + 4 * (lane & 3));
        } else {
#pragma unroll
            for (int t = 0; t < TILES; ++t) at[t] = Tile<T, ORDER, R>::outer_at(4 * h, first[t] + l31);
        }
    }

    __device__ uintx4 frag(const char *lds, int first, int t, int s) const
    {
        if (ORDER == kInner) return *reinterpret_cast<const uintx4 *>(lds + at[s] + first * 128);
        uintx4 v;
        if (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) shortx4 lds_vec;
            const char *p = lds + at[t] + s * 16 * kRowBytes;
            const uintx2 lo = __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec *)(p)));
            const uintx2 hi = __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec *)(p + 4 * kRowBytes)));
            v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)      // (k + 8: the same exchange of units)
                v[j] = *reinterpret_cast<const unsigned *>(lds + at[t] + (8 * s + j) * kRowBytes);
        }
        return v;
    }
};

template <class T> __device__ inline floatx16 multiply(uintx4 b, uintx4 a, floatx16 c)
{
    if constexpr (sizeof(T) == 4) {
        const floatx4 bf = __builtin_bit_cast(floatx4, b), af = __builtin_bit_cast(floatx4, a);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(bf[j], af[j], c, 0, 0, 0);
        return c;
    } else if constexpr (Type<T>::kCode == FPN_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, b), __builtin_bit_cast(halfx8, a), c, 0, 0, 0);
    }
}

// A wave's accumulators to memory through its own piece of LDS, 32 rows at a time: written as they lie (a lane has four
// consecutive columns of one row), read back as runs of eight columns of consecutive rows - whole lines for the
// loads and stores, bias loaded once, and one copy of the epilogue's arithmetic (unrolled over a wave's tiles it was 200 KB
// of code for an activation and spilled registers).  `lds` is the wave's, epilogue_bytes(TN); nobody else uses it.
constexpr int epilogue_bytes(int tn) { return 32 * (32 * tn * 4 + 16); }

// MODE: a plain product, a gated one, or the gated block's backward epilogue on a plain one
enum { kPlainMode = 0, kGatedMode = 1, kGateGradMode = 2 };

template <class T, int MODE, int TM, int TN>
__device__ inline void store_piece(const Args &p, const floatx16 (&acc)[TM][TN], char *lds, int member, int split, long m0, int n0, int lane)
{
    constexpr bool EXACT = sizeof(T) == 4, GATED = MODE == kGatedMode;
    constexpr int kTN = TN, kEpilogueRow = 32 * kTN * 4 + 16;
    const int l31 = lane & 31, h = lane >> 5;
    constexpr int kRuns = GATED ? 2 * kTN : 4 * kTN, kRowsAtOnce = 64 / kRuns, kBatch = EXACT || MODE == kGateGradMode ? 1 : 2;     // runs of eight columns per row
    const int run = lane % kRuns, row0 = lane / kRuns;
    const int n = n0 + run * 8;
    const long left = p.n - n;
    auto put = [&](const floatx16 (&c)[kTN]) {
#pragma unroll
        for (int j = 0; j < kTN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                floatx4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = c[j][4 * q + e];
                *reinterpret_cast<floatx4 *>(lds + l31 * kEpilogueRow + (32 * j + 8 * q + 4 * h) * 4) = v;
            }
    };
    float bias[8] = {}, bias2[8] = {};
    if (MODE != kGateGradMode && left > 0 && p.bias[GATED ? 0 : member]) load8(reinterpret_cast<const T *>(p.bias[GATED ? 0 : member]) + n, left, bias);
    if (GATED && left > 0 && p.bias[1]) load8(reinterpret_cast<const T *>(p.bias[1]) + n, left, bias2);
    // the residual of the next rows is on its way while the present ones are finished (8192 x 4096 x 4096 bf16 with gelu and
    // residual: 251 us without, 244 with)
    constexpr bool RESIDUAL = MODE == kPlainMode;
    Raw8<T> res[RESIDUAL ? kBatch : 1];
    auto fetch = [&](long row) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) res[RESIDUAL ? b : 0].load(reinterpret_cast<const T *>(p.residual) + min(row + b * kRowsAtOnce, p.m - 1) * p.ldr + n, left);
    };
    const bool adds = RESIDUAL && p.residual && !p.partial && left > 0;
    if (adds) fetch(m0 + row0);
#pragma unroll 1
    for (int i = 0; i < TM; ++i) {
        if (i == 0) put(acc[0]);
        else if (TM == 2 || i == 1) put(acc[TM > 1 ? 1 : 0]);
        else if (i == 2) put(acc[TM > 2 ? 2 : 0]);
        else put(acc[TM > 2 ? 3 : 0]);
        if (left <= 0) continue;
        // two rows' loads at a time, then their arithmetic, then their stores: with one wave per SIMD nothing else
        // would cover the latency
#pragma unroll 1
        for (int r = row0; r < 32; r += kRowsAtOnce * kBatch) {
            const long m = m0 + 32 * i + r;
            float v[kBatch][8], v2[GATED ? kBatch : 1][8];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const float *from = reinterpret_cast<const float *>(lds + (r + b * kRowsAtOnce) * kEpilogueRow) + run * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[b][e] = from[e];
                    if (GATED) v2[b][e] = from[16 * kTN + e];
                }
            }
            if constexpr (MODE == kGateGradMode) {
                // the gated block's backward pass: dh in, dg and du out, rounded to T as the next products' operands like
                // grad_kernel's (no bias in such a product: its registers take the column sums)
                float g[kBatch][8], u[kBatch][8];
#pragma unroll
                for (int b = 0; b < kBatch; ++b) {
                    const long row = min(m + b * kRowsAtOnce, p.m - 1);
                    load8(p.gate + row * p.ldp + n, left, g[b]);
                    load8(p.up + row * p.ldp + n, left, u[b]);
                }
                for_activation(p.act, [&](auto tag) {
#pragma unroll
                    for (int b = 0; b < kBatch; ++b)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float value;
                            const float slope = activate_grad<decltype(tag)::value, EXACT>(g[b][e], value);
                            g[b][e] = v[b][e] * u[b][e] * slope;
                            u[b][e] = v[b][e] * value;
                        }
                });
#pragma unroll
                for (int b = 0; b < kBatch; ++b)
                    if (m + b * kRowsAtOnce < p.m) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            bias[e] += g[b][e];
                            bias2[e] += u[b][e];
                        }
                        store8(reinterpret_cast<T *>(p.c[0]) + (m + b * kRowsAtOnce) * p.ldc + n, left, g[b]);
                        store8(reinterpret_cast<T *>(p.c[1]) + (m + b * kRowsAtOnce) * p.ldc + n, left, u[b]);
                    }
                continue;
            }
            if (p.partial) {
#pragma unroll
                for (int b = 0; b < kBatch; ++b)
                    if (m + b * kRowsAtOnce < p.m) {
                        float *to = p.partial + ((((long)member * p.splits + split) * (GATED ? 2 : 1)) * p.m + m + b * kRowsAtOnce) * p.n + n;
                        store8(to, left, v[b]);
                        if (GATED) store8(to + p.m * p.n, left, v2[b]);
                    }
                continue;
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[b][e] += bias[e];
                    if (GATED) v2[b][e] += bias2[e];
                }
            if (p.pre[0])
#pragma unroll
                for (int b = 0; b < kBatch; ++b)
                    if (m + b * kRowsAtOnce < p.m) {
                        store8(p.pre[0] + (m + b * kRowsAtOnce) * p.ldp + n, left, v[b]);
                        if (GATED) store8(p.pre[1] + (m + b * kRowsAtOnce) * p.ldp + n, left, v2[b]);
                    }
            if (p.act != FPN_ACT_NONE)
                for_activation(p.act, [&](auto tag) {
#pragma unroll
                    for (int b = 0; b < kBatch; ++b)
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[b][e] = activate<decltype(tag)::value, EXACT>(v[b][e]);
                });
            if (adds) {
#pragma unroll
                for (int b = 0; b < kBatch; ++b) res[RESIDUAL ? b : 0].add_to(v[b]);
                // (behind a piece's last rows come the next piece's first)
                fetch(r + kRowsAtOnce * kBatch < 32 ? m + kRowsAtOnce * kBatch : m0 + 32 * (i + 1) + row0);
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (GATED) v[b][e] *= v2[b][e];
                if (m + b * kRowsAtOnce < p.m) {
                    if (p.c_float) store8(reinterpret_cast<float *>(p.c[member]) + (m + b * kRowsAtOnce) * p.ldc + n, left, v[b]);
                    else store8(reinterpret_cast<T *>(p.c[member]) + (m + b * kRowsAtOnce) * p.ldc + n, left, v[b]);
                }
            }
        }
    }
    if constexpr (MODE == kGateGradMode) {
        if (!p.sums) return;
        // the column sums of this wave's rows: the lanes of one run of columns, in a fixed order
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int far = kRuns; far < 64; far *= 2) {
                bias[e] += __shfl_xor(bias[e], far);
                bias2[e] += __shfl_xor(bias2[e], far);
            }
        if (row0 == 0 && left > 0) {
            float *to = p.sums + m0 / (32 * TM) * 2 * p.n + n;
            store8(to, left, bias);
            store8(to + p.n, left, bias2);
        }
    }
}

// Workgroup -> (output tile, batch member, split).  Workgroups go round the eight XCDs; each XCD takes a contiguous
// piece of the tile sequence, in which groups of eight tile rows are walked column by column: the tiles that share
// operands run on one XCD at about the same time and meet in its L2.
struct Place { long mt; int nt, member, split; };
__device__ inline Place place(const Args &p, long block, long blocks)
{
    const long each = blocks >> 3, more = blocks & 7, xcd = block & 7;
    long i = xcd * each + min(xcd, more) + (block >> 3);
    Place r;
    const long tiles = p.mt * p.nt;
    const long z = i / tiles;
    i -= z * tiles;
    r.split = (int)(z % p.splits);
    r.member = (int)(z / p.splits);
    constexpr long kGroup = 8;
    const long group = i / (kGroup * p.nt);
    const long height = min(kGroup, p.mt - group * kGroup);
    const long in = i - group * kGroup * p.nt;
    r.mt = group * kGroup + in % height;
    r.nt = (int)(in / height);
    return r;
}

template <class T, int ORDER_A, int ORDER_B, int BM, int BN, int WM, int WN, bool GATED>
__global__ __launch_bounds__(kThreads) void product_kernel(const Args p)
{
    static_assert(WM * WN == 4, "four waves");
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    extern __shared__ char lds[];
    constexpr int kABytes = BM * kTileBytes, kStage = (BM + BN) * kTileBytes;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;
    const Place at = place(p, blockIdx.x, gridDim.x);
    constexpr int kCols = GATED ? BN / 2 : BN;                 // output columns of the tile
    const long m0 = at.mt * BM;
    const int n0 = at.nt * kCols;

    Tile<T, ORDER_A, BM> ta;
    Tile<T, ORDER_B, kCols> tb[GATED ? 2 : 1];                 // GATED: the gate half, the up half
    ta.init(p.m - m0, p.m, p.k, tid);
#pragma unroll
    for (int g = 0; g < (GATED ? 2 : 1); ++g) tb[g].init(p.n - n0, p.n, p.k, tid);

    int am[TM], bn[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) am[i] = (wm * TM + i) * 32;
    // GATED: the first half of a wave's column tiles are gate columns, the second half the same columns of up
#pragma unroll
    for (int j = 0; j < TN; ++j) bn[j] = GATED ? (wn * (TN / 2) + j % (TN / 2)) * 32 : (wn * TN + j) * 32;
    Reader<T, ORDER_A, BM, TM> ra;
    Reader<T, ORDER_B, kCols, TN> rb;
    ra.init(am, lane);
    rb.init(bn, lane);

    const long per_seg = (p.k + Tile<T, ORDER_A, BM>::BK - 1) / Tile<T, ORDER_A, BM>::BK;
    const long first = at.split * p.tiles_per_split, last = min(first + p.tiles_per_split, per_seg * p.segs);

    floatx16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    int seg = -1;
    auto load = [&](long t) {
        const int s = t >= per_seg;
        if (s != seg) {
            seg = s;
            ta.segment(p.a[s], p.lda[s], m0, p.k, tid);
            if (GATED) {
                tb[0].segment(p.b[0], p.ldb[0], n0, p.k, tid);
                tb[GATED].segment(p.b[1], p.ldb[1], n0, p.k, tid);
            } else {
                tb[0].segment(p.b[s + at.member], p.ldb[s + at.member], n0, p.k, tid);
            }
        }
        ta.load(t - s * per_seg, tid);
        tb[0].load(t - s * per_seg, tid);
        if (GATED) tb[GATED].load(t - s * per_seg, tid);
    };
    auto put = [&](char *stage) {
        ta.put(stage);
        tb[0].put(stage + kABytes);
        if (GATED) tb[GATED].put(stage + kABytes + kCols * kTileBytes);
    };
    if (first < last) {
        load(first);
        put(lds);
    }
    __syncthreads();
    for (long t = first; t < last; ++t) {
        const char *cur = lds + ((t - first) & 1) * kStage;
        char *next = lds + ((t - first + 1) & 1) * kStage;
        if (t + 1 < last) load(t + 1);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            uintx4 fa[TM], fb[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) fa[i] = ra.frag(cur, am[i], i, s);
#pragma unroll
            for (int j = 0; j < TN; ++j)
                fb[j] = rb.frag(cur + kABytes + (GATED && j >= TN / 2 ? kCols * kTileBytes : 0), bn[j], j, s);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int i = 0; i < TM; ++i) acc[i][j] = multiply<T>(fb[j], fa[i], acc[i][j]);
        }
        if (t + 1 < last) put(next);
        __syncthreads();
    }

    store_piece<T, GATED ? kGatedMode : kPlainMode, TM, TN>(p, acc, lds + wave * epilogue_bytes(TN), at.member, at.split, m0 + am[0], n0 + bn[0], lane);
}

// Joins the partial sums of a split product: a workgroup takes 32 runs of eight columns, its eight rows of threads
// every eighth split each, and the eight sums meet in LDS in a fixed order.
template <class T, bool GATED> __global__ __launch_bounds__(kThreads) void join_kernel(const Args p)
{
    __shared__ float part[GATED ? 2 : 1][8][32][8];
    const int g = threadIdx.x & 31, lane_split = threadIdx.x >> 5;
    const int per_row = (p.n + 7) / 8;
    const long run = (long)blockIdx.x * 32 + g;
    const int member = blockIdx.y;
    const long m = run / per_row;
    const int n = (int)(run % per_row) * 8;
    float v[8] = {}, v2[8] = {};
    if (m < p.m) {
        const long plane = p.m * p.n, step = plane * (GATED ? 2 : 1);
        const float *from = p.partial + ((long)member * p.splits) * step + m * p.n + n;
        for (int s = lane_split; s < p.splits; s += 8) {
            float w[8];
            load8(from + s * step, p.n - n, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += w[i];
            if (GATED) {
                load8(from + s * step + plane, p.n - n, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) v2[i] += w[i];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        part[0][lane_split][g][i] = v[i];
        if (GATED) part[GATED][lane_split][g][i] = v2[i];
    }
    __syncthreads();
    if (lane_split || m >= p.m) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        for (int s = 1; s < 8; ++s) {
            v[i] += part[0][s][g][i];
            if (GATED) v2[i] += part[GATED][s][g][i];
        }
    }
    finish8<T, GATED>(p, member, m, n, v, v2);
}

// ---- host side --------------------------------------------------------------------------------------------------

// How a product is cut: tile, splits of k, and the bytes of partial sums that takes
struct Plan {
    bool few;               // the few-row kernel (feed_forward_few.h), its MT and NT in bm and bn
    bool wide;              // the kernel of feed_forward_wide.h
    int bm, bn;
    int splits;
    long tiles_per_split;
    size_t partial_bytes;
};
// threads of a workgroup of the pipelined kernel's shapes, which have BM output rows
constexpr int wide_threads(int bm) { return bm == 64 ? 256 : 512; }
// (aligned: every operand consists of whole 16-byte chunks at 16-byte addresses)
Plan plan_product(int dtype, long m, int n, long k, int segs, int batch, bool gated, bool aligned, int order_a, int order_b);

// whether an operand consists of whole 16-byte chunks
inline bool whole_chunks(const void *p, long ld, int order, long extent, int element)
{
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * element % 16 == 0 && (order == kInner || extent * element % 16 == 0);
}

template <class T> int launch_few(const Args &p, int order_b, bool gated, int mt, int nt, hipStream_t stream);
template <class T> int launch_wide(const Args &p, int order_a, int order_b, bool gated, int bm, int bn, long blocks, hipStream_t stream);

// workgroups of a planned product (of the tiled kernels)
inline long plan_blocks(const Args &p, bool gated, const Plan &plan)
{
    const int cols = gated ? plan.bn / 2 : plan.bn;
    return (p.m + plan.bm - 1) / plan.bm * ((p.n + cols - 1) / cols) * plan.splits * p.batch;
}

// Launches a planned product (p.partial and the plan's fields are filled in here)
template <class T> int launch_product(Args p, int order_a, int order_b, bool gated, const Plan &plan, float *partial, hipStream_t stream);

#ifndef FPN_FF_INSTANTIATE          // (defined by the one file per type that compiles the kernels)
extern template int launch_product<float>(Args, int, int, bool, const Plan &, float *, hipStream_t);
extern template int launch_product<__bf16>(Args, int, int, bool, const Plan &, float *, hipStream_t);
extern template int launch_product<_Float16>(Args, int, int, bool, const Plan &, float *, hipStream_t);
extern template int launch_wide<float>(const Args &, int, int, bool, int, int, long, hipStream_t);
extern template int launch_wide<__bf16>(const Args &, int, int, bool, int, int, long, hipStream_t);
extern template int launch_wide<_Float16>(const Args &, int, int, bool, int, int, long, hipStream_t);
extern template int launch_few<float>(const Args &, int, bool, int, int, hipStream_t);
extern template int launch_few<__bf16>(const Args &, int, bool, int, int, hipStream_t);
extern template int launch_few<_Float16>(const Args &, int, bool, int, int, hipStream_t);
#endif

// (a launch has fewer than 2^32 threads)
inline int check_grid(long blocks, int threads)
{
    if (blocks > 0xffffffffl / threads) return fail(FPN_E_UNSUPPORTED, "a launch of %ld workgroups of %d threads", blocks, threads);
    return FPN_OK;
}

#define FPN_FF_LAUNCH(A, B, BM_, BN_, WM_, WN_, G)                                                                            \
    do {                                                                                                                      \
        auto kern = product_kernel<T, A, B, BM_, BN_, WM_, WN_, G>;                                                           \
        constexpr int bytes = std::max(2 * (BM_ + BN_) * kTileBytes, WM_ * WN_ * epilogue_bytes(BN_ / WN_ / 32));             \
        if (check_grid(blocks, kThreads) != FPN_OK) return FPN_E_UNSUPPORTED;                                                 \
        if (!allow_dynamic_lds(reinterpret_cast<const void *>(kern), bytes))                                                  \
            return fail(FPN_E_LAUNCH, "%d bytes of LDS refused", bytes);                                                      \
        hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(kThreads), bytes, stream, p);                                   \
    } while (0)

template <class T, int BM, int BN, int WM, int WN>
int launch_tiles(const Args &p, int order_a, int order_b, bool gated, long blocks, hipStream_t stream)
{
    if (gated) {
        if (order_b == kOuter) FPN_FF_LAUNCH(kInner, kOuter, BM, BN, WM, WN, true);
        else FPN_FF_LAUNCH(kInner, kInner, BM, BN, WM, WN, true);
    } else if (order_a == kOuter) {
        FPN_FF_LAUNCH(kOuter, kOuter, BM, BN, WM, WN, false);
    } else if (order_b == kOuter) {
        FPN_FF_LAUNCH(kInner, kOuter, BM, BN, WM, WN, false);
    } else {
        FPN_FF_LAUNCH(kInner, kInner, BM, BN, WM, WN, false);
    }
    return check_launch("feed-forward product");
}

template <class T> int launch_join(const Args &p, bool gated, hipStream_t stream)
{
    const long runs8 = p.m * ((p.n + 7) / 8);
    const long join_blocks = (runs8 + 31) / 32;             // (partial sums are at most 128 MB, or those of 64 rows)
    const dim3 grid((unsigned)join_blocks, p.batch);
    if (gated) hipLaunchKernelGGL((join_kernel<T, true>), grid, dim3(kThreads), 0, stream, p);
    else hipLaunchKernelGGL((join_kernel<T, false>), grid, dim3(kThreads), 0, stream, p);
    return check_launch("join of a split product");
}

template <class T> int launch_product(Args p, int order_a, int order_b, bool gated, const Plan &plan, float *partial, hipStream_t stream)
{
    p.splits = plan.splits;
    p.tiles_per_split = plan.tiles_per_split;
    p.partial = plan.splits > 1 ? partial : nullptr;
    if (plan.few) {
        const int rc = launch_few<T>(p, order_b, gated, plan.bm, plan.bn, stream);
        return rc != FPN_OK || !p.partial ? rc : launch_join<T>(p, gated, stream);
    }
    const int cols = gated ? plan.bn / 2 : plan.bn;
    p.mt = (p.m + plan.bm - 1) / plan.bm;
    p.nt = (p.n + cols - 1) / cols;
    const long blocks = plan_blocks(p, gated, plan);
    int rc;
    if (plan.wide) rc = launch_wide<T>(p, order_a, order_b, gated, plan.bm, plan.bn, blocks, stream);
    else if (plan.bm == 128) rc = launch_tiles<T, 128, 128, 2, 2>(p, order_a, order_b, gated, blocks, stream);
    else rc = launch_tiles<T, 64, 128, 2, 2>(p, order_a, order_b, gated, blocks, stream);
    if (rc != FPN_OK || !p.partial) return rc;
    return launch_join<T>(p, gated, stream);
}

}  // namespace ff
}  // namespace fpn
