// The feed-forward products' kernel for few rows (single tokens, a handful of frustums): bound by reading the weights
// once, so what counts is how many bytes of them are on their way at any time, and that one launch does it all.
//
// A workgroup owns 16 NT columns (of each half where GATED) and all rows, in MT groups of 16; its waves (sixteen, or eight where
// a step is over 3 KB) split k.
// A wave walks its share in steps of one 64-byte stretch of k (32 sixteen-bit elements, 16 floats): per step 1 KB of weights
// per 16 columns and 1 KB of x per 16 rows come straight into the wave's own ring in LDS (160 KB a CU, all of
// it requested before the first wait), from where MFMAs of 16 x 16 take them.  No wave waits for
// another until its share is done; then the partial tiles meet in LDS and are summed in wave order, so a result
// does not depend on timing, and the epilogue follows.
#pragma once
#include "feed_forward_wide.h"

namespace fpn {
namespace ff {

template <int MT, int NT, bool GATED> struct FewShape {
    static constexpr int kB = NT * (GATED ? 2 : 1);            // 16-column groups of weights per step
    static constexpr int kSlot = kB + MT;                      // KB (= requests) per step
    static constexpr int kWaves = kSlot <= 3 ? 16 : 8, kThreads = 64 * kWaves;
    static constexpr int kRing = 160 / kWaves / kSlot;         // steps on their way
    static constexpr int kBytes = std::max(kWaves * kRing * kSlot * 1024, kWaves * kB * MT * 1024);
    static_assert(kBytes <= 160 * 1024, "LDS of a CU");
};

// wait until at most LEFT of this wave's requests are on their way
template <int LEFT> __device__ inline void landed()
{
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LEFT) : "memory");
}

// 16 G rows (m or n) x 64 bytes of k, G requests.  LDS image, kInner: rows of 64 bytes, chunks permuted by row >> 2 & 3;
// kOuter: k rows of 16 G elements (the wider, the fewer cache lines a request touches), the stretches of 16 elements
// permuted by k, so that the rows that are read together lie on different banks.
template <class T, int ORDER, int G> struct FewTile {
    static constexpr int E = Type<T>::kE, BK = 64 / (int)sizeof(T), kRow = 16 * G * (int)sizeof(T);
    static constexpr int kLanes = kRow / 16;                    // kOuter: lanes of a k row
    const char *base;
    long step;
    unsigned off[G];

    __device__ static int turn(int k) { return (sizeof(T) == 2 ? k : k >> 2) & (G - 1); }

    // the chunk request i's slot of this lane takes: kInner: m / n and first k; kOuter: k and first m / n
    __device__ static void slot(int i, int lane, int &row, int &first)
    {
        if (ORDER == kInner) {
            row = 16 * i + (lane >> 2);
            first = ((lane & 3) ^ (row >> 2 & 3)) * E;
        } else {
            constexpr int kPer = 16 / E;                        // chunks of a stretch
            row = i * (64 / kLanes) + lane / kLanes;
            const int c = lane % kLanes;
            first = (((c / kPer) ^ turn(row)) * kPer + c % kPer) * E;
        }
    }

    __device__ void init(const void *p, long ld, long start, long left, int lane)
    {
        base = reinterpret_cast<const char *>(p) + (ORDER == kInner ? start * ld : start) * (long)sizeof(T);
        step = (ORDER == kInner ? 1 : ld) * BK * (long)sizeof(T);
#pragma unroll
        for (int i = 0; i < G; ++i) {
            int row, first;
            slot(i, lane, row, first);
            off[i] = ORDER == kInner ? (unsigned)((min((long)row, left - 1) * ld + first) * (long)sizeof(T))
                                     : (unsigned)((row * ld + min((long)first, left - E)) * (long)sizeof(T));
        }
    }

    __device__ void issue(unsigned lds, long kt) const
    {
#pragma unroll
        for (int i = 0; i < G; ++i) request<0>(lds + i * 1024, off[i], base + kt * step);
    }

    __device__ void put_tail(char *lds, long kt, int left_k, int lane) const
    {
        const char *at = base + kt * step;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            int row, first;
            slot(i, lane, row, first);
            const int inside = ORDER == kInner ? left_k - first : (row < left_k ? E : 0);
            uintx4 v = {0, 0, 0, 0};
            if (inside >= E) {
                v = *reinterpret_cast<const uintx4_u *>(at + off[i]);
            } else if (inside > 0) {
                typedef T vec __attribute__((ext_vector_type(E)));
                vec e;
#pragma unroll
                for (int j = 0; j < E; ++j) e[j] = j < inside ? reinterpret_cast<const T *>(at + off[i])[min(j, inside - 1)] : (T)0.f;
                v = __builtin_bit_cast(uintx4, e);
            }
            *reinterpret_cast<uintx4 *>(lds + i * 1024 + lane * 16) = v;
        }
    }

    // a lane's operand of group i: m / n = 16 i + (lane & 15), k = 8 (lane >> 4) + 0..7 (16 bit) or 4 (lane >> 4) + 0..3
    __device__ static uintx4 frag(const char *lds, int i, int lane)
    {
        const int r = lane & 15, g = lane >> 4;
        if (ORDER == kInner) return *reinterpret_cast<const uintx4 *>(lds + i * 1024 + r * 64 + ((g ^ (r >> 2 & 3)) << 4));
        uintx4 v;
        if (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) shortx4 lds_vec;
            const int k = 8 * g + (lane >> 2 & 3);
            const uintx2 lo = __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                             (lds_vec *)(lds + k * kRow + ((i ^ turn(k)) << 5) + (lane & 3) * 8)));
            const uintx2 hi = __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                             (lds_vec *)(lds + (k + 4) * kRow + ((i ^ turn(k + 4)) << 5) + (lane & 3) * 8)));
            v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = *reinterpret_cast<const unsigned *>(lds + (4 * g + j) * kRow + ((i ^ turn(4 * g)) << 6) + r * 4);
        }
        return v;
    }
};

template <class T> __device__ inline floatx4 multiply16(uintx4 b, uintx4 a, floatx4 c)
{
    if constexpr (sizeof(T) == 4) {
        const floatx4 bf = __builtin_bit_cast(floatx4, b), af = __builtin_bit_cast(floatx4, a);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(bf[j], af[j], c, 0, 0, 0);
        return c;
    } else if constexpr (Type<T>::kCode == FPN_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, b), __builtin_bit_cast(halfx8, a), c, 0, 0, 0);
    }
}

// one output element's epilogue
template <class T, bool GATED> __device__ inline void finish1(const Args &p, long m, int n, float v, float v2)
{
    constexpr bool EXACT = sizeof(T) == 4;
    if (p.bias[0]) v += (float)reinterpret_cast<const T *>(p.bias[0])[n];
    if (GATED && p.bias[1]) v2 += (float)reinterpret_cast<const T *>(p.bias[1])[n];
    if (p.pre[0]) {
        p.pre[0][m * p.ldp + n] = v;
        if (GATED) p.pre[1][m * p.ldp + n] = v2;
    }
    if (p.act != FPN_ACT_NONE) for_activation(p.act, [&](auto tag) { v = activate<decltype(tag)::value, EXACT>(v); });
    if (GATED) v *= v2;
    if (p.residual) v += (float)reinterpret_cast<const T *>(p.residual)[m * p.ldr + n];
    if (p.c_float) reinterpret_cast<float *>(p.c[0])[m * p.ldc + n] = v;
    else reinterpret_cast<T *>(p.c[0])[m * p.ldc + n] = (T)v;
}

template <class T, int ORDER_B, int MT, int NT, bool GATED>
__global__ __launch_bounds__((FewShape<MT, NT, GATED>::kThreads)) void few_product_kernel(const Args p)
{
    using F = FewShape<MT, NT, GATED>;
    using TileA = FewTile<T, kInner, MT>;
    using TileB = FewTile<T, ORDER_B, NT>;
    constexpr int kHalves = GATED ? 2 : 1;
    constexpr int kB = F::kB, kRing = F::kRing, kSlot = F::kSlot, kWaves = F::kWaves, BK = TileA::BK;
    extern __shared__ char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Workgroups go round the eight XCDs: neighbouring columns, which may share cache lines of row-major weights, on one XCD
    const int each = gridDim.x >> 3, more = gridDim.x & 7, xcd = blockIdx.x & 7;
    const int block = xcd * each + min(xcd, more) + (int)(blockIdx.x >> 3), split = block % p.splits, n0 = block / p.splits * (16 * NT);

    TileA ta;
    TileB tb[kHalves];
    ta.init(p.a[0], p.lda[0], 0, p.m, lane);
#pragma unroll
    for (int g = 0; g < kHalves; ++g) tb[g].init(p.b[g], p.ldb[g], n0, (ORDER_B == kOuter ? p.load_n : p.n) - n0, lane);
    const int full = (int)(p.k / BK);                       // (k is a layer's width here: below 2^21)
    const int share = split * kWaves + wave, shares = p.splits * kWaves;
    const int s0 = (int)((long)full * share / shares), len = (int)((long)full * (share + 1) / shares) - s0;
    char *ring = lds + wave * (kRing * kSlot * 1024);
    const unsigned ring0 = lds_address(ring);

    floatx4 acc[MT][kB];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < kB; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

    auto ask = [&](long s, int slot) {
        const unsigned to = ring0 + slot * (kSlot * 1024);
#pragma unroll
        for (int g = 0; g < kHalves; ++g) tb[g].issue(to + g * NT * 1024, s);
        ta.issue(to + kB * 1024, s);
    };
    uintx4 fa[MT], fb[kB];
    auto read = [&](int slot) {
        const char *from = ring + slot * (kSlot * 1024);
#pragma unroll
        for (int j = 0; j < kB; ++j) fb[j] = TileB::frag(from + j / NT * NT * 1024, j % NT, lane);
#pragma unroll
        for (int i = 0; i < MT; ++i) fa[i] = TileA::frag(from + kB * 1024, i, lane);
    };
    auto multiply_all = [&] {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < kB; ++j) acc[i][j] = multiply16<T>(fb[j], fa[i], acc[i][j]);
    };
    if (len > 0) {
        int next = 0;                                     // the step asked for next, from s0 (behind the share's end: read, not used)
        auto ask_next = [&](int slot) {
            ask(s0 + next, slot);
            next = next + 1 == len ? 0 : next + 1;
        };
#pragma unroll
        for (int i = 0; i < kRing; ++i) ask_next(i);
        int slot = 0;
        for (int s = 0; s < len; ++s) {
            landed<(kRing - 1) * kSlot>();
            read(slot);
            // the reads have returned before the slot is asked for again
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
            ask_next(slot);
            multiply_all();
            slot = slot == kRing - 1 ? 0 : slot + 1;
        }
        landed<0>();
    }
    const int left = (int)(p.k - full * BK);
    if (left && share == shares - 1) {
#pragma unroll
        for (int g = 0; g < kHalves; ++g) tb[g].put_tail(ring + g * NT * 1024, full, left, lane);
        ta.put_tail(ring + kB * 1024, full, left, lane);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        read(0);
        multiply_all();
    }
    // partial tiles: register r of a lane = column 4 (lane >> 4) + r, row lane & 15
    __syncthreads();
    float *part = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < kB; ++j)
            *reinterpret_cast<floatx4 *>(part + ((wave * MT + i) * kB + j) * 256 + (lane & 15) * 16 + (lane >> 4) * 4) = acc[i][j];
    __syncthreads();
    for (int e = tid; e < MT * NT * 256; e += F::kThreads) {
        const int group = e >> 8, i = group / NT, j = group % NT;
        const long m = 16l * i + (e >> 4 & 15);
        const int n = n0 + 16 * j + (e & 15);
        if (m >= p.m || n >= p.n) continue;
        float v = 0.f, v2 = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            v += part[((w * MT + i) * kB + j) * 256 + (e & 255)];
            if (GATED) v2 += part[((w * MT + i) * kB + NT + j) * 256 + (e & 255)];
        }
        if (p.partial) {
            float *to = p.partial + ((long)split * kHalves * p.m + m) * p.n + n;
            *to = v;
            if (GATED) to[p.m * p.n] = v2;
        } else {
            finish1<T, GATED>(p, m, n, v, v2);
        }
    }
}

#define FPN_FF_FEW(B, MT, NT, G)                                                                                              \
    do {                                                                                                                      \
        auto kern = few_product_kernel<T, B, MT, NT, G>;                                                                      \
        constexpr int bytes = FewShape<MT, NT, G>::kBytes;                                                                    \
        if (!allow_dynamic_lds(reinterpret_cast<const void *>(kern), bytes))                                                  \
            return fail(FPN_E_LAUNCH, "%d bytes of LDS refused", bytes);                                                      \
        hipLaunchKernelGGL(kern, dim3((unsigned)((p.n + 16 * NT - 1) / (16 * NT) * p.splits)), dim3((FewShape<MT, NT, G>::kThreads)), bytes, stream, p);     \
        return check_launch("feed-forward product, few rows");                                                                \
    } while (0)

template <class T> int launch_few(const Args &p, int order_b, bool gated, int mt, int nt, hipStream_t stream)
{
#define FPN_FF_FEW_ORDER(MT, NT, G)                             \
    do {                                                        \
        if (order_b == kOuter) FPN_FF_FEW(kOuter, MT, NT, G);   \
        if constexpr (NT < 4) FPN_FF_FEW(kInner, MT, NT, G);    \
    } while (0)
    // (64 columns: 16-bit weights only; floats fill a cache line with 32)
    if constexpr (sizeof(T) == 2) {
        if (nt == 4 && gated && mt == 1) FPN_FF_FEW_ORDER(1, 4, true);
        if (nt == 4 && mt == 1) FPN_FF_FEW_ORDER(1, 4, false);
        if (nt == 4) FPN_FF_FEW_ORDER(2, 4, false);
    }
    if (nt == 2 && gated && mt == 1) FPN_FF_FEW_ORDER(1, 2, true);
    if (nt == 2 && gated && mt == 2) FPN_FF_FEW_ORDER(2, 2, true);
    if (nt == 2 && gated) FPN_FF_FEW_ORDER(4, 2, true);
    if (nt == 2 && mt == 1) FPN_FF_FEW_ORDER(1, 2, false);
    if (nt == 2 && mt == 2) FPN_FF_FEW_ORDER(2, 2, false);
    if (nt == 2) FPN_FF_FEW_ORDER(4, 2, false);
    if (gated && mt == 1) FPN_FF_FEW_ORDER(1, 1, true);
    if (gated && mt == 2) FPN_FF_FEW_ORDER(2, 1, true);
    if (gated) FPN_FF_FEW_ORDER(4, 1, true);
    if (mt == 1) FPN_FF_FEW_ORDER(1, 1, false);
    if (mt == 2) FPN_FF_FEW_ORDER(2, 1, false);
    FPN_FF_FEW_ORDER(4, 1, false);
    return fail(FPN_E_UNSUPPORTED, "no few-row kernel for this shape");
}

}  // namespace ff
}  // namespace fpn
