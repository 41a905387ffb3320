// The feed-forward products' pipelined kernel: operands are brought into LDS by loads that write it directly.
//
// A workgroup of the largest shape makes a 256 x 256 tile with eight waves, each 128 x 64 of it: 8 MFMA tiles of 32 x 32, 128
// accumulator registers, two waves per SIMD, so that one wave's MFMAs run while the other's requests wait to be taken
// (four waves of 128 x 128 read less from LDS, but every request that waited stopped the SIMD: 247 us against 235 for the product
// of 8192 x 4096 x 4096 bf16).  The smaller shapes are for fewer rows and columns, where 256 x 256 tiles leave CUs without
// work; fp32 uses only the two smallest, whose matrix rate (153 TFLOP/s at most) bounds it with any tile.
//
// LDS holds four to eight stages of 64 bytes of k per row: 32 sixteen-bit elements, 16 floats.  Stages are asked for in
// pairs, each row's two 64-byte halves of a cache line one right after the other: what a CU receives from L2 comes by whole
// lines, and the halves of a line asked for a stage apart were fetched twice (the product above: 241 us, in pairs 224; with
// 64 x 64 tiles 532 and 403).  A pair is asked for as soon as everyone has read the one that had its place, half of it
// behind the barrier and half in the next step; a wave reads the next half stage while it multiplies the present one:
// one barrier per pair, nothing else waits.  (A second one between a pair's two stages makes no difference in the largest shape,
// twelve alternating runs each: gated 8192 x 2048 x 2 x 8192 455 - 461 us with it and 456 - 466 without, the product above
// 220.4 - 221.0 and 220.6 - 221.5, weights held (out,in) 219.7 - 221.0 and 218.8 - 219.8; the smaller are up to 2 % slower with it.)
//
// The requests are written in assembly because the compiler, which cannot tell the stages apart, would wait for all of
// them before every LDS read.  They have no result registers; the counts in `arrive` are theirs alone, since the loop
// has no other vector memory access.
#pragma once
#include "feed_forward.h"

namespace fpn {
namespace ff {

constexpr int kStretch = 64;                                // bytes of k per stage: 32 sixteen-bit elements, 16 floats
// A shape of workgroup: BM x BN tile, WM x WN waves of TM x TN MFMA tiles, stages in LDS, workgroups per CU.
template <int BM_, int BN_, int WM_, int WN_, int STAGES, int PER_CU> struct Shape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, kStages = STAGES;
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves, TM = BM / WM / 32, TN = BN / WN / 32;
    static constexpr int kStage = (BM + BN) * kStretch;            // bytes: BM rows of a, BN of b
    static_assert(kThreads == wide_threads(BM), "what the host checks a grid with");
    static constexpr int kPerSimd = kWaves * PER_CU / 4;               // waves
    static constexpr int kEpilogueBytes = epilogue_bytes(TN);
    static constexpr int kBytes = std::max(kStages * kStage, kWaves * kEpilogueBytes);
};
using Large = Shape<256, 256, 2, 4, 4, 1>;
using Medium = Shape<256, 128, 4, 2, 6, 1>;
using Small = Shape<128, 128, 4, 2, 4, 2>;
// (one MFMA tile per wave: a product of 1024 x 1024 x 1024 fp32 27 us, with two tiles on half as many waves 42)
using Tiny = Shape<64, 64, 2, 2, 4, 4>;
// Where few workgroups share a CU and k is long, twice the stages cover the latency that the neighbours would have covered
// (16 bits, k from 40 stages on: 4096 x 8192 x 1024 77 us against 82, 1088 x 2000 x 512 15.6 against 20.4; at 34 stages as fast)
using SmallDeep = Shape<128, 128, 4, 2, 8, 1>;
using TinyDeep = Shape<64, 64, 2, 2, 8, 2>;

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"             // (m0 is reserved: nothing here indexes registers through it)
// 16 bytes per lane from base + off to LDS at lds + AT + 16 lane
template <int AT> __device__ inline void request(unsigned lds, unsigned off, const void *base)
{
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 : : "s"(lds), "v"(off), "s"(base), "i"(AT) : "m0", "scc");
}
#pragma clang diagnostic pop

// All of this wave's requests but the youngest LEFT have written LDS and all its LDS reads have returned; then
// everyone's.
template <int LEFT> __device__ inline void arrive()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(LEFT) : "memory");
}

__device__ inline unsigned lds_address(const char *p)
{
    return (unsigned)(size_t)(const __attribute__((address_space(3))) char *)p;
}

// One operand's R rows (m or n) x 64 bytes of k of a stage.  A request fills 1 KB: kInner 16 rows of 64 bytes, the four 16-byte
// chunks of row r permuted by r >> 2 & 3; kOuter rows (k) of R elements, permuted as in Tile.  The permutation is on
// the source side: the lane that fills a slot fetches the chunk that belongs there.
template <class T, int ORDER, int R, int WAVES> struct Stream {
    static constexpr int E = Type<T>::kE, BK = kStretch / (int)sizeof(T);
    static constexpr int kPer = R * kStretch / 1024 / WAVES;    // requests per wave
    static constexpr int kRowBytes = R * (int)sizeof(T);        // kOuter
    const char *base;                                       // uniform: k = 0 of the segment
    const char *next[2];                                    // the two stages to be requested next
    long step;                                              // bytes between stages
    unsigned off[kPer];

    // which chunk of the tile request i's slot of this lane takes: row (m, n or k) and first element along the row
    __device__ static void slot(int i, int wave, int lane, int &row, int &first)
    {
        const int q = wave * kPer + i;
        if (ORDER == kInner) {
            row = q * 16 + (lane >> 2);
            first = ((lane & 3) ^ (row >> 2 & 3)) * E;
        } else {
            constexpr int kLanes = kRowBytes / 16;
            row = q * (64 / kLanes) + lane / kLanes;
            // (the place whose image is the slot: both permutations are their own inverses)
            first = (int)(Tile<T, kOuter, R>::outer_at(row, lane % kLanes * E) - row * kRowBytes) / (int)sizeof(T);
        }
    }

    // (widths along kOuter rows are whole chunks; chunks beyond the end repeat the last, rows likewise)
    __device__ void init(const void *p, long ld, long start, long left, int wave, int lane)
    {
        base = reinterpret_cast<const char *>(p) + (ORDER == kInner ? start * ld : start) * (long)sizeof(T);
        step = (ORDER == kInner ? 1 : ld) * BK * (long)sizeof(T);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            int row, first;
            slot(i, wave, lane, row, first);
            if (ORDER == kInner) off[i] = (unsigned)((min((long)row, left - 1) * ld + first) * (long)sizeof(T));
            else off[i] = (unsigned)((row * ld + min((long)first, left - E)) * (long)sizeof(T));
        }
    }

    // request I of kPer of one of the two; lds: the stage's piece for this operand and wave
    template <int I> __device__ void issue(unsigned lds, int half) const { request<I * 1024>(lds, off[I], next[half]); }

    // the last, partial stage of a segment, through registers, zeros behind the last k
    __device__ void put_tail(char *lds, long kt, int left_k, int wave, int lane) const
    {
        const char *at = base + kt * step;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            int row, first;
            slot(i, wave, lane, row, first);
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
            *reinterpret_cast<uintx4 *>(lds + (wave * kPer + i) * 1024 + lane * 16) = v;
        }
    }
};

// A lane's operands of TILES 32-row groups, half a stage of k at a time
template <class T, int ORDER, int R, int TILES> struct StreamReader {
    static constexpr int kRowBytes = R * (int)sizeof(T);
    unsigned at[ORDER == kInner ? 2 : TILES];

    __device__ void init(const int (&first)[TILES], int lane)
    {
        const int l31 = lane & 31, h = lane >> 5;
        if (ORDER == kInner) {
#pragma unroll
            for (int s = 0; s < 2; ++s) at[s] = l31 * 64 + (((2 * s + h) ^ (l31 >> 2 & 3)) << 4);
        } else {
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                at[t] = sizeof(T) == 2 ? Tile<T, kOuter, R>::outer_at(8 * h + (lane >> 2 & 3), first[t] + (lane & 16) + 4 * (lane & 3))
                                       : Tile<T, kOuter, R>::outer_at(4 * h, first[t] + l31);
        }
    }

    __device__ uintx4 frag(const char *lds, int first, int t, int s) const
    {
        if (ORDER == kInner) return *reinterpret_cast<const uintx4 *>(lds + at[s] + first * 64);
        if (sizeof(T) == 4) {
            uintx4 f;
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const unsigned *>(lds + at[t] + (8 * s + j) * kRowBytes);
            return f;
        }
        typedef __attribute__((address_space(3))) shortx4 lds_vec;
        const char *p = lds + at[t] + s * 16 * kRowBytes;
        const uintx2 lo = __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec *)(p)));
        const uintx2 hi = __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec *)(p + 4 * kRowBytes)));
        uintx4 v;
        v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
        return v;
    }
};

// f(0), f(1) .. f(COUNT - 1), each with its number as a type
template <int COUNT, int FROM = 0, class F> __device__ inline void each(F &&f)
{
    if constexpr (FROM < COUNT) {
        f(ActTag<FROM>());
        each<COUNT, FROM + 1>(f);
    }
}

template <class T, int ORDER_A, int ORDER_B, int MODE, class S>
__global__ __launch_bounds__(S::kThreads, S::kPerSimd) void wide_product_kernel(const Args p)
{
    extern __shared__ char lds[];
    constexpr bool GATED = MODE == kGatedMode;
    constexpr int kWaves = S::kWaves, kStages = S::kStages, kStage = S::kStage, kTM = S::TM, kTN = S::TN, BM = S::BM;
    constexpr int kHalves = GATED ? 2 : 1, kCols = S::BN / kHalves, kABytes = BM * kStretch, kHalfBytes = kCols * kStretch;
    // (where a half of b is less than a request per wave, half of the waves request each)
    constexpr bool kDealt = GATED && kHalfBytes / 1024 < kWaves;
    constexpr int kStreams = kDealt ? 1 : kHalves, kWavesB = kDealt ? kWaves / 2 : kWaves;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % S::WM, wn = wave / S::WM;
    const int wave_b = wave % kWavesB, dealt = wave / kWavesB;
    const Place at = place(p, blockIdx.x, gridDim.x);
    const long m0 = at.mt * BM;
    const int n0 = at.nt * kCols;

    int am[kTM], bn[kTN];
#pragma unroll
    for (int i = 0; i < kTM; ++i) am[i] = (wm * kTM + i) * 32;
    // GATED: the first half of a wave's column tiles are of the gate half, the second the same columns of the up half; where a
    // wave has one column tile, gate and up are two waves' (kApart)
    constexpr bool kApart = GATED && kTN == 1;
    static_assert(!kApart || (S::WN == 2 && kTM == 1 && S::WM * (epilogue_bytes(2) + 4096) <= S::kBytes), "two halves, joined in LDS");
#pragma unroll
    for (int j = 0; j < kTN; ++j) bn[j] = kApart ? 0 : GATED ? (wn * (kTN / 2) + j % std::max(kTN / 2, 1)) * 32 : (wn * kTN + j) * 32;
    StreamReader<T, ORDER_A, BM, kTM> ra;
    StreamReader<T, ORDER_B, kCols, kTN> rb;
    ra.init(am, lane);
    rb.init(bn, lane);

    floatx16 acc[kTM][kTN];
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
        for (int j = 0; j < kTN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    Stream<T, ORDER_A, BM, kWaves> sa;
    Stream<T, ORDER_B, kCols, kWavesB> sb[kStreams];
    const long full = p.k / decltype(sa)::BK;               // whole stages of a segment
    const long first = at.split * p.tiles_per_split, last = min(first + p.tiles_per_split, full * p.segs);
    const unsigned lds0 = lds_address(lds);

    const long left_n = (ORDER_B == kOuter ? p.load_n : p.n) - n0;
    auto segment = [&](int s) {
        sa.init(p.a[s], p.lda[s], m0, (ORDER_A == kOuter ? p.load_m : p.m) - m0, wave, lane);
        if (kDealt) {
            sb[0].init(dealt ? p.b[1] : p.b[0], dealt ? p.ldb[1] : p.ldb[0], n0, left_n, wave_b, lane);
        } else if (GATED) {
            sb[0].init(p.b[0], p.ldb[0], n0, left_n, wave, lane);
            sb[kStreams - 1].init(p.b[1], p.ldb[1], n0, left_n, wave, lane);
        } else {
            sb[0].init(p.b[s + at.member], p.ldb[s + at.member], n0, left_n, wave, lane);
        }
    };
    constexpr int kPerA = decltype(sa)::kPer, kPerB = Stream<T, ORDER_B, kCols, kWavesB>::kPer, kPer = kPerA + kStreams * kPerB;
    static_assert(kPerA > 0 && kPerB > 0 && kStages % 2 == 0, "a wave has requests of both operands");
    const unsigned lds_a = lds0 + wave * (kPerA * 1024), lds_b = lds0 + kABytes + (kDealt ? dealt * kHalfBytes : 0) + wave_b * (kPerB * 1024);
    // request Q of a wave's 2 kPer of a pair of stages, the first of which is `stage`: the two stages in turn
    auto issue = [&](auto q, int stage) {
        constexpr int H = decltype(q)::value & 1, Q = decltype(q)::value >> 1;
        constexpr int G = (Q - kPerA) / kPerB * (Q >= kPerA);
        if constexpr (Q < kPerA) sa.template issue<Q>(lds_a + (stage + H) * kStage, H);
        else sb[G].template issue<(Q - kPerA) % kPerB>(lds_b + G * kHalfBytes + (stage + H) * kStage, H);
    };
    auto read_a = [&](const char *stage, int i, int s) { return ra.frag(stage, am[i], i, s); };
    auto read_b = [&](const char *stage, int j, int s) {
        return rb.frag(stage + kABytes + (kApart ? wn * kHalfBytes : GATED && j >= kTN / 2 ? kHalfBytes : 0), bn[j], j, s);
    };
    // Half a stage: multiplies ca, cb while na, nb come from `stage`, and issues requests Q to Q + kPer (none: Q < 0) of the
    // pair at `to`.  A wave issues in order: an MFMA occupies its unit for 32 cycles, in which seven other instructions can go
    // out, so the reads and requests are dealt out among the MFMAs one by one (all in front of a group of four MFMAs cost
    // 12 %); no read is left for the last two, which cover their latency.
    auto step = [&](const uintx4 (&ca)[kTM], const uintx4 (&cb)[kTN], uintx4 (&na)[kTM], uintx4 (&nb)[kTN], const char *stage, int s,
                    auto q, int to) {
        constexpr int Q = decltype(q)::value;
        constexpr int kAll = kTM * kTN;
#pragma unroll
        for (int i = 0; i < kAll; ++i) {
            acc[i % kTM][i / kTM] = multiply<T>(cb[i / kTM], ca[i % kTM], acc[i % kTM][i / kTM]);
#pragma unroll
            for (int r = 0; r < kTM + kTN; ++r)
                if (r * kAll / (kTM + kTN + 2) == i) {
                    if (r < kTM) na[r] = read_a(stage, r, s);
                    else nb[r - kTM] = read_b(stage, r - kTM, s);
                }
            if constexpr (Q >= 0)
                each<kPer>([&](auto j) {
                    constexpr int J = decltype(j)::value;
                    if ((2 * J + 1) * kAll / (2 * kPer) == i) issue(ActTag<Q + J>(), to);
                });
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    uintx4 fa[2][kTM], fb[2][kTN];
    auto read = [&](uintx4 (&a)[kTM], uintx4 (&b)[kTN], int s) {             // of the first stage
#pragma unroll
        for (int i = 0; i < kTM; ++i) a[i] = read_a(lds, i, s);
#pragma unroll
        for (int j = 0; j < kTN; ++j) b[j] = read_b(lds, j, s);
    };

    // segment by segment; a segment's whole stages in this split are [t0, t1)
    for (int s = 0; s < p.segs; ++s) {
        const long t0 = max(first - s * full, 0l), t1 = min(last - s * full, full);
        segment(s);
        if (t0 < t1) {
            const long n = t1 - t0;
            // Behind the segment's end its last stage is asked for again, which nobody reads: a loop without branches, and
            // counts that hold.  On their way at a barrier are the pairs behind the one read next.
            long asked = 0;
            auto aim = [&] {
                const long first_at = t0 + min(asked, n - 1), second_at = t0 + min(asked + 1, n - 1);
                auto point = [&](auto &stream) {
                    stream.next[0] = stream.base + first_at * stream.step;
                    stream.next[1] = stream.base + second_at * stream.step;
                };
                point(sa);
#pragma unroll
                for (int g = 0; g < kStreams; ++g) point(sb[g]);
                asked += 2;
            };
#pragma unroll
            for (int i = 0; i < kStages; i += 2) {
                aim();
                each<kPer>([&](auto j) { issue(ActTag<decltype(j)::value>(), i); });
                if (i < kStages - 2) each<kPer>([&](auto j) { issue(ActTag<kPer + decltype(j)::value>(), i); });
            }
            arrive<(kStages - 4) * kPer + kPer>();
            read(fa[0], fb[0], 0);
            int pair = 0;                                   // its first stage
            for (long t = 1; t < n; t += 2) {
                step(fa[0], fb[0], fa[1], fb[1], lds + pair * kStage, 1, ActTag<kPer>(), pair ? pair - 2 : kStages - 2);
                step(fa[1], fb[1], fa[0], fb[0], lds + (pair + 1) * kStage, 0, ActTag<-1>(), 0);
                step(fa[0], fb[0], fa[1], fb[1], lds + (pair + 1) * kStage, 1, ActTag<-1>(), 0);
                aim();
                arrive<(kStages - 4) * kPer>();
                const int freed = pair;
                pair = pair == kStages - 2 ? 0 : pair + 2;
                step(fa[1], fb[1], fa[0], fb[0], lds + pair * kStage, 0, ActTag<0>(), freed);
            }
            if (n & 1) {                                    // (the second step reads what is not used)
                step(fa[0], fb[0], fa[1], fb[1], lds + pair * kStage, 1, ActTag<-1>(), 0);
                step(fa[1], fb[1], fa[0], fb[0], lds + pair * kStage, 0, ActTag<-1>(), 0);
            }
            arrive<0>();
        }
        // what is left of k, with the last split
        const int left = (int)(p.k - full * decltype(sa)::BK);
        if (left && at.split == p.splits - 1) {
            __syncthreads();
            sa.put_tail(lds, full, left, wave, lane);
#pragma unroll
            for (int g = 0; g < kStreams; ++g)
                sb[g].put_tail(lds + kABytes + (kDealt ? dealt * kHalfBytes : g * kHalfBytes), full, left, wave_b, lane);
            __syncthreads();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                read(fa[0], fb[0], q);
#pragma unroll
                for (int i = 0; i < kTM * kTN; ++i) acc[i % kTM][i / kTM] = multiply<T>(fb[0][i / kTM], fa[0][i % kTM], acc[i % kTM][i / kTM]);
            }
        }
        __syncthreads();
    }
    if constexpr (kApart) {
        float *const meet = reinterpret_cast<float *>(lds + S::WM * epilogue_bytes(2) + wm * 4096) + lane;
        if (wn) {
#pragma unroll
            for (int r = 0; r < 16; ++r) meet[r * 64] = acc[0][0][r];
        }
        __syncthreads();
        if (wn) return;
        floatx16 both[1][2];
        both[0][0] = acc[0][0];
#pragma unroll
        for (int r = 0; r < 16; ++r) both[0][1][r] = meet[r * 64];
        store_piece<T, MODE, 1, 2>(p, both, lds + wave * epilogue_bytes(2), at.member, at.split, m0 + wm * 32, n0, lane);
        return;
    }
    store_piece<T, MODE, kTM, kTN>(p, acc, lds + wave * S::kEpilogueBytes, at.member, at.split, m0 + wm * 32 * kTM,
                             n0 + wn * 32 * (GATED ? kTN / 2 : kTN), lane);
}

#define FPN_FF_WIDE(A, B, G)                                                                                                  \
    do {                                                                                                                      \
        auto kern = wide_product_kernel<T, A, B, G, S>;                                                                       \
        if (check_grid(blocks, S::kThreads) != FPN_OK) return FPN_E_UNSUPPORTED;                                              \
        if (!allow_dynamic_lds(reinterpret_cast<const void *>(kern), S::kBytes))                                              \
            return fail(FPN_E_LAUNCH, "%d bytes of LDS refused", S::kBytes);                                                  \
        hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(S::kThreads), S::kBytes, stream, p);                            \
    } while (0)

template <class T, class S> int launch_shape(const Args &p, int order_a, int order_b, bool gated, long blocks, hipStream_t stream)
{
    if (gated) {
        if (order_b == kOuter) FPN_FF_WIDE(kInner, kOuter, kGatedMode);
        else FPN_FF_WIDE(kInner, kInner, kGatedMode);
    } else if (p.gate) {
        if (order_b == kOuter) FPN_FF_WIDE(kInner, kOuter, kGateGradMode);
        else FPN_FF_WIDE(kInner, kInner, kGateGradMode);
    } else if (order_a == kOuter) {
        FPN_FF_WIDE(kOuter, kOuter, kPlainMode);
    } else if (order_b == kOuter) {
        FPN_FF_WIDE(kInner, kOuter, kPlainMode);
    } else {
        FPN_FF_WIDE(kInner, kInner, kPlainMode);
    }
    return check_launch("feed-forward product, wide");
}

template <class T> int launch_wide(const Args &p, int order_a, int order_b, bool gated, int bm, int bn, long blocks, hipStream_t stream)
{
    if constexpr (sizeof(T) == 2) {                         // (fp32 is bound by its matrix rate with any tile)
        if (bn == 256) return launch_shape<T, Large>(p, order_a, order_b, gated, blocks, stream);
        if (bm == 256) return launch_shape<T, Medium>(p, order_a, order_b, gated, blocks, stream);
        if (p.tiles_per_split >= 40 && blocks <= (bm == 128 ? 1 : 2) * (long)current_device_cus()) {
            if (bm == 128) return launch_shape<T, SmallDeep>(p, order_a, order_b, gated, blocks, stream);
            return launch_shape<T, TinyDeep>(p, order_a, order_b, gated, blocks, stream);
        }
    }
    if (bm == 128) return launch_shape<T, Small>(p, order_a, order_b, gated, blocks, stream);
    return launch_shape<T, Tiny>(p, order_a, order_b, gated, blocks, stream);
}

}  // namespace ff
}  // namespace fpn
