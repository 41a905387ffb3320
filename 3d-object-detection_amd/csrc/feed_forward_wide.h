// The feed-forward products' kernel for large products of 16-bit operands: 256 x 256 output tiles, operands brought
// into LDS by loads that write it directly.
//
// Four waves, each a 128 x 128 quadrant: 16 MFMA tiles of 32 x 32, 256 accumulator registers, one wave per SIMD.
// Per 16 of k a wave reads 8 KB of operands from LDS for 512 cycles of MFMA (half of what the LDS delivers); with 128 x 128
// tiles and 64 x 64 quadrants it is as much for 256 cycles, and the LDS, not the matrix unit, sets the pace.
//
// LDS holds four stages of 32 k (32 KB each).  A wave requests its quarter of stage t + 4 as soon as everyone has read
// stage t, so a request has three stages' time (3072 cycles of MFMA) to arrive, and reads the next 16 of k
// while it multiplies the present ones: one barrier per 32 MFMAs, nothing else waits.
//
// The requests are written in assembly because the compiler, which cannot tell the stages apart, would wait for all of
// them before every LDS read.  They have no result registers; the counts in `arrive` are theirs alone, since the loop
// has no other vector memory access.
#pragma once
#include "feed_forward.h"

namespace fpn {
namespace ff {

constexpr int kWideK = 32;                                  // k per stage
constexpr int kStages = 4;
constexpr int kWideStage = 512 * kWideK * 2;                // bytes: 256 rows of a, 256 of b

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
    if (LEFT == 16) asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)\n\ts_barrier" : : : "memory");
    else if (LEFT == 20) asm volatile("s_waitcnt vmcnt(20) lgkmcnt(0)\n\ts_barrier" : : : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

__device__ inline unsigned lds_address(const char *p)
{
    return (unsigned)(size_t)(const __attribute__((address_space(3))) char *)p;
}

// One operand's R rows (m or n) x 32 k of a stage.  A request fills 1 KB: kInner 16 rows of 64 bytes, the four 16-byte
// chunks of row r permuted by r >> 2 & 3; kOuter 2 or 4 rows (k) of R elements, permuted as in Tile.  The permutation is on
// the source side: the lane that fills a slot fetches the chunk that belongs there.
template <class T, int ORDER, int R> struct Stream {
    static constexpr int kPer = R * 64 / 1024 / 4;          // requests per wave
    static constexpr int kRowBytes = R * 2;                 // kOuter
    const char *base;                                       // uniform: k = 0 of the segment
    const char *next;                                       // the stage to be requested next
    long step;                                              // bytes between stages
    unsigned off[kPer];

    // which chunk of the tile request i's slot of this lane takes: row (m, n or k) and first element along the row
    __device__ static void slot(int i, int wave, int lane, int &row, int &first)
    {
        const int q = wave * kPer + i;
        if (ORDER == kInner) {
            row = q * 16 + (lane >> 2);
            first = ((lane & 3) ^ (row >> 2 & 3)) * 8;
        } else {
            constexpr int kLanes = kRowBytes / 16;
            row = q * (64 / kLanes) + lane / kLanes;
            const int g = ((row & 1) << 1) ^ ((row >> 1 & 1) * 5);
            first = ((lane % kLanes >> 1) ^ g) * 16 + (lane & 1) * 8;
        }
    }

    // (widths along kOuter rows are multiples of 8; chunks beyond the end repeat the last, rows likewise)
    __device__ void init(const void *p, long ld, long start, long left, int wave, int lane)
    {
        base = reinterpret_cast<const char *>(p) + (ORDER == kInner ? start * ld : start) * 2;
        step = (ORDER == kInner ? 1 : ld) * kWideK * 2;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            int row, first;
            slot(i, wave, lane, row, first);
            if (ORDER == kInner) off[i] = (unsigned)((min((long)row, left - 1) * ld + first) * 2);
            else off[i] = (unsigned)((row * ld + min((long)first, left - 8)) * 2);
        }
    }

    // request I of kPer; lds: the stage's piece for this operand and wave
    template <int I> __device__ void issue(unsigned lds) const { request<I * 1024>(lds, off[I], next); }

    // the last, partial stage of a segment, through registers, zeros behind the last k
    __device__ void put_tail(char *lds, long kt, int left_k, int wave, int lane) const
    {
        const char *at = base + kt * step;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            int row, first;
            slot(i, wave, lane, row, first);
            const int inside = ORDER == kInner ? left_k - first : (row < left_k ? 8 : 0);
            uintx4 v = {0, 0, 0, 0};
            if (inside >= 8) {
                v = *reinterpret_cast<const uintx4_u *>(at + off[i]);
            } else if (inside > 0) {
                typedef T vec __attribute__((ext_vector_type(8)));
                vec e;
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = j < inside ? reinterpret_cast<const T *>(at + off[i])[min(j, inside - 1)] : (T)0.f;
                v = __builtin_bit_cast(uintx4, e);
            }
            *reinterpret_cast<uintx4 *>(lds + (wave * kPer + i) * 1024 + lane * 16) = v;
        }
    }
};

// A lane's operands of four 32-row groups, 16 of k at a time
template <class T, int ORDER, int R> struct StreamReader {
    static constexpr int kRowBytes = R * 2;
    unsigned at[ORDER == kInner ? 2 : 4];

    __device__ void init(const int (&first)[4], int lane)
    {
        const int l31 = lane & 31, h = lane >> 5;
        if (ORDER == kInner) {
#pragma unroll
            for (int s = 0; s < 2; ++s) at[s] = l31 * 64 + (((2 * s + h) ^ (l31 >> 2 & 3)) << 4);
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t)
                at[t] = Tile<T, kOuter, R>::outer_at(8 * h + (lane >> 2 & 3), first[t] + (lane & 16) + 4 * (lane & 3));
        }
    }

    __device__ uintx4 frag(const char *lds, int first, int t, int s) const
    {
        if (ORDER == kInner) return *reinterpret_cast<const uintx4 *>(lds + at[s] + first * 64);
        typedef __attribute__((address_space(3))) shortx4 lds_vec;
        const char *p = lds + at[t] + s * 16 * kRowBytes;
        const uintx2 lo = __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec *)(p)));
        const uintx2 hi = __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec *)(p + 4 * kRowBytes)));
        uintx4 v;
        v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
        return v;
    }
};

// A wave's accumulators to memory through its own piece of LDS, 32 rows at a time: written as they lie (a lane has four
// consecutive columns of one row), read back as runs of eight columns of consecutive rows - whole lines for the
// loads and stores, one copy of the epilogue's arithmetic, bias loaded once.  `lds` is the wave's:
// kEpilogueBytes; nobody else uses it.
constexpr int kEpilogueRow = 128 * 4 + 16;
constexpr int kEpilogueBytes = 32 * kEpilogueRow;

template <class T, bool GATED>
__device__ inline void store_quadrant(const Args &p, const floatx16 (&acc)[4][4], char *lds, int member, int split, long m0, int n0, int lane)
{
    constexpr bool EXACT = sizeof(T) == 4;
    const int l31 = lane & 31, h = lane >> 5;
    constexpr int kRuns = GATED ? 8 : 16, kRowsAtOnce = 64 / kRuns, kBatch = 4;     // runs of eight columns per row
    const int run = lane % kRuns, row0 = lane / kRuns;
    const int n = n0 + run * 8;
    const long left = p.n - n;
    auto put = [&](const floatx16 (&c)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                floatx4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = c[j][4 * q + e];
                *reinterpret_cast<floatx4 *>(lds + l31 * kEpilogueRow + (32 * j + 8 * q + 4 * h) * 4) = v;
            }
    };
    float bias[8] = {}, bias2[8] = {};
    if (left > 0 && p.bias[GATED ? 0 : member]) load8(reinterpret_cast<const T *>(p.bias[GATED ? 0 : member]) + n, left, bias);
    if (GATED && left > 0 && p.bias[1]) load8(reinterpret_cast<const T *>(p.bias[1]) + n, left, bias2);
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        if (i == 0) put(acc[0]);
        else if (i == 1) put(acc[1]);
        else if (i == 2) put(acc[2]);
        else put(acc[3]);
        if (left <= 0) continue;
        // four rows' loads at a time, then their arithmetic, then their stores: with one wave per SIMD nothing else
        // would cover the latency
#pragma unroll 1
        for (int r = row0; r < 32; r += kRowsAtOnce * kBatch) {
            const long m = m0 + 32 * i + r;
            float v[kBatch][8], v2[GATED ? kBatch : 1][8], res[kBatch][8];
            if (p.residual)
#pragma unroll
                for (int b = 0; b < kBatch; ++b)
                    load8(reinterpret_cast<const T *>(p.residual) + min(m + b * kRowsAtOnce, p.m - 1) * p.ldr + n, left, res[b]);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const float *from = reinterpret_cast<const float *>(lds + (r + b * kRowsAtOnce) * kEpilogueRow) + run * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[b][e] = from[e];
                    if (GATED) v2[b][e] = from[64 + e];
                }
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
                        store8(reinterpret_cast<T *>(p.pre[0]) + (m + b * kRowsAtOnce) * p.ldp + n, left, v[b]);
                        if (GATED) store8(reinterpret_cast<T *>(p.pre[1]) + (m + b * kRowsAtOnce) * p.ldp + n, left, v2[b]);
                    }
            if (p.act != FPN_ACT_NONE)
                for_activation(p.act, [&](auto tag) {
#pragma unroll
                    for (int b = 0; b < kBatch; ++b)
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[b][e] = activate<decltype(tag)::value, EXACT>(v[b][e]);
                });
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (GATED) v[b][e] *= v2[b][e];
                    if (p.residual) v[b][e] += res[b][e];
                }
                if (m + b * kRowsAtOnce < p.m) store8(reinterpret_cast<T *>(p.c[member]) + (m + b * kRowsAtOnce) * p.ldc + n, left, v[b]);
            }
        }
    }
}

template <class T, int ORDER_A, int ORDER_B, bool GATED>
__global__ __launch_bounds__(kThreads) void wide_product_kernel(const Args p)
{
    extern __shared__ char lds[];
    constexpr int kHalves = GATED ? 2 : 1, kCols = 256 / kHalves, kABytes = 256 * kWideK * 2;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave & 1, wn = wave >> 1;
    const Place at = place(p, blockIdx.x, gridDim.x);
    const long m0 = at.mt * 256;
    const int n0 = at.nt * kCols;

    int am[4], bn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) am[i] = wm * 128 + i * 32;
    // GATED: two column groups of the gate half, then the same columns of the up half
#pragma unroll
    for (int j = 0; j < 4; ++j) bn[j] = GATED ? wn * 64 + j % 2 * 32 : wn * 128 + j * 32;
    StreamReader<T, ORDER_A, 256> ra;
    StreamReader<T, ORDER_B, kCols> rb;
    ra.init(am, lane);
    rb.init(bn, lane);

    floatx16 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    const long full = p.k / kWideK;                         // whole stages of a segment
    const long first = at.split * p.tiles_per_split, last = min(first + p.tiles_per_split, full * p.segs);
    const unsigned lds0 = lds_address(lds);

    Stream<T, ORDER_A, 256> sa;
    Stream<T, ORDER_B, kCols> sb[kHalves];
    auto segment = [&](int s) {
        sa.init(p.a[s], p.lda[s], m0, p.m - m0, wave, lane);
        if (GATED) {
            sb[0].init(p.b[0], p.ldb[0], n0, p.n - n0, wave, lane);
            sb[kHalves - 1].init(p.b[1], p.ldb[1], n0, p.n - n0, wave, lane);
        } else {
            sb[0].init(p.b[s + at.member], p.ldb[s + at.member], n0, p.n - n0, wave, lane);
        }
    };
    // request Q of a wave's eight of a stage
    constexpr int kPerB = Stream<T, ORDER_B, kCols>::kPer;
    const unsigned lds_a = lds0 + wave * 4096, lds_b = lds0 + kABytes + wave * (kPerB * 1024);
    auto issue = [&](auto q, int stage) {
        constexpr int Q = decltype(q)::value;
        if constexpr (Q < 4) sa.template issue<Q>(lds_a + stage * kWideStage);
        else if constexpr (Q < 4 + kPerB) sb[0].template issue<Q - 4>(lds_b + stage * kWideStage);
        else sb[kHalves - 1].template issue<(Q - 4) % kPerB>(lds_b + kCols * kWideK * 2 + stage * kWideStage);
    };
    long asked = 0, most = 0;                               // stages whose requests are complete, and the last to ask for
    auto advance = [&] {
        const bool on = asked < most;
        ++asked;
        sa.next += on ? sa.step : 0;
#pragma unroll
        for (int g = 0; g < kHalves; ++g) sb[g].next += on ? sb[g].step : 0;
    };
    auto read_a = [&](const char *stage, int i, int s) { return ra.frag(stage, am[i], i, s); };
    auto read_b = [&](const char *stage, int j, int s) {
        return rb.frag(stage + kABytes + (GATED && j >= 2 ? kCols * kWideK * 2 : 0), bn[j], j, s);
    };
    // 16 of k: multiplies ca, cb while na, nb come from `stage`, and issues requests Q .. Q + 3 to stage `to`.  A wave
    // issues in order: an MFMA occupies its unit for 32 cycles, in which seven other instructions can go out, so the
    // reads and requests are dealt out among the MFMAs one by one (all in front of a group of four MFMAs cost 12 %);
    // no read is left for the last quarter, which covers their latency.
    auto step = [&](const uintx4 (&ca)[4], const uintx4 (&cb)[4], uintx4 (&na)[4], uintx4 (&nb)[4], const char *stage, int s,
                    auto q, int to) {
        constexpr int Q = decltype(q)::value;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            acc[i & 3][i >> 2] = multiply<T>(cb[i >> 2], ca[i & 3], acc[i & 3][i >> 2]);
            if (i == 0) na[0] = read_a(stage, 0, s);
            if (i == 1) na[1] = read_a(stage, 1, s);
            if (i == 2) issue(ActTag<Q>(), to);
            if (i == 3) na[2] = read_a(stage, 2, s);
            if (i == 4) na[3] = read_a(stage, 3, s);
            if (i == 5) nb[0] = read_b(stage, 0, s);
            if (i == 6) issue(ActTag<Q + 1>(), to);
            if (i == 7) nb[1] = read_b(stage, 1, s);
            if (i == 8) nb[2] = read_b(stage, 2, s);
            if (i == 9) nb[3] = read_b(stage, 3, s);
            if (i == 10) issue(ActTag<Q + 2>(), to);
            if (i == 12) issue(ActTag<Q + 3>(), to);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    uintx4 fa[2][4], fb[2][4];

    // segment by segment; a segment's whole stages in this split are [t0, t1)
    for (int s = 0; s < p.segs; ++s) {
        const long t0 = max(first - s * full, 0l), t1 = min(last - s * full, full);
        segment(s);
        if (t0 < t1) {
            const long n = t1 - t0;
            // Stage t + 4 is requested in two halves: behind the barrier of t, and in the first half of t + 1 (behind the
            // segment's end its last stage again, which nobody reads: a loop without branches, and counts that hold).
            // In flight at a barrier are the three stages ahead; the one read next must be there.
            most = n - 1;
            asked = 0;
            sa.next = sa.base + t0 * sa.step;
#pragma unroll
            for (int g = 0; g < kHalves; ++g) sb[g].next = sb[g].base + t0 * sb[g].step;
#pragma unroll
            for (int i = 0; i < kStages; ++i) {
                issue(ActTag<0>(), i);
                issue(ActTag<1>(), i);
                issue(ActTag<2>(), i);
                issue(ActTag<3>(), i);
                if (i == kStages - 1) break;
                issue(ActTag<4>(), i);
                issue(ActTag<5>(), i);
                issue(ActTag<6>(), i);
                issue(ActTag<7>(), i);
                advance();
            }
            arrive<20>();
#pragma unroll
            for (int i = 0; i < 4; ++i) { fa[0][i] = read_a(lds, i, 0); fb[0][i] = read_b(lds, i, 0); }
            int stage = 0;
            for (long t = 0; t < n; ++t) {
                step(fa[0], fb[0], fa[1], fb[1], lds + stage * kWideStage, 1, ActTag<4>(), (stage + 3) & 3);
                advance();
                arrive<16>();
                const int freed = stage;
                stage = (stage + 1) & 3;
                step(fa[1], fb[1], fa[0], fb[0], lds + stage * kWideStage, 0, ActTag<0>(), freed);
            }
            arrive<0>();
        }
        // what is left of k, with the last split
        const int left = (int)(p.k - full * kWideK);
        if (left && at.split == p.splits - 1) {
            __syncthreads();
            sa.put_tail(lds, full, left, wave, lane);
            sb[0].put_tail(lds + kABytes, full, left, wave, lane);
            if (GATED) sb[kHalves - 1].put_tail(lds + kABytes + kCols * kWideK * 2, full, left, wave, lane);
            __syncthreads();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
#pragma unroll
                for (int i = 0; i < 4; ++i) { fa[0][i] = read_a(lds, i, q); fb[0][i] = read_b(lds, i, q); }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[i][j] = multiply<T>(fb[0][j], fa[0][i], acc[i][j]);
            }
        }
        __syncthreads();
    }
    store_quadrant<T, GATED>(p, acc, lds + wave * kEpilogueBytes, at.member, at.split, m0 + wm * 128,
                             n0 + (GATED ? wn * 64 : wn * 128), lane);
}

#define FPN_FF_WIDE(A, B, G)                                                                                                  \
    do {                                                                                                                      \
        auto kern = wide_product_kernel<T, A, B, G>;                                                                          \
        const size_t bytes = kStages * kWideStage;                                                                            \
        static_assert(4 * kEpilogueBytes <= kStages * kWideStage, "the epilogue's pieces lie in the stages");                 \
        if (!allow_dynamic_lds(reinterpret_cast<const void *>(kern), bytes))                                                  \
            return fail(FPN_E_LAUNCH, "%zu bytes of LDS refused", bytes);                                                     \
        hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(kThreads), bytes, stream, p);                                   \
    } while (0)

template <class T> int launch_wide(const Args &p, int order_a, int order_b, bool gated, long blocks, hipStream_t stream)
{
    if (gated) {
        if (order_b == kOuter) FPN_FF_WIDE(kInner, kOuter, true);
        else FPN_FF_WIDE(kInner, kInner, true);
    } else if (order_a == kOuter) {
        FPN_FF_WIDE(kOuter, kOuter, false);
    } else if (order_b == kOuter) {
        FPN_FF_WIDE(kInner, kOuter, false);
    } else {
        FPN_FF_WIDE(kInner, kInner, false);
    }
    return check_launch("feed-forward product, wide");
}

}  // namespace ff
}  // namespace fpn
