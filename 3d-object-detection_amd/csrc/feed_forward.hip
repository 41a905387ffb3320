// The feed-forward operators' entry points: dense (act(x W + b) + r) and gated (act(x Wg + bg) * (x Wu + bu)),
// forward and backward, and the element-wise half of the backward pass.  The products are in feed_forward.h.
#include "feed_forward.h"

namespace fpn {
namespace ff {
namespace {

// ---- dpre and the bias gradients --------------------------------------------------------------------------------
//
// dense: d = dy act'(pre); gated: dg = dh u act'(g), du = dh act(g).  One pass: every input is read once, d written
// once, and the column sums (the bias gradients) are taken from the unrounded fp32 values on the way: a thread owns
// eight columns and every eighth row of its workgroup's rows, the eight row sums meet in LDS in a fixed order and the
// workgroups' sums in column_join_kernel - no atomics, so a step's gradients repeat bit for bit.
// d (dg, du) is rounded to the call's type because it is the operand of the next products, which the matrix units take in 16
// bits: dx and dw then carry two independent roundings of at most half a step, the result's and its factor's, so that their
// error is about sqrt 2 of one rounding's (1999 x 1091 x 515 fp16 against float64: 2.9e-4 of the norm, one rounding 2.1e-4).  Two
// products each, for d's high and low half, would avoid that at twice the time.  fp32 calls lose nothing.
// Bound by memory.
struct GradArgs {
    long rows;
    int n;
    const void *dy;          // of the kernel's DY type
    long lddy;
    const float *pre[2];     // null where the activation is the identity
    long ldp;
    int act;
    void *d[2];              // (rows, n), or null: column sums only
    long ldd;
    float *sums;             // (gridDim.y, 1 or 2, n), or null
    long rows_per_block;
};

template <class T, class DY, bool GATED> __global__ __launch_bounds__(kThreads) void grad_kernel(const GradArgs p)
{
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ float part[8][32][8];
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
    const int n = (int)blockIdx.x * 256 + c * 8;
    const long left = p.n - n;
    const long m0 = (long)blockIdx.y * p.rows_per_block, m1 = min(m0 + p.rows_per_block, p.rows);
    float sum[2][8] = {};
    if (left > 0) {
        for_activation(p.act, [&](auto tag) {
            constexpr int ACT = decltype(tag)::value;
            for (long m = m0 + r; m < m1; m += 8) {
                float d[8], g[8], u[8], du[8];
                load8(reinterpret_cast<const DY *>(p.dy) + m * p.lddy + n, left, d);
                if (GATED || ACT != FPN_ACT_NONE) load8(p.pre[0] + m * p.ldp + n, left, g);
                if (GATED) load8(p.pre[1] + m * p.ldp + n, left, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float value = 0.f;
                    const float slope = ACT == FPN_ACT_NONE && !GATED ? 1.f : activate_grad<ACT, EXACT>(g[i], value);
                    if (GATED) {
                        du[i] = d[i] * value;
                        d[i] = d[i] * u[i] * slope;
                        sum[1][i] += du[i];
                    } else {
                        d[i] *= slope;
                    }
                    sum[0][i] += d[i];
                }
                if (p.d[0]) {
                    store8(reinterpret_cast<T *>(p.d[0]) + m * p.ldd + n, left, d);
                    if (GATED) store8(reinterpret_cast<T *>(p.d[1]) + m * p.ldd + n, left, du);
                }
            }
        });
    }
    if (!p.sums) return;                                       // (uniform)
#pragma unroll
    for (int g = 0; g < (GATED ? 2 : 1); ++g) {
        if (g) __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) part[r][c][i] = sum[g][i];
        __syncthreads();
        if (r == 0 && left > 0) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = part[0][c][i];
                for (int s = 1; s < 8; ++s) v[i] += part[s][c][i];
            }
            store8(p.sums + ((long)blockIdx.y * (GATED ? 2 : 1) + g) * p.n + n, left, v);
        }
    }
}

// out[j][n] = sum over the workgroups of sums[.][j][n]: 32 columns a workgroup, every 32nd row a row of threads, eight of
// those loads at a time (one by one 512 rows took 12 us of latencies)
template <class T> __global__ __launch_bounds__(1024) void column_join_kernel(int n, int blocks, int planes, const float *sums, T *out0, T *out1)
{
    __shared__ float part[32][33];
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
    const int col = (int)blockIdx.x * 32 + c, j = blockIdx.y;
    float v = 0.f;
    if (col < n)
#pragma unroll 8
        for (int s = r; s < blocks; s += 32) v += sums[((long)s * planes + j) * n + col];
    part[r][c] = v;
    __syncthreads();
    if (r || col >= n) return;
#pragma unroll
    for (int s = 1; s < 32; ++s) v += part[s][c];
    (j ? out1 : out0)[col] = (T)v;
}

int grad_rows_grid(long rows, int n)
{
    // 2048 workgroups fill the chip eight deep; a workgroup takes at least 16 rows, and the second pass reads one
    // fp32 row per workgroup row, so that there are at most 512 of those
    const long cols = (n + 255) / 256;
    return (int)std::max(1l, std::min({(rows + 15) / 16, (2048 + cols - 1) / cols, 512l}));
}

template <class T>
int launch_column_join(int n, int blocks, bool gated, const float *sums, void *const (&sums_out)[2], hipStream_t stream)
{
    hipLaunchKernelGGL((column_join_kernel<T>), dim3((n + 31) / 32, gated ? 2 : 1), dim3(1024), 0, stream, n, blocks, gated ? 2 : 1,
                       sums, reinterpret_cast<T *>(sums_out[0]), reinterpret_cast<T *>(sums_out[1]));
    return check_launch("bias gradient");
}

template <class T>
int launch_grad(GradArgs p, bool gated, bool dy_float, void *const (&sums_out)[2], hipStream_t stream)
{
    const int gy = grad_rows_grid(p.rows, p.n), gx = (p.n + 255) / 256;
    p.rows_per_block = (p.rows + gy - 1) / gy;
    if (gated && dy_float) hipLaunchKernelGGL((grad_kernel<T, float, true>), dim3(gx, gy), dim3(kThreads), 0, stream, p);
    else if (gated) hipLaunchKernelGGL((grad_kernel<T, T, true>), dim3(gx, gy), dim3(kThreads), 0, stream, p);
    else hipLaunchKernelGGL((grad_kernel<T, T, false>), dim3(gx, gy), dim3(kThreads), 0, stream, p);
    int rc = check_launch("feed-forward gradient");
    if (rc != FPN_OK || !p.sums) return rc;
    return launch_column_join<T>(p.n, gy, gated, p.sums, sums_out, stream);
}

// ---- copies of operands whose rows do not consist of whole 16-byte chunks ------------------------------------------
//
// Such rows cannot be brought straight into LDS, and reading them at their own alignment costs the load path several
// passes per instruction.  Where there is enough to multiply they are copied once, rows padded with zeros to whole chunks
// (a dense product of 1999 x 1091 x 515 in 16 bits: 26 us without, 22 with; 4000 x 2001 x 1001: 55 and 39).
struct CopyArgs {
    struct { const void *from; void *to; long rows, ld, ldto; int cols; } of[3];
};

template <class T> __global__ __launch_bounds__(kThreads) void copy_kernel(const CopyArgs p)
{
    constexpr int E = Type<T>::kE;
    const auto &o = p.of[blockIdx.y];
    const long chunks = o.ldto / E, all = o.rows * chunks;
    for (long i = (long)blockIdx.x * kThreads + threadIdx.x; i < all; i += (long)gridDim.x * kThreads) {
        const long row = i / chunks;
        const int first = (int)(i - row * chunks) * E, inside = o.cols - first;
        const T *from = reinterpret_cast<const T *>(o.from) + row * o.ld + first;
        typedef T vec __attribute__((ext_vector_type(E)));
        vec v;
        if (inside >= E) {
            v = __builtin_bit_cast(vec, (uintx4)*reinterpret_cast<const uintx4_u *>(from));
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = j < inside ? from[j] : (T)0.f;
        }
        *reinterpret_cast<vec *>(reinterpret_cast<T *>(o.to) + row * o.ldto + first) = v;
    }
}

// ---- host side --------------------------------------------------------------------------------------------------

int element_size(int dtype) { return dtype == FPN_F32 ? 4 : 2; }

// the largest of the partial sums that a product's plans ask for, whatever its operands' alignment and b's order
size_t partial_bytes(int dtype, long m, int n, long k, int segs, int batch, bool gated, int order_a)
{
    size_t most = 0;
    for (int aligned = 0; aligned < 2; ++aligned)
        for (int order_b : {kInner, kOuter})
            if (order_a == kInner || order_b == kOuter)
                most = std::max(most, plan_product(dtype, m, n, k, segs, batch, gated, aligned, order_a, order_b).partial_bytes);
    return most;
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

Plan plan_of(int dtype, const Args &p, int order_a, int order_b, bool gated)
{
    bool aligned = true;
    for (int i = 0; i < p.segs; ++i)
        aligned = aligned && whole_chunks(p.a[i], order_a == kInner && p.m == 1 ? 0 : p.lda[i], order_a, p.load_m, element_size(dtype));
    for (int i = 0; i < std::max({p.segs, p.batch, gated ? 2 : 1}); ++i)
        aligned = aligned && whole_chunks(p.b[i], p.ldb[i], order_b, p.load_n, element_size(dtype));
    return plan_product(dtype, p.m, p.n, p.k, p.segs, p.batch, gated, aligned, order_a, order_b);
}

int run_product(int dtype, const Args &p, int order_a, int order_b, bool gated, float *partial, size_t partial_bytes, hipStream_t stream)
{
    const Plan plan = plan_of(dtype, p, order_a, order_b, gated);
    if (plan.partial_bytes && (!partial || plan.partial_bytes > partial_bytes))
        return fail(FPN_E_INVALID_ARG, "workspace of %zu bytes needed for partial sums, got %zu", plan.partial_bytes, partial ? partial_bytes : 0);
    if (dtype == FPN_F32) return launch_product<float>(p, order_a, order_b, gated, plan, partial, stream);
    if (dtype == FPN_BF16) return launch_product<__bf16>(p, order_a, order_b, gated, plan, partial, stream);
    return launch_product<_Float16>(p, order_a, order_b, gated, plan, partial, stream);
}

// Whether a product's grid fits one launch.  An entry point asks this of all its products before it launches anything.
int check_product(int dtype, const Args &p, int order_a, int order_b, bool gated)
{
    const Plan plan = plan_of(dtype, p, order_a, order_b, gated);
    if (plan.few) return FPN_OK;                  // (widths below 2^21: at most 2^29 threads)
    return check_grid(plan_blocks(p, gated, plan), plan.wide ? wide_threads(plan.bm) : kThreads);
}

constexpr int kStretchBytes = 64;             // of k per stage of the wide kernel
constexpr long kMostLd = (1l << 21) - 1;      // a tile's byte offsets inside an operand are 32 bits
// Rows times the widest row of floats are 2^61 bytes, and the largest workspace (dg, du, dh and the copies of x and dy: five
// such matrices) and every byte offset stay inside 64 bits.  No gradient of more rows would fit a card.
constexpr long kMostRows = 1l << 38;

int check_common(int dtype, long rows, int cin, int cout, int activation)
{
    FPN_REQUIRE(dtype == FPN_F32 || dtype == FPN_BF16 || dtype == FPN_F16, "dtype %d is none of FPN_F32, FPN_BF16, FPN_F16", dtype);
    FPN_REQUIRE(rows >= 0 && cin >= 1 && cout >= 1, "rows %ld, cin %d, cout %d: rows >= 0 and widths >= 1 are needed", rows, cin, cout);
    if (rows > kMostRows) return fail(FPN_E_UNSUPPORTED, "up to %ld rows are supported, got %ld", kMostRows, rows);
    FPN_REQUIRE(activation >= FPN_ACT_NONE && activation <= FPN_ACT_GELU_TANH, "unknown activation %d", activation);
    if (cin > kMostLd || cout > kMostLd) return fail(FPN_E_UNSUPPORTED, "widths up to %ld are supported, got %d and %d", kMostLd, cin, cout);
    return FPN_OK;
}

// a matrix argument: present, its rows apart by at least `width` (0: any stride, one row repeated) and addressable
int check_matrix(const char *name, const void *p, long ld, long width, int dtype, bool broadcast = false)
{
    FPN_REQUIRE(p, "%s is null", name);
    FPN_REQUIRE(reinterpret_cast<uintptr_t>(p) % element_size(dtype) == 0, "%s is not aligned to its elements", name);
    FPN_REQUIRE(ld >= width || (broadcast && ld == 0), "%s: row stride %ld is less than its %ld columns", name, ld, width);
    if (ld > kMostLd) return fail(FPN_E_UNSUPPORTED, "%s: row stride %ld is over %ld elements", name, ld, kMostLd);
    return FPN_OK;
}

int check_vector(const char *name, const void *p, int dtype)
{
    FPN_REQUIRE(!p || reinterpret_cast<uintptr_t>(p) % element_size(dtype) == 0, "%s is not aligned to its elements", name);
    return FPN_OK;
}

int check_workspace(const void *ws, size_t have, size_t need)
{
    FPN_REQUIRE(need == 0 || (ws && have >= need), "workspace of %zu bytes needed, got %zu", need, ws ? have : 0);
    FPN_REQUIRE(reinterpret_cast<uintptr_t>(ws) % 16 == 0, "workspace must be 16-byte aligned");
    return FPN_OK;
}

#define FPN_FF_TRY(call)                \
    do {                                \
        const int rc_ = (call);         \
        if (rc_ != FPN_OK) return rc_;  \
    } while (0)

// The parts of a backward pass' workspace: dpre (one matrix, or two where gated), the workgroups' column sums, and
// the partial sums of dx and dw, which run one after the other
struct GradSpace {
    size_t d, sums, dh, partial, copies, total;
};
// a row length in whole chunks
long padded(int dtype, long cols)
{
    const int e = 16 / element_size(dtype);
    return (cols + e - 1) / e * e;
}

// whether operands with ragged rows are copied: a copy's launch and traffic (4 us and more) against what the pipelined
// kernel saves, which takes half the time from about 10^8 operations on (an output narrower than its tile counts as 64
// columns: 40189 x 1280 x 3 bf16 90 us without copies of the weights, 23 with; 40189 x 1281 x 3, where x is copied too, 96 and
// 56; but 70000 x 131 x 37 24 either way and its weights' gradient 29 and 38, so that a narrow one wants a longer sum)
bool worth_copies(long rows, int cin, int cout)
{
    return rows > 64 && cin >= (cout >= 64 ? 64 : 192) && 2.0 * rows * cin * std::max(cout, 64) >= 1e8;
}

// the bytes of copies of a matrix in either storage order
size_t copy_bytes(int dtype, long rows, long cols) { return align256((size_t)rows * padded(dtype, cols) * element_size(dtype)); }
size_t weight_copy_bytes(int dtype, int cin, int cout) { return std::max(copy_bytes(dtype, cin, cout), copy_bytes(dtype, cout, cin)); }

// A matrix of a call, which may be replaced by its copy.  `wide`: what may be read of its rows.
struct Matrix {
    const void *p;
    long ld, rows;
    int cols;
    long wide;
};

// Collects the copies that a call makes, and makes them in one launch
struct Copies {
    CopyArgs args = {};
    int count = 0;
    char *at;
    size_t left;
    int dtype;

    Copies(int dtype_, void *space, size_t bytes) : at(reinterpret_cast<char *>(space)), left(space ? bytes : 0), dtype(dtype_) {}

    // outer: the matrix is read along its rows' direction in chunks (kOuter), so that its width counts too
    void take(Matrix &m, bool outer)
    {
        const int e = element_size(dtype);
        if (reinterpret_cast<uintptr_t>(m.p) % 16 == 0 && m.ld * e % 16 == 0 && (!outer || m.wide * e % 16 == 0)) return;
        const size_t bytes = copy_bytes(dtype, m.rows, m.cols);
        if (bytes > left || count == 3) return;                        // (no room: the kernel that reads any rows takes it)
        const long ld = padded(dtype, m.cols);
        args.of[count++] = {m.p, at, m.rows, m.ld, ld, m.cols};
        m = {at, ld, m.rows, m.cols, ld};
        at += bytes;
        left -= bytes;
    }

    int make(hipStream_t stream)
    {
        if (!count) return FPN_OK;
        long most = 0;
        for (int i = 0; i < count; ++i) most = std::max(most, args.of[i].rows * args.of[i].ldto);
        const long blocks = std::min(2048l, (most * element_size(dtype) / 16 + kThreads - 1) / kThreads);
        const dim3 grid((unsigned)blocks, count);
        if (dtype == FPN_F32) hipLaunchKernelGGL((copy_kernel<float>), grid, dim3(kThreads), 0, stream, args);
        else if (dtype == FPN_BF16) hipLaunchKernelGGL((copy_kernel<__bf16>), grid, dim3(kThreads), 0, stream, args);
        else hipLaunchKernelGGL((copy_kernel<_Float16>), grid, dim3(kThreads), 0, stream, args);
        return check_launch("copy of ragged operands");
    }
};

Matrix weights(const void *p, long ld, int cin, int cout, int transposed)
{
    return transposed ? Matrix{p, ld, cout, cin, cin} : Matrix{p, ld, cin, cout, cout};
}

// (down: the width of the block's result where dh is formed from its gradient, else 0; whole: no operand will be copied)
GradSpace grad_space(int dtype, long rows, int cin, int n, bool gated, bool with_d, bool whole, int down = 0)
{
    GradSpace s;
    const int planes = gated ? 2 : 1;
    s.d = with_d ? align256((size_t)rows * padded(dtype, n) * element_size(dtype)) * planes : 0;
    s.sums = align256((size_t)std::max<long>(grad_rows_grid(rows, n), down ? (rows + 255) / 256 * 8 : 0) * planes * n * sizeof(float));
    s.dh = down ? align256((size_t)rows * n * sizeof(float)) : 0;
    s.partial = align256(std::max({partial_bytes(dtype, rows, cin, n, planes, 1, false, kInner),
                                   partial_bytes(dtype, cin, n, rows, 1, planes, false, kOuter),
                                   partial_bytes(dtype, n, cin, rows, 1, 1, false, kOuter)}));
    if (down) s.partial = std::max(s.partial, align256(partial_bytes(dtype, rows, n, down, 1, 1, false, kInner)));
    s.copies = 0;
    if (!whole && worth_copies(rows, cin, n))
        s.copies = copy_bytes(dtype, rows, cin) + planes * weight_copy_bytes(dtype, cin, n) + (with_d ? 0 : copy_bytes(dtype, rows, n));
    if (!whole && down && worth_copies(rows, down, n)) s.copies += copy_bytes(dtype, rows, down) + weight_copy_bytes(dtype, n, down);
    s.total = s.d + s.sums + s.dh + s.partial + s.copies;
    return s;
}

Args product(long m, int n, long k)
{
    Args p = {};
    p.m = m;
    p.n = n;
    p.k = k;
    p.segs = 1;
    p.batch = 1;
    p.act = FPN_ACT_NONE;
    p.load_m = m;
    p.load_n = n;
    return p;
}

// dw = x^T d for one or two d, in the weights' own storage order: one product or two
int weight_products(const Matrix &x, const Matrix (&d)[2], int members, void *const (&dw)[2], long lddw, int transposed, Args (&out)[2])
{
    if (!transposed) {
        Args &p = out[0] = product(x.cols, d[0].cols, x.rows);
        p.load_m = x.wide;
        p.load_n = (int)d[0].wide;
        p.a[0] = x.p;
        p.lda[0] = x.ld;
        p.batch = members;
        for (int i = 0; i < members; ++i) { p.b[i] = d[i].p; p.ldb[i] = d[i].ld; p.c[i] = dw[i]; }
        p.ldc = lddw;
        return 1;
    }
    // held (out,in): the operands change places (one product each, x is the b side of both)
    for (int i = 0; i < members; ++i) {
        Args &p = out[i] = product(d[i].cols, x.cols, x.rows);
        p.load_m = d[i].wide;
        p.load_n = (int)x.wide;
        p.a[0] = d[i].p;
        p.lda[0] = d[i].ld;
        p.b[0] = x.p;
        p.ldb[0] = x.ld;
        p.c[0] = dw[i];
        p.ldc = lddw;
    }
    return members;
}

// the operands of a forward product (or two, gated)
void set_operands(Args &p, const Matrix &x, const Matrix *w, int count)
{
    p.a[0] = x.p;
    p.lda[0] = x.ld;
    for (int i = 0; i < count; ++i) {
        p.b[i] = w[i].p;
        p.ldb[i] = w[i].ld;
    }
}

int run_grad(int dtype, const GradArgs &p, bool gated, bool dy_float, void *const (&sums_out)[2], hipStream_t stream)
{
    if (dtype == FPN_F32) return launch_grad<float>(p, gated, dy_float, sums_out, stream);
    if (dtype == FPN_BF16) return launch_grad<__bf16>(p, gated, dy_float, sums_out, stream);
    return launch_grad<_Float16>(p, gated, dy_float, sums_out, stream);
}

int run_column_join(int dtype, int n, int blocks, const float *sums, void *const (&out)[2], hipStream_t stream)
{
    if (dtype == FPN_F32) return launch_column_join<float>(n, blocks, true, sums, out, stream);
    if (dtype == FPN_BF16) return launch_column_join<__bf16>(n, blocks, true, sums, out, stream);
    return launch_column_join<_Float16>(n, blocks, true, sums, out, stream);
}

}  // namespace

namespace {

// The time of a launch of `tiles` workgroups of one shape, in us, from what these took on a 256-CU chip: a stage of k (32
// sixteen-bit elements, 16 floats) with workgroups on few CUs, with one on every CU and with `per_cu` on every CU - the
// sixteen-bit shapes are bound by what a CU receives from L2, 60 to 80 bytes/ns -, and what a round of workgroups costs besides (first loads,
// epilogue).  Measured, bf16, k not split, us:   large  medium  small  tiny
//   8192 x 4096 x 4096                             230     272    287   414
//   4096 x 2048 x 2048                              51      41     42    58
//   2048 x 2048 x 2048                              49      36     27    32
//   1024 x 1024 x 1024                              28      18     14    10
//   4096 x 8192 x 1024                             148     110     79   102
struct Pace { int bm, bn, per_cu; double few, one, full, round; };
constexpr Pace kWide[] = {
    {256, 256, 1, 0.54, 0.82, 0.82, 10.0},
    {256, 128, 1, 0.40, 0.52, 0.52, 6.0},
    {128, 128, 2, 0.25, 0.30, 0.53, 6.2},
    {64, 64, 4, 0.18, 0.19, 0.41, 4.5},
};
// fp32: bound by its matrix rate, so the smallest tiles that keep it fed (us, k not split: small 265, tiny 270 at
// 1024 x 4096 x 4096, 68 and 25 at 1024 x 1024 x 1024)
constexpr Pace kWideF32[] = {
    {128, 128, 2, 0.97, 1.02, 2.00, 6.0},
    {64, 64, 4, 0.29, 0.31, 1.02, 5.5},
};

double launch_time(const Pace &p, long tiles, double stages, int cus)
{
    const long at_once = (long)cus * p.per_cu, rounds = tiles / at_once, rest = tiles - rounds * at_once;
    double us = rounds * (p.full * stages + p.round);
    if (rest > cus) us += (p.one + (p.full - p.one) * ((rest - 1) / cus) / (p.per_cu - 1)) * stages + p.round;
    else if (rest) us += (p.few + (p.one - p.few) * rest / cus) * stages + p.round;
    return us;
}

// writing and reading the partial sums of a split, and the join's launch
double join_time(double bytes) { return 5.0 + bytes / 4e6; }

Plan make_plan(int dtype, long m, int n, long k, int segs, int batch, bool gated, bool aligned, int order_a, int order_b, int cus)
{
    Plan p = {};
    auto tiles = [&](int bm, int bn) { return (m + bm - 1) / bm * ((n + (gated ? bn / 2 : bn) - 1) / (gated ? bn / 2 : bn)) * batch; };
    const double plane = (double)batch * (gated ? 2 : 1) * m * n * sizeof(float);
    constexpr double kMostPartial = 128 << 20;
    // Few rows: the kernel that streams the weights, measured (graphs of calls, bf16, us) against the wide kernel with k split:
    // 1024 x 512 4.6 : 9 at 1 row, 6 : 9 at 64; 4096 x 4096 held (out,in) 8.2 : 15 at 1 row, 12.6 : 14.3 at 32, 17.5 : 15.5 at 64,
    // held (in,out) 12.2 : 14.8, 14.3 : 14.2, 17.8 : 15.8; gated 17.5 : 23 and 25 : 27 at 1 row, 20 : 22 and 26 : 23 at 16.
    const bool big = (double)k * n * (gated ? 2 : 1) * element_size(dtype) > 8e6;
    if (aligned && m > 0 && segs == 1 && batch == 1 && order_a == kInner &&
        m <= (dtype == FPN_F32 || !big ? 64 : !gated ? 32 : order_b == kInner ? 16 : 4)) {
        p.few = true;
        p.bm = m <= 16 ? 1 : m <= 32 ? 2 : 4;
        // Columns per workgroup, in 16.  What a CU has on its way is counted in cache lines, so row-major weights want whole
        // lines (64 columns, 32 floats) and, where that leaves CUs without work, k split over workgroups; weights held (out,in)
        // and small ones want as many workgroups as there are CUs.
        p.splits = 1;
        const int line = dtype == FPN_F32 ? 2 : 4;
        if (n >= 32 * cus || (order_b == kOuter && !big && dtype != FPN_F32)) p.bn = 2;
        else if (order_b == kOuter && big && !(gated && p.bm == 4)) {
            p.bn = line;
            while (p.splits < 4 && 2l * p.splits * ((n + 16 * line - 1) / (16 * line)) <= cus) p.splits *= 2;
        } else p.bn = 1;
        p.partial_bytes = p.splits > 1 ? (size_t)(plane * p.splits) : 0;
        return p;
    }
    if (aligned && m > 0) {
        const long full = k / (kStretchBytes / element_size(dtype)) * segs;
        double best = 0;
        const Pace *const first = dtype == FPN_F32 ? kWideF32 : kWide;
        const Pace *const last = first + (dtype == FPN_F32 ? sizeof kWideF32 : sizeof kWide) / sizeof(Pace);
        for (const Pace *q = first; q < last; ++q)
            for (long splits = 1; splits <= 256; splits *= 2) {
                const long each = std::max(1l, (full + splits - 1) / splits);
                if (splits > 1 && (each < 8 || plane * splits > kMostPartial)) break;
                const double us = launch_time(*q, tiles(q->bm, q->bn) * splits, (double)each, cus) + (splits > 1 ? join_time(plane * splits) : 0);
                if (!p.wide || us < best) {
                    best = us;
                    p.wide = true;
                    p.bm = q->bm;
                    p.bn = q->bn;
                    p.tiles_per_split = each;
                    p.splits = (int)std::max(1l, (full + each - 1) / each);
                }
            }
    } else {
        const int bk = kTileBytes / element_size(dtype);
        const long kt = (k + bk - 1) / bk * segs;
        p.bm = m > 64 && tiles(128, 128) >= 256 ? 128 : 64;
        p.bn = 128;
        const long t = std::max(1l, tiles(p.bm, p.bn));
        // too few tiles for the chip: k is split so that about 512 workgroups run, each with at least four k tiles
        long splits = t >= 256 ? 1 : std::max(1l, std::min({512 / t, kt / 4, 256l, (long)(kMostPartial / std::max(plane, 1.0))}));
        p.tiles_per_split = std::max(1l, (kt + splits - 1) / splits);
        p.splits = (int)std::max(1l, (kt + p.tiles_per_split - 1) / p.tiles_per_split);
    }
    p.partial_bytes = p.splits > 1 ? (size_t)(plane * p.splits) : 0;
    return p;
}

}  // namespace

// A plan depends on the sizes only; a call asks for a few of them, so each thread keeps the last ones it made.
Plan plan_product(int dtype, long m, int n, long k, int segs, int batch, bool gated, bool aligned, int order_a, int order_b)
{
    struct Entry { long key[4]; Plan plan; };
    constexpr int kKept = 64;
    static thread_local Entry kept[kKept] = {};
    const int cus = current_device_cus() > 0 ? current_device_cus() : 256;
    const long key[4] = {m, k, n, 1 + (dtype | segs << 4 | batch << 8 | (gated ? 1 << 12 : 0) | (aligned ? 1 << 13 : 0) | order_a << 14 | order_b << 15 |
                                       (long)cus << 16)};
    Entry &e = kept[(unsigned long)(key[0] * 31 + key[1] * 17 + key[2] * 7 + key[3] * 3 + (key[3] >> 13)) % kKept];
    if (!std::equal(key, key + 4, e.key)) {
        e.plan = make_plan(dtype, m, n, k, segs, batch, gated, aligned, order_a, order_b, cus);
        std::copy(key, key + 4, e.key);
    }
    return e.plan;
}

}  // namespace ff
}  // namespace fpn

using namespace fpn;
using namespace fpn::ff;

extern "C" {

size_t fpn_dense_workspace_bytes(int dtype, long rows, int cin, int cout, int whole)
{
    if (check_common(dtype, rows, cin, cout, FPN_ACT_NONE) != FPN_OK) return 0;
    const size_t partial = partial_bytes(dtype, rows, cout, cin, 1, 1, false, kInner);
    if (whole || !worth_copies(rows, cin, cout)) return partial;
    return align256(partial) + copy_bytes(dtype, rows, cin) + weight_copy_bytes(dtype, cin, cout);
}

int fpn_dense(int dtype, long rows, int cin, int cout, const void *x, long ldx, const void *w, long ldw, int w_transposed,
              const void *bias, int activation, const void *residual, long ldr, void *y, long ldy, float *pre, long ldp,
              void *workspace, size_t workspace_bytes, void *stream)
{
    FPN_FF_TRY(check_common(dtype, rows, cin, cout, activation));
    if (rows == 0) return FPN_OK;
    FPN_FF_TRY(check_matrix("x", x, ldx, cin, dtype, true));
    FPN_FF_TRY(check_matrix("w", w, ldw, w_transposed ? cin : cout, dtype));
    FPN_FF_TRY(check_matrix("y", y, ldy, cout, dtype));
    FPN_FF_TRY(check_vector("bias", bias, dtype));
    if (residual) FPN_FF_TRY(check_matrix("residual", residual, ldr, cout, dtype, true));
    if (pre) FPN_FF_TRY(check_matrix("pre", pre, ldp, cout, FPN_F32));
    FPN_FF_TRY(check_workspace(workspace, workspace_bytes, 0));
    const int order_b = w_transposed ? kInner : kOuter;
    const hipStream_t st = as_stream(stream);
    Matrix mx = {x, ldx, rows, cin, cin}, mw = weights(w, ldw, cin, cout, w_transposed);
    size_t partial_space = workspace_bytes;
    Copies copies(dtype, nullptr, 0);
    if (worth_copies(rows, cin, cout)) {
        const size_t partial = align256(partial_bytes(dtype, rows, cout, cin, 1, 1, false, kInner));
        if (workspace && workspace_bytes > partial) {
            copies = Copies(dtype, reinterpret_cast<char *>(workspace) + partial, workspace_bytes - partial);
            copies.take(mx, false);
            copies.take(mw, order_b == kOuter);
            partial_space = partial;
        }
    }
    Args p = product(rows, cout, cin);
    set_operands(p, mx, &mw, 1);
    if (order_b == kOuter) p.load_n = (int)mw.wide;
    p.bias[0] = bias;
    p.act = activation;
    p.residual = residual;
    p.ldr = ldr;
    p.c[0] = y;
    p.ldc = ldy;
    p.pre[0] = pre;
    p.ldp = ldp;
    FPN_FF_TRY(check_product(dtype, p, kInner, order_b, false));
    FPN_FF_TRY(copies.make(st));
    return run_product(dtype, p, kInner, order_b, false, reinterpret_cast<float *>(workspace), partial_space, st);
}

size_t fpn_dense_grad_workspace_bytes(int dtype, long rows, int cin, int cout, int activation, int whole)
{
    if (check_common(dtype, rows, cin, cout, activation) != FPN_OK) return 0;
    return grad_space(dtype, rows, cin, cout, false, activation != FPN_ACT_NONE, whole).total;
}

int fpn_dense_grad(int dtype, long rows, int cin, int cout, const void *dy, long lddy, const void *x, long ldx, const void *w,
                   long ldw, int w_transposed, const float *pre, long ldp, int activation, void *dx, long lddx, void *dw, long lddw,
                   void *dbias, void *workspace, size_t workspace_bytes, void *stream)
{
    FPN_FF_TRY(check_common(dtype, rows, cin, cout, activation));
    const bool act = activation != FPN_ACT_NONE;
    if (rows > 0) {
        FPN_FF_TRY(check_matrix("dy", dy, lddy, cout, dtype));
        if (act) FPN_FF_TRY(check_matrix("pre", pre, ldp, cout, FPN_F32));
        if (dw) FPN_FF_TRY(check_matrix("x", x, ldx, cin, dtype, true));
        if (dx) FPN_FF_TRY(check_matrix("w", w, ldw, w_transposed ? cin : cout, dtype));
        if (dx) FPN_FF_TRY(check_matrix("dx", dx, lddx, cin, dtype));
    }
    if (dw) FPN_FF_TRY(check_matrix("dw", dw, lddw, w_transposed ? cin : cout, dtype));
    FPN_FF_TRY(check_vector("dbias", dbias, dtype));
    // (with a smaller workspace than ragged operands' copies take, the products read them as they are)
    GradSpace space = grad_space(dtype, rows, cin, cout, false, act, true);
    FPN_FF_TRY(check_workspace(workspace, workspace_bytes, space.total));
    char *ws = reinterpret_cast<char *>(workspace);
    float *partial = reinterpret_cast<float *>(ws + space.d + space.sums + space.dh);
    const hipStream_t st = as_stream(stream);

    Matrix mx = {x, ldx, rows, cin, cin}, mw = weights(w, ldw, cin, cout, w_transposed), md[2] = {{dy, lddy, rows, cout, cout}, {}};
    Copies copies(dtype, ws + space.total, workspace_bytes - space.total);
    if (worth_copies(rows, cin, cout)) {
        if (dw) copies.take(mx, true);
        if (dx) copies.take(mw, w_transposed);
        if (!act) copies.take(md[0], dw);
    }
    GradArgs g = {};
    g.rows = rows;
    g.n = cout;
    g.dy = dy;
    g.lddy = lddy;
    g.pre[0] = pre;
    g.ldp = ldp;
    g.act = activation;
    if (act) {
        const long ldd = padded(dtype, cout);
        g.d[0] = ws;
        g.ldd = ldd;
        md[0] = {ws, ldd, rows, cout, ldd};
    }
    g.sums = dbias ? reinterpret_cast<float *>(ws + space.d) : nullptr;
    Args px = product(rows, cin, cout), pw[2];
    const int order_x = w_transposed ? kOuter : kInner;
    const bool want_x = dx && rows > 0;
    if (want_x) {
        set_operands(px, md[0], &mw, 1);
        if (w_transposed) px.load_n = (int)mw.wide;
        px.c[0] = dx;
        px.ldc = lddx;
        FPN_FF_TRY(check_product(dtype, px, kInner, order_x, false));
    }
    void *const dw_out[2] = {dw, nullptr};
    if (dw) {
        weight_products(mx, md, 1, dw_out, lddw, w_transposed, pw);
        FPN_FF_TRY(check_product(dtype, pw[0], kOuter, kOuter, false));
    }

    FPN_FF_TRY(copies.make(st));
    if (act || dbias) {
        void *const out[2] = {dbias, nullptr};
        FPN_FF_TRY(run_grad(dtype, g, false, false, out, st));
    }
    if (want_x) FPN_FF_TRY(run_product(dtype, px, kInner, order_x, false, partial, space.partial, st));
    if (dw) FPN_FF_TRY(run_product(dtype, pw[0], kOuter, kOuter, false, partial, space.partial, st));
    return FPN_OK;
}

size_t fpn_gated_workspace_bytes(int dtype, long rows, int cin, int cout, int whole)
{
    if (check_common(dtype, rows, cin, cout, FPN_ACT_NONE) != FPN_OK) return 0;
    const size_t partial = partial_bytes(dtype, rows, cout, cin, 1, 1, true, kInner);
    if (whole || !worth_copies(rows, cin, cout)) return partial;
    return align256(partial) + copy_bytes(dtype, rows, cin) + 2 * weight_copy_bytes(dtype, cin, cout);
}

int fpn_gated(int dtype, long rows, int cin, int cout, const void *x, long ldx, const void *w_gate, long ldg, const void *w_up, long ldu,
              int w_transposed, const void *bias_gate, const void *bias_up, int activation, void *h, long ldh, float *gate, float *up,
              long ldp, void *workspace, size_t workspace_bytes, void *stream)
{
    FPN_FF_TRY(check_common(dtype, rows, cin, cout, activation));
    FPN_REQUIRE(!gate == !up, "gate and up are kept together or not at all");
    if (rows == 0) return FPN_OK;
    FPN_FF_TRY(check_matrix("x", x, ldx, cin, dtype, true));
    FPN_FF_TRY(check_matrix("w_gate", w_gate, ldg, w_transposed ? cin : cout, dtype));
    FPN_FF_TRY(check_matrix("w_up", w_up, ldu, w_transposed ? cin : cout, dtype));
    FPN_FF_TRY(check_matrix("h", h, ldh, cout, dtype));
    FPN_FF_TRY(check_vector("bias_gate", bias_gate, dtype));
    FPN_FF_TRY(check_vector("bias_up", bias_up, dtype));
    if (gate) FPN_FF_TRY(check_matrix("gate", gate, ldp, cout, FPN_F32));
    if (up) FPN_FF_TRY(check_matrix("up", up, ldp, cout, FPN_F32));
    FPN_FF_TRY(check_workspace(workspace, workspace_bytes, 0));
    const int order_b = w_transposed ? kInner : kOuter;
    const hipStream_t st = as_stream(stream);
    Matrix mx = {x, ldx, rows, cin, cin}, mw[2] = {weights(w_gate, ldg, cin, cout, w_transposed), weights(w_up, ldu, cin, cout, w_transposed)};
    size_t partial_space = workspace_bytes;
    Copies copies(dtype, nullptr, 0);
    if (worth_copies(rows, cin, cout)) {
        const size_t partial = align256(partial_bytes(dtype, rows, cout, cin, 1, 1, true, kInner));
        if (workspace && workspace_bytes > partial) {
            copies = Copies(dtype, reinterpret_cast<char *>(workspace) + partial, workspace_bytes - partial);
            copies.take(mx, false);
            copies.take(mw[0], order_b == kOuter);
            copies.take(mw[1], order_b == kOuter);
            partial_space = partial;
        }
    }
    Args p = product(rows, cout, cin);
    set_operands(p, mx, mw, 2);
    if (order_b == kOuter) p.load_n = (int)std::min(mw[0].wide, mw[1].wide);
    p.bias[0] = bias_gate;
    p.bias[1] = bias_up;
    p.act = activation;
    p.c[0] = h;
    p.ldc = ldh;
    p.pre[0] = gate;
    p.pre[1] = up;
    p.ldp = ldp;
    FPN_FF_TRY(check_product(dtype, p, kInner, order_b, true));
    FPN_FF_TRY(copies.make(st));
    return run_product(dtype, p, kInner, order_b, true, reinterpret_cast<float *>(workspace), partial_space, st);
}

size_t fpn_gated_grad_workspace_bytes(int dtype, long rows, int cin, int cout, int cdown, int whole)
{
    if (check_common(dtype, rows, cin, cout, FPN_ACT_NONE) != FPN_OK || cdown < 0 || cdown > kMostLd) return 0;
    return grad_space(dtype, rows, cin, cout, true, true, whole, cdown).total;
}

int fpn_gated_grad(int dtype, long rows, int cin, int cout, int cdown, const void *dh, long lddh, const void *w_down, long ldd,
                   int down_transposed, const void *x, long ldx, const void *w_gate, long ldg, const void *w_up, long ldu,
                   int w_transposed, const float *gate, const float *up, long ldp, int activation, void *dx, long lddx, void *dw_gate,
                   void *dw_up, long lddw, void *dbias_gate, void *dbias_up, void *workspace, size_t workspace_bytes, void *stream)
{
    FPN_FF_TRY(check_common(dtype, rows, cin, cout, activation));
    FPN_REQUIRE(cdown >= 0, "cdown %d is negative", cdown);
    if (cdown > kMostLd) return fail(FPN_E_UNSUPPORTED, "widths up to %ld are supported, got %d", kMostLd, cdown);
    FPN_REQUIRE(!dw_gate == !dw_up && !dbias_gate == !dbias_up, "the gradients of gate and up are wanted together or not at all");
    if (rows > 0) {
        FPN_FF_TRY(check_matrix("dh", dh, lddh, cdown ? cdown : cout, dtype));
        if (cdown) FPN_FF_TRY(check_matrix("w_down", w_down, ldd, down_transposed ? cout : cdown, dtype));
        FPN_FF_TRY(check_matrix("gate", gate, ldp, cout, FPN_F32));
        FPN_FF_TRY(check_matrix("up", up, ldp, cout, FPN_F32));
        if (dw_gate) FPN_FF_TRY(check_matrix("x", x, ldx, cin, dtype, true));
        if (dx) {
            FPN_FF_TRY(check_matrix("w_gate", w_gate, ldg, w_transposed ? cin : cout, dtype));
            FPN_FF_TRY(check_matrix("w_up", w_up, ldu, w_transposed ? cin : cout, dtype));
            FPN_FF_TRY(check_matrix("dx", dx, lddx, cin, dtype));
        }
    }
    if (dw_gate) {
        FPN_FF_TRY(check_matrix("dw_gate", dw_gate, lddw, w_transposed ? cin : cout, dtype));
        FPN_FF_TRY(check_matrix("dw_up", dw_up, lddw, w_transposed ? cin : cout, dtype));
    }
    FPN_FF_TRY(check_vector("dbias_gate", dbias_gate, dtype));
    FPN_FF_TRY(check_vector("dbias_up", dbias_up, dtype));
    // (with a smaller workspace than ragged operands' copies take, the products read them as they are)
    const GradSpace space = grad_space(dtype, rows, cin, cout, true, true, true, cdown);
    FPN_FF_TRY(check_workspace(workspace, workspace_bytes, space.total));
    char *ws = reinterpret_cast<char *>(workspace);
    float *partial = reinterpret_cast<float *>(ws + space.d + space.sums + space.dh);
    const hipStream_t st = as_stream(stream);
    const int order_down = down_transposed ? kOuter : kInner;

    Matrix mx = {x, ldx, rows, cin, cin}, mw[2] = {weights(w_gate, ldg, cin, cout, w_transposed), weights(w_up, ldu, cin, cout, w_transposed)};
    Matrix mdy = {dh, lddh, rows, cdown, cdown}, mdown = weights(w_down, ldd, cout, cdown, down_transposed);
    Copies copies(dtype, ws + space.total, workspace_bytes - space.total);
    if (worth_copies(rows, cin, cout)) {
        if (dw_gate) copies.take(mx, true);
        if (dx) copies.take(mw[0], w_transposed);
        if (dx) copies.take(mw[1], w_transposed);
    }
    const bool down = cdown && rows > 0;
    Copies more(dtype, copies.at, copies.left);
    if (down && worth_copies(rows, cdown, cout)) {
        more.take(mdy, false);
        more.take(mdown, order_down == kOuter);
    }

    const long ldd_own = padded(dtype, cout);
    GradArgs g = {};
    g.rows = rows;
    g.n = cout;
    g.dy = dh;
    g.lddy = lddh;
    g.pre[0] = gate;
    g.pre[1] = up;
    g.ldp = ldp;
    g.act = activation;
    g.d[0] = ws;
    g.d[1] = ws + space.d / 2;
    g.ldd = ldd_own;
    const Matrix md[2] = {{g.d[0], ldd_own, rows, cout, ldd_own}, {g.d[1], ldd_own, rows, cout, ldd_own}};
    g.sums = dbias_gate ? reinterpret_cast<float *>(ws + space.d) : nullptr;
    void *const sums_out[2] = {dbias_gate, dbias_up};
    Args ph = product(rows, cout, cdown), px = product(rows, cin, cout), pw[2];
    Plan plan_h = {};
    bool fused = false;                           // dg and du straight from the product that forms dh
    if (down) {                                   // dh = dy w_down^T, never rounded to 16 bits
        set_operands(ph, mdy, &mdown, 1);
        if (order_down == kOuter) ph.load_n = (int)mdown.wide;
        plan_h = plan_of(dtype, ph, kInner, order_down, false);
        fused = plan_h.wide && plan_h.splits == 1;
        if (fused) {
            ph.c[0] = g.d[0];
            ph.c[1] = g.d[1];
            ph.ldc = ldd_own;
            ph.act = activation;
            ph.gate = gate;
            ph.up = up;
            ph.ldp = ldp;
            ph.sums = g.sums;
        } else {
            ph.c[0] = ws + space.d + space.sums;
            ph.ldc = cout;
            ph.c_float = true;
            g.dy = ph.c[0];
            g.lddy = cout;
        }
        FPN_FF_TRY(check_product(dtype, ph, kInner, order_down, false));
    }
    const int order_x = w_transposed ? kOuter : kInner;
    const bool want_x = dx && rows > 0;
    if (want_x) {                                 // dg Wg^T + du Wu^T: one sum over both
        px.segs = 2;
        set_operands(px, md[0], mw, 2);
        px.a[1] = md[1].p;
        px.lda[1] = md[1].ld;
        if (w_transposed) px.load_n = (int)std::min(mw[0].wide, mw[1].wide);
        px.c[0] = dx;
        px.ldc = lddx;
        FPN_FF_TRY(check_product(dtype, px, kInner, order_x, false));
    }
    void *const dw_out[2] = {dw_gate, dw_up};
    const int dws = dw_gate ? weight_products(mx, md, 2, dw_out, lddw, w_transposed, pw) : 0;
    for (int i = 0; i < dws; ++i) FPN_FF_TRY(check_product(dtype, pw[i], kOuter, kOuter, false));

    FPN_FF_TRY(copies.make(st));
    FPN_FF_TRY(more.make(st));
    if (down) {
        FPN_FF_TRY(run_product(dtype, ph, kInner, order_down, false, partial, space.partial, st));
        if (fused && g.sums) {
            const int rows_each = plan_h.bn == 256 ? 128 : plan_h.bm == 256 ? 64 : 32;       // (of a wave: 32 TM of feed_forward_wide.h)
            FPN_FF_TRY(run_column_join(dtype, cout, (int)((rows + plan_h.bm - 1) / plan_h.bm * (plan_h.bm / rows_each)), g.sums, sums_out, st));
        }
    }
    if (!fused) FPN_FF_TRY(run_grad(dtype, g, true, down, sums_out, st));
    if (want_x) FPN_FF_TRY(run_product(dtype, px, kInner, order_x, false, partial, space.partial, st));
    for (int i = 0; i < dws; ++i) FPN_FF_TRY(run_product(dtype, pw[i], kOuter, kOuter, false, partial, space.partial, st));
    return FPN_OK;
}

}  // extern "C"
