// Orthogonalised matrices by Newton-Schulz products, alone and as a momentum update.
//
//   X_0 = U / |U|_F,   X <- p X  with  p = a I + b A + c A^2,  A = X X^T        (steps times)
//
// moves every singular value s of X to a s + b s^3 + c s^5; with (a, b, c) = (3.4445, -4.7750, 2.0315) five steps
// bring all but tiny ones into about [0.7, 1.2]. A matrix with more rows than columns is taken transposed, so A is
// m x m with m the smaller side.
//
// Products: the matrix cores multiply float16 sixteen times as fast as float32. Every matrix is therefore kept as two
// float16 planes, hi = round(x) and lo = round(x - hi), which hold 22 bits and a sign, and a product is taken as
// hi hi + hi lo + lo hi with float32 sums: the part left out, lo lo, and the rounding of lo are both below 2^-22 of
// the entry's magnitude, of the size of the float32 sums' own rounding. float16's range is no limit here: the
// singular values stay below 1.21 (the polynomial's largest value over [0, 1.21]), hence |X| <= 1.21, |A| <= 1.45 and
// |p| <= 3.45 entry by entry, and the planes hold the entries times 2^15, 2^15 and 2^14, with an absolute resolution
// of 2^-40 and 2^-39 at their small end.
//
// A and p are symmetric: only the tiles on and above the diagonal are computed and each is written twice. X is kept
// in both orientations, so every product has both operands contiguous along the summed axis.
#include "common.h"

#pragma clang fp contract(off)

namespace bship {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr int kPad = 128;                  // sides of the planes are multiples of this, filled with zeros
constexpr float kScaleX = 32768.0f, kScaleP = 16384.0f;      // X and A are kept times 2^15, p times 2^14

struct Planes {                            // hi at p, lo `plane` elements behind it; matrices `each` elements apart
    _Float16* p;
    int64_t plane, each;
    int ld;
};

__device__ __forceinline__ void split(float x, _Float16& hi, _Float16& lo) {
    hi = static_cast<_Float16>(x);
    lo = static_cast<_Float16>(x - static_cast<float>(hi));
}

struct UpdateArgs {
    const float* grad;                     // the matrices themselves when `velocity` is NULL
    float *velocity, *out;                 // out: the result, or the parameters that the update is added to
    float momentum, factor;
    int nesterov, add;
    int64_t rows, cols;
    double* part;                          // (count, parts) partial sums of squares
    int parts;
};

// The matrix to orthogonalise: the gradient, or momentum and gradient as two float32 operations each.
__device__ __forceinline__ float update_of(const UpdateArgs& a, float g, float v) {
    if (!a.velocity) return g;
    if (!a.nesterov) return v;
    const float w = a.momentum * v;
    return g + w;
}

// velocity = momentum velocity + gradient, and partial sums of the squares of what is orthogonalised (float64: the
// squares of float32 values neither overflow nor vanish there).
__global__ __launch_bounds__(kBlock) void ns_norm_kernel(UpdateArgs a) {
    __shared__ double s[4];
    const int64_t n = a.rows * a.cols, base = static_cast<int64_t>(blockIdx.y) * n;
    double sum = 0.0;
    for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x) * 4; i < n;
         i += static_cast<int64_t>(gridDim.x) * kBlock * 4) {
        const int left = n - i < 4 ? static_cast<int>(n - i) : 4;
        f4 g = {0.0f, 0.0f, 0.0f, 0.0f}, v = g;
        const float* gp = a.grad + base + i;
        float* vp = a.velocity ? a.velocity + base + i : nullptr;
        if (left == 4) {
            g = *reinterpret_cast<const f4u*>(gp);
            if (vp) v = *reinterpret_cast<const f4u*>(vp);
        } else {
            for (int r = 0; r < left; ++r) {
                g[r] = gp[r];
                if (vp) v[r] = vp[r];
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (vp) {
                const float w = a.momentum * v[r];
                v[r] = w + g[r];
            }
            const double u = r < left ? update_of(a, g[r], v[r]) : 0.0f;
            sum += u * u;
        }
        if (vp) {
            if (left == 4) *reinterpret_cast<f4u*>(vp) = v;
            else
                for (int r = 0; r < left; ++r) vp[r] = v[r];
        }
    }
    for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) a.part[blockIdx.y * gridDim.x + blockIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
}

// X_0 and its transpose, 64 x 64 entries per workgroup. `tall`: the matrix has more rows than columns and X is its
// transpose. Entries outside the matrix are zeros. A matrix of zeros stays one; NaN and infinities go through.
__global__ __launch_bounds__(kBlock) void ns_start_kernel(UpdateArgs a, Planes x, Planes xt, int tall) {
    __shared__ float tile[64][65];
    __shared__ double s[kBlock];
    const int64_t n = a.rows * a.cols, base = static_cast<int64_t>(blockIdx.z) * n;
    double sum = 0.0;
    for (int i = threadIdx.x; i < a.parts; i += kBlock) sum += a.part[static_cast<int64_t>(blockIdx.z) * a.parts + i];
    s[threadIdx.x] = sum;
    for (int d = kBlock / 2; d > 0; d >>= 1) {
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < d) s[threadIdx.x] += s[threadIdx.x + d];
    }
    __syncthreads();
    const double inv = s[0] == 0.0 ? 0.0 : 1.0 / sqrt(s[0]);
    // the planes along the matrix's own rows, and those along its columns
    const Planes& along = tall ? xt : x;
    const Planes& across = tall ? x : xt;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * 64, c0 = static_cast<int64_t>(blockIdx.x) * 64;
    for (int e = threadIdx.x; e < 64 * 64; e += kBlock) {
        const int64_t r = r0 + e / 64, c = c0 + e % 64;
        float u = 0.0f;
        if (r < a.rows && c < a.cols) {
            const int64_t at = base + r * a.cols + c;
            u = static_cast<float>(static_cast<double>(update_of(a, a.grad[at], a.velocity ? a.velocity[at] : 0.0f)) * inv);
        }
        u *= kScaleX;
        tile[e / 64][e % 64] = u;
        _Float16 hi, lo;
        split(u, hi, lo);
        _Float16* p = along.p + blockIdx.z * along.each + r * along.ld + c;
        p[0] = hi;
        p[along.plane] = lo;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 64 * 64; e += kBlock) {
        _Float16 hi, lo;
        split(tile[e % 64][e / 64], hi, lo);
        _Float16* p = across.p + blockIdx.z * across.each + (c0 + e / 64) * across.ld + r0 + e % 64;
        p[0] = hi;
        p[across.plane] = lo;
    }
}

struct ProductArgs {
    Planes p, q;             // C = P Q^T, both contiguous along k
    int k;                   // multiple of 32
    Planes c, ct;            // the result and its transpose
    UpdateArgs u;            // the last step's product goes there
    int tall;
};

__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// 16 bytes per lane from memory into LDS, behind each other from `to` on
__device__ __forceinline__ void load_to_lds(const _Float16* from, _Float16* to) {
    __builtin_amdgcn_global_load_lds(from, to, 16, 0, 0);
}

enum { kGram, kPoly, kNext, kLast };

// C (TM x TM per workgroup of four wavefronts, each (TM / 2)^2) = P Q^T on 16 x 16 x 32 float16 matrix instructions:
// lane l holds P[l % 16][8 (l / 16) .. + 7] and, of the result, rows 4 (l / 16) + r, column l % 16. Rows of 32 entries
// (64 bytes) lie in LDS as four 16-byte pieces whose order is turned by the row (piece ^ (row / 4 % 4)), so that the
// 16 lanes that read one piece of 16 rows meet all banks; loads go straight to LDS and fetch in that order.
template <int TM, int MODE>
__global__ __launch_bounds__(kBlock) void ns_product_kernel(ProductArgs a) {
    constexpr int W = TM / 32;                     // tiles of 16 on a side of a wavefront's part
    constexpr int kPlane = TM * 32;                // elements of one plane of one operand in LDS
    __shared__ __attribute__((aligned(16))) _Float16 lds[2][4][kPlane];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int l16 = lane & 15, lq = lane >> 4;
    int bi, bj;
    if constexpr (MODE == kGram || MODE == kPoly) {
        // tile t of the upper triangle, column by column: bj (bj + 1) / 2 <= t
        const int t = blockIdx.x;
        bj = static_cast<int>((sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
        while ((bj + 1) * (bj + 2) / 2 <= t) ++bj;
        while (bj * (bj + 1) / 2 > t) --bj;
        bi = t - bj * (bj + 1) / 2;
    } else {
        const int tiles = a.p.each / a.p.ld / TM;   // along the smaller side
        bi = blockIdx.x % tiles;
        bj = blockIdx.x / tiles;
    }
    const _Float16* src[4] = {a.p.p + blockIdx.z * a.p.each + static_cast<int64_t>(bi) * TM * a.p.ld, nullptr,
                              a.q.p + blockIdx.z * a.q.each + static_cast<int64_t>(bj) * TM * a.q.ld, nullptr};
    src[1] = src[0] + a.p.plane;
    src[3] = src[2] + a.q.plane;

    auto request = [&](int buf, int k0) {
#pragma unroll
        for (int op = 0; op < 4; ++op)
#pragma unroll
            for (int m = 0; m < TM / 64; ++m) {
                const int slot = m * kBlock + wave * kWave + lane, row = slot >> 2, piece = (slot & 3) ^ (row >> 2 & 3);
                const int ld = op < 2 ? a.p.ld : a.q.ld;
                load_to_lds(src[op] + static_cast<int64_t>(row) * ld + k0 + piece * 8,
                            &lds[buf][op][(m * kBlock + wave * kWave) * 8]);
            }
    };
    const int wr = (wave & 1) * (TM / 2), wc = (wave >> 1) * (TM / 2);
    f4 acc[W][W];
#pragma unroll
    for (int x = 0; x < W; ++x)
#pragma unroll
        for (int y = 0; y < W; ++y) acc[x][y] = f4{0.0f, 0.0f, 0.0f, 0.0f};

    request(0, 0);
    const int steps = a.k / 32;
    for (int s = 0; s < steps; ++s) {
        wait_until_outstanding<0>();               // this wavefront's pieces of step s are there
        __syncthreads();                           // everybody's are, and the other buffer is free
        if (s + 1 < steps) request((s + 1) & 1, (s + 1) * 32);
        const _Float16* ph = lds[s & 1][0];
        const _Float16* qh = lds[s & 1][2];
        auto piece = [&](const _Float16* plane, int row) {
            return *reinterpret_cast<const h8*>(plane + row * 32 + ((lq ^ (row >> 2 & 3)) * 8));
        };
        h8 q_hi[W], q_lo[W];
#pragma unroll
        for (int y = 0; y < W; ++y) {
            q_hi[y] = piece(qh, wc + 16 * y + l16);
            q_lo[y] = piece(qh + kPlane, wc + 16 * y + l16);
        }
#pragma unroll
        for (int x = 0; x < W; ++x) {
            const h8 p_hi = piece(ph, wr + 16 * x + l16), p_lo = piece(ph + kPlane, wr + 16 * x + l16);
#pragma unroll
            for (int y = 0; y < W; ++y) {
                acc[x][y] = mfma(p_lo, q_hi[y], acc[x][y]);
                acc[x][y] = mfma(p_hi, q_lo[y], acc[x][y]);
                acc[x][y] = mfma(p_hi, q_hi[y], acc[x][y]);
            }
        }
    }

#pragma unroll
    for (int x = 0; x < W; ++x)
#pragma unroll
        for (int y = 0; y < W; ++y) {
            const int64_t i = static_cast<int64_t>(bi) * TM + wr + 16 * x + 4 * lq;      // rows i .. i + 3
            const int64_t j = static_cast<int64_t>(bj) * TM + wc + 16 * y + l16;
            f4 v = acc[x][y];
            if constexpr (MODE == kLast) {
                v *= 1.0f / (kScaleP * kScaleX);
                const int64_t base = static_cast<int64_t>(blockIdx.z) * a.u.rows * a.u.cols;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t row = a.tall ? j : i + r, col = a.tall ? i + r : j;
                    if (row >= a.u.rows || col >= a.u.cols) continue;
                    float* o = a.u.out + base + row * a.u.cols + col;
                    if (a.u.add) {
                        const float w = a.u.factor * v[r];
                        *o = *o + w;
                    } else {
                        *o = v[r];
                    }
                }
            } else {
                if constexpr (MODE == kGram) {
                    v *= 1.0f / kScaleX;
                } else if constexpr (MODE == kPoly) {
                    const _Float16* e = a.p.p + blockIdx.z * a.p.each + i * a.p.ld + j;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float gram = static_cast<float>(e[r * a.p.ld]) + static_cast<float>(e[r * a.p.ld + a.p.plane]);
                        v[r] = (kB * kScaleP / kScaleX) * gram + (kC * kScaleP / (kScaleX * kScaleX)) * v[r];
                        if (i + r == j) v[r] += kA * kScaleP;
                    }
                } else {
                    v *= 1.0f / kScaleP;
                }
                h4 hi, lo;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    _Float16 vh, vl;
                    split(v[r], vh, vl);
                    hi[r] = vh;
                    lo[r] = vl;
                }
                _Float16* t = a.ct.p + blockIdx.z * a.ct.each + j * a.ct.ld + i;
                *reinterpret_cast<h4*>(t) = hi;
                *reinterpret_cast<h4*>(t + a.ct.plane) = lo;
                // a symmetric result's diagonal tile is complete with its transpose
                if (MODE == kNext || bi != bj) {
                    _Float16* c = a.c.p + blockIdx.z * a.c.each + i * a.c.ld + j;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        c[static_cast<int64_t>(r) * a.c.ld] = hi[r];
                        c[static_cast<int64_t>(r) * a.c.ld + a.c.plane] = lo[r];
                    }
                }
            }
        }
}

template <int MODE>
int launch_product(const ProductArgs& a, int tile, unsigned tiles, unsigned count) {
    if (tile == 128)
        hipLaunchKernelGGL((ns_product_kernel<128, MODE>), dim3(tiles, 1, count), dim3(kBlock), 0, ctx().stream, a);
    else
        hipLaunchKernelGGL((ns_product_kernel<64, MODE>), dim3(tiles, 1, count), dim3(kBlock), 0, ctx().stream, a);
    return check_launch("orthogonalize, product");
}

int orthogonal(UpdateArgs u, int64_t count, int steps) {
    const int tall = u.rows > u.cols;
    const int64_t m = ceil_div(tall ? u.cols : u.rows, kPad) * kPad, n = ceil_div(tall ? u.rows : u.cols, kPad) * kPad;
    // planes: X, its transpose, the next X and its transpose, A, p
    const size_t x_elems = static_cast<size_t>(count) * m * n * 2, a_elems = static_cast<size_t>(count) * m * m * 2;
    int64_t parts = ceil_div(u.rows * u.cols, 16 * kBlock);
    if (parts > 512) parts = 512;
    const size_t part_bytes = static_cast<size_t>(count) * parts * sizeof(double);
    void* space = nullptr;
    int st = pool_alloc_raw((4 * x_elems + 2 * a_elems) * sizeof(_Float16) + part_bytes, &space);
    if (st != 0) return st;
    _Float16* at = static_cast<_Float16*>(space);
    auto take = [&](int64_t rows, int64_t cols) {
        Planes p = {at, count * rows * cols, rows * cols, static_cast<int>(cols)};
        at += 2 * count * rows * cols;
        return p;
    };
    Planes x = take(m, n), xt = take(n, m), y = take(m, n), yt = take(n, m), gram = take(m, m), poly = take(m, m);
    u.part = reinterpret_cast<double*>(at);
    u.parts = static_cast<int>(parts);
    const unsigned z = static_cast<unsigned>(count);
    hipLaunchKernelGGL(ns_norm_kernel, dim3(static_cast<unsigned>(parts), z), dim3(kBlock), 0, ctx().stream, u);
    st = check_launch("orthogonalize, norm");
    if (st == 0) {
        hipLaunchKernelGGL(ns_start_kernel, dim3(static_cast<unsigned>((tall ? m : n) / 64), static_cast<unsigned>((tall ? n : m) / 64), z),
                           dim3(kBlock), 0, ctx().stream, u, x, xt, tall);
        st = check_launch("orthogonalize, start");
    }
    const int tile = count * (m / 128) * (n / 128) >= ctx().num_cus ? 128 : 64;
    const unsigned side = static_cast<unsigned>(m / tile), triangle = side * (side + 1) / 2,
                   all = side * static_cast<unsigned>(n / tile);
    for (int s = 0; s < steps && st == 0; ++s) {
        ProductArgs a = {};
        a.u = u;
        a.tall = tall;
        a.p = a.q = x;
        a.k = static_cast<int>(n);
        a.c = a.ct = gram;
        if ((st = launch_product<kGram>(a, tile, triangle, z)) != 0) break;
        a.p = a.q = gram;
        a.k = static_cast<int>(m);
        a.c = a.ct = poly;
        if ((st = launch_product<kPoly>(a, tile, triangle, z)) != 0) break;
        a.p = poly;
        a.q = xt;
        a.c = y;
        a.ct = yt;
        if (s + 1 < steps) st = launch_product<kNext>(a, tile, all, z);
        else st = launch_product<kLast>(a, tile, all, z);
        Planes t = x; x = y; y = t;
        t = xt; xt = yt; yt = t;
    }
    (void)pool_free_raw(space);
    return st;
}

int check_matrices(const char* fn, int64_t count, int64_t rows, int64_t cols, int steps) {
    if (count < 0 || rows < 0 || cols < 0 || rows > (int64_t(1) << 20) || cols > (int64_t(1) << 20) || count > 65535)
        return set_error(BSHIP_ERR_BAD_DIMENSION, "%s: sizes out of range", fn);
    if (steps < 1 || steps > 100) return set_error(BSHIP_ERR_BAD_DIMENSION, "%s: %d steps: 1 to 100 are possible", fn, steps);
    return 0;
}

}  // namespace
}  // namespace bship

using namespace bship;

extern "C" {

int bship_orthogonalize_f32(const float* in, float* out, int64_t count, int64_t rows, int64_t cols, int steps) {
    BSHIP_REQUIRE_INIT();
    int st = check_matrices(__func__, count, rows, cols, steps);
    if (st != 0) return st;
    if (count == 0 || rows == 0 || cols == 0) return 0;
    BSHIP_REQUIRE_PTR(in);
    BSHIP_REQUIRE_PTR(out);
    BSHIP_REQUIRE_F32_ALIGNED(in);
    BSHIP_REQUIRE_F32_ALIGNED(out);
    UpdateArgs u = {};
    u.grad = in;
    u.out = out;
    u.rows = rows;
    u.cols = cols;
    return orthogonal(u, count, steps);
}

int bship_orthogonal_update_f32(float momentum, float neg_learning_rate, int nesterov, const float* gradients,
                                float* velocity, float* parameters, int64_t count, int64_t rows, int64_t cols, int steps) {
    BSHIP_REQUIRE_INIT();
    int st = check_matrices(__func__, count, rows, cols, steps);
    if (st != 0) return st;
    if (count == 0 || rows == 0 || cols == 0) return 0;
    BSHIP_REQUIRE_PTR(gradients);
    BSHIP_REQUIRE_PTR(velocity);
    BSHIP_REQUIRE_PTR(parameters);
    BSHIP_REQUIRE_F32_ALIGNED(gradients);
    BSHIP_REQUIRE_F32_ALIGNED(velocity);
    BSHIP_REQUIRE_F32_ALIGNED(parameters);
    UpdateArgs u = {};
    u.grad = gradients;
    u.velocity = velocity;
    u.out = parameters;
    u.momentum = momentum;
    u.factor = neg_learning_rate * sqrtf(rows > cols ? static_cast<float>(rows) / static_cast<float>(cols) : 1.0f);
    u.nesterov = nesterov != 0;
    u.add = 1;
    u.rows = rows;
    u.cols = cols;
    return orthogonal(u, count, steps);
}

}  // extern "C"
