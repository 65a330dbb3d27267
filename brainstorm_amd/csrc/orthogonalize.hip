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
//
// The float16 matrix rate bounds large matrices (a large product reaches 1349 TFLOP/s, three of them for each of ours):
// the momentum update of 4096 x 4096 takes 3.59 ms, of which products that cannot be left out 3.05; 4 x 1000 x 1000 take
// 0.42 ms (0.18): the L2 caches, from which tiles small enough to fill the card read 268 MB a product, 9 TB/s; 1200 x 784 takes 0.18 ms (0.03): 17 launches of 10 to 13 us, each
// a chain of its steps' waits.
#include "common.h"

#pragma clang fp contract(off)

namespace bship {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr int kPad = 128;                  // sides of the planes are multiples of this, filled with zeros
constexpr float kScaleX = 32768.0f, kScaleP = 16384.0f;      // X and A are kept times 2^15, p times 2^14

// A matrix (rows, 32 blocks) as two planes of blocks of 16 x 32 entries, block after block along a row of blocks. A block
// holds its four 16 x 8 parts one after the other, each row of 8 entries (16 bytes) behind the one before: what a matrix
// instruction takes from 64 lanes is one run of 1 KiB, in memory as in LDS, where it meets every bank once. (With plain rows,
// whose pieces have to be turned in LDS, a product of 4096 x 4096 took 12 % more cycles.)
struct Planes {
    _Float16* p;
    int64_t plane, each;                   // distance of the lo plane, of the matrices of a stack
    int rows, blocks;
    // the entry (row, k) of matrix z
    __device__ __forceinline__ _Float16* at(unsigned z, int row, int k) const {
        return p + z * each + (static_cast<int64_t>(row >> 4) * blocks + (k >> 5)) * 512 + (k >> 3 & 3) * 128 + (row & 15) * 8 + (k & 7);
    }
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
    __shared__ double s[4];
    const int64_t n = a.rows * a.cols, base = static_cast<int64_t>(blockIdx.z) * n;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * 64, c0 = static_cast<int64_t>(blockIdx.x) * 64;
    float u[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) {
        const int64_t r = r0 + x * 4 + threadIdx.x / 64, c = c0 + threadIdx.x % 64;
        u[x] = 0.0f;
        if (r < a.rows && c < a.cols) {
            const int64_t at = base + r * a.cols + c;
            u[x] = update_of(a, a.grad[at], a.velocity ? a.velocity[at] : 0.0f);
        }
    }
    double sum = 0.0;
    for (int i = threadIdx.x; i < a.parts; i += kBlock) sum += a.part[static_cast<int64_t>(blockIdx.z) * a.parts + i];
    for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = (s[0] + s[1]) + (s[2] + s[3]);
    const double inv = sum == 0.0 ? 0.0 : 1.0 / sqrt(sum);
    // the planes along the matrix's own rows, and those along its columns
    const Planes& along = tall ? xt : x;
    const Planes& across = tall ? x : xt;
#pragma unroll
    for (int x = 0; x < 16; ++x)
        tile[x * 4 + threadIdx.x / 64][threadIdx.x % 64] = static_cast<float>(static_cast<double>(u[x]) * inv) * kScaleX;
    __syncthreads();
    // rows of 8 entries: 16 bytes of each plane
    for (int e = threadIdx.x; e < 64 * 8; e += kBlock) {
        const int row = e % 64, k = e / 64 * 8;
        h8 hi, lo;
        auto store = [&](const Planes& to, int64_t to_row, int64_t to_k) {
            _Float16* p = to.at(blockIdx.z, static_cast<int>(to_row), static_cast<int>(to_k));
            *reinterpret_cast<h8*>(p) = hi;
            *reinterpret_cast<h8*>(p + to.plane) = lo;
        };
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            _Float16 h, l;
            split(tile[row][k + x], h, l);
            hi[x] = h;
            lo[x] = l;
        }
        store(along, r0 + row, c0 + k);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            _Float16 h, l;
            split(tile[k + x][row], h, l);
            hi[x] = h;
            lo[x] = l;
        }
        store(across, c0 + row, r0 + k);
    }
}

struct ProductArgs {
    Planes p, q;             // C = P Q^T, both contiguous along k
    int k;                   // multiple of 32
    int used_p, used_q;      // rows of P and Q that are not only padding
    int tiles_p;             // tiles along the rows of P
    unsigned tiles;          // of a matrix
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

// C (T x T per workgroup) = P Q^T on 16 x 16 x 32 float16 matrix instructions: lane l holds P[l % 16][8 (l / 16) .. + 7] and, of
// the result, rows 4 (l / 16) + r, column l % 16. WM x WN wavefronts share the tile; G such groups share the summed axis
// (every G-th step of 32 each) and add their sums up in LDS at the end: a small tile's step is a chain of waits, which
// other groups' steps fill. Loads go straight to LDS, a block of a plane per instruction, STAGES - 1 steps ahead.
//
// FINE: lo lo is taken too, and all that is not hi hi is summed apart, where sums are 2^11 times smaller and so is what they
// round off. Sums over few entries need it: what three products leave out and round does not average out there. (Error against
// 64 bits over that of the same steps in plain float32, 150 matrices of random sides from 8 to 1200: smaller sides up to 64,
// median 1.04, largest 1.84; with it 0.83 and 1.25; longer ones 0.47 without. 2 x 53 x 16: 64 us, with it 67; 4 x 1000 x 1000
// would take 6 % more.)
template <int T, int WM, int WN, int G, int STAGES, int MODE, bool FINE>
__global__ __launch_bounds__(WM * WN * G * kWave, WM * WN * G / 4) void ns_product_kernel(ProductArgs a) {
    constexpr int kWaves = WM * WN;                      // of one group
    constexpr int X = T / WM / 16, Y = T / WN / 16;      // tiles of 16 on the sides of a wavefront's part
    constexpr int kPlane = T * 32;                       // elements of one plane of one operand in LDS
    constexpr int kRequests = T / 16;                    // blocks of one plane per step
    constexpr int kLoads = 4 * kRequests / kWaves;       // of one wavefront per step
    static_assert(4 * kRequests % kWaves == 0, "whole loads per wavefront");
    static_assert(G == 1 || static_cast<size_t>(T) * T * 4 * G <= sizeof(_Float16) * G * STAGES * 4 * kPlane, "the sums fit");
    __shared__ __attribute__((aligned(16))) _Float16 lds[G][STAGES][4 * kPlane];
    const int tid = threadIdx.x, lane = tid & 63, all_wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wave = all_wave % kWaves, group = all_wave / kWaves;
    const int l16 = lane & 15, lq = lane >> 4;
    const int rows_p = a.p.rows, rows_q = a.q.rows;      // multiples of 128; a tile of 192 or 256 may reach behind them
    // Consecutive workgroups go to the 8 XCDs in turn: each XCD takes a run of tiles that lie close to each other, so
    // that its L2 holds what they share: four rows of tiles, column by column, and four columns of the upper triangle.
    const unsigned run = gridDim.x / 8;
    const unsigned in_order = blockIdx.x < 8 * run ? blockIdx.x % 8 * run + blockIdx.x / 8 : blockIdx.x;
    const unsigned z = in_order / a.tiles;
    const int t = static_cast<int>(in_order % a.tiles);
    int bi, bj;
    if constexpr (MODE == kGram || MODE == kPoly) {
        // columns 4 g .. 4 g + 3 begin at tile 8 g^2 + 2 g: 4 g rows of them and a triangle
        int g = static_cast<int>((sqrtf(32.0f * t + 4.0f) - 2.0f) * 0.0625f);
        while (8 * (g + 1) * (g + 1) + 2 * (g + 1) <= t) ++g;
        while (8 * g * g + 2 * g > t) --g;
        const int width = a.tiles_p - 4 * g < 4 ? a.tiles_p - 4 * g : 4;
        int rest = t - (8 * g * g + 2 * g);
        if (rest < 4 * g * width) {
            bi = rest / width;
            bj = 4 * g + rest % width;
        } else {
            rest -= 4 * g * width;
            bi = 4 * g;
            for (int left = width; rest >= left; --left, ++bi) rest -= left;
            bj = bi + rest;
        }
    } else {
        const int tiles_q = static_cast<int>(a.tiles) / a.tiles_p, g = t / (4 * tiles_q), rest = t % (4 * tiles_q);
        const int width = a.tiles_p - 4 * g < 4 ? a.tiles_p - 4 * g : 4;
        bi = 4 * g + rest % width;
        bj = rest / width;
    }

    const _Float16* from[kLoads];                        // the same in all lanes
#pragma unroll
    for (int m = 0; m < kLoads; ++m) {
        const int load = wave + m * kWaves, op = load / kRequests;
        const Planes& side = op < 2 ? a.p : a.q;
        const int block = (op < 2 ? bi : bj) * kRequests + load % kRequests, blocks = side.rows >> 4;
        from[m] = side.p + z * side.each + (op & 1) * side.plane +
                  (static_cast<int64_t>(block < blocks ? block : blocks - 1) * side.blocks + group) * 512;
    }
    auto request = [&](int buf, int step) {
#pragma unroll
        for (int m = 0; m < kLoads; ++m)
            load_to_lds(from[m] + step * (512 * G) + lane * 8, &lds[group][buf][(wave + m * kWaves) * 512]);
    };
    const int wr = wave % WM * (T / WM), wc = wave / WM * (T / WN);
    f4 acc[X][Y];
#pragma unroll
    for (int x = 0; x < X; ++x)
#pragma unroll
        for (int y = 0; y < Y; ++y) acc[x][y] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    f4 fine[FINE ? X : 1][FINE ? Y : 1];
    if constexpr (FINE)
#pragma unroll
        for (int x = 0; x < X; ++x)
#pragma unroll
            for (int y = 0; y < Y; ++y) fine[x][y] = f4{0.0f, 0.0f, 0.0f, 0.0f};

    // steps of this group; all groups go through as many as the first, the last one perhaps without products
    const int blocks_k = a.k / 32, steps = (blocks_k + G - 1) / G;
    const int own = (blocks_k - group + G - 1) / G;
    auto piece = [&](const _Float16* plane, int row) { return *reinterpret_cast<const h8*>(plane + row * 32 + lane * 8); };
    struct Side { h8 hi[Y], lo[Y]; };
    struct Row { h8 hi, lo; };
    auto read_side = [&](Side& to, int buf) {
#pragma unroll
        for (int y = 0; y < Y; ++y) {
            to.hi[y] = piece(lds[group][buf] + 2 * kPlane, wc + 16 * y);
            to.lo[y] = piece(lds[group][buf] + 3 * kPlane, wc + 16 * y);
        }
    };
    auto read_row = [&](Row& to, int buf, int x) {
        to.hi = piece(lds[group][buf], wr + 16 * x);
        to.lo = piece(lds[group][buf] + kPlane, wr + 16 * x);
    };
    // Step s with its q in `now` and its first rows of p in row[0]. Everything is read from LDS before the last X-th of the
    // products; then the wavefronts meet, the step's buffer is given to the loads of step s + STAGES, and the first
    // operands of step s + 1 are read while those products run.
    Row row[2];
    int buf = 0;                                       // s % STAGES
    auto step = [&](int s, const Side& now, Side& next) {
        const int after = buf + 1 == STAGES ? 0 : buf + 1;
#pragma unroll
        for (int x = 0; x < X; ++x) {
            if (x + 1 < X) {
                read_row(row[(x + 1) & 1], buf, x + 1);
            } else if (s + 1 < steps) {
                __builtin_amdgcn_s_waitcnt(0xc07f);    // lgkmcnt(0): this wavefront's reads have come
                // and its pieces of step s + 1 are there: those of the steps behind it, if all of them are asked for,
                // may be missing
                if (s + STAGES - 1 < own) wait_until_outstanding<(STAGES - 2) * kLoads>();
                else wait_until_outstanding<0>();
                __builtin_amdgcn_s_barrier();          // everybody's
                asm volatile("" ::: "memory");
                if (s + STAGES < own) request(buf, s + STAGES);
                read_side(next, after);
                read_row(row[X & 1], after, 0);
            }
            __builtin_amdgcn_sched_barrier(0);         // the reads above are under way during the products below
            if (G > 1 && s >= own) continue;
            const Row& p = row[x & 1];
            if constexpr (FINE) {
#pragma unroll
                for (int y = 0; y < Y; ++y) fine[x][y] = mfma(p.lo, now.lo[y], fine[x][y]);
#pragma unroll
                for (int y = 0; y < Y; ++y) fine[x][y] = mfma(p.lo, now.hi[y], fine[x][y]);
#pragma unroll
                for (int y = 0; y < Y; ++y) fine[x][y] = mfma(p.hi, now.lo[y], fine[x][y]);
            } else {
#pragma unroll
                for (int y = 0; y < Y; ++y) acc[x][y] = mfma(p.lo, now.hi[y], acc[x][y]);
#pragma unroll
                for (int y = 0; y < Y; ++y) acc[x][y] = mfma(p.hi, now.lo[y], acc[x][y]);
            }
#pragma unroll
            for (int y = 0; y < Y; ++y) acc[x][y] = mfma(p.hi, now.hi[y], acc[x][y]);
            __builtin_amdgcn_sched_barrier(0);
        }
        buf = after;
    };
    static_assert(X % 2 == 0, "the rows of p take turns in two registers");
    Side even, odd;
    for (int s = 0; s < STAGES && s < own; ++s) request(s, s);
    wait_until_outstanding<0>();
    __syncthreads();
    read_side(even, 0);
    read_row(row[0], 0, 0);
    for (int s = 0; s < steps; s += 2) {
        step(s, even, odd);
        if (s + 1 < steps) step(s + 1, odd, even);
    }
    if constexpr (FINE)
#pragma unroll
        for (int x = 0; x < X; ++x)
#pragma unroll
            for (int y = 0; y < Y; ++y) acc[x][y] += fine[x][y];

    // a 16 x 16 tile of the result: rows i .. i + 3, column j
    auto finish = [&](f4 v, int i, int j) {
        if (i >= rows_p || j >= rows_q) return;
        if constexpr (MODE == kLast) {
            v *= 1.0f / (kScaleP * kScaleX);
            const int64_t base = static_cast<int64_t>(z) * a.u.rows * a.u.cols;
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
                // the matrix is symmetric: rows i .. i + 3 of column j lie side by side as columns of row j
                const _Float16* e = a.p.at(z, j, i);
                const h4 e_hi = *reinterpret_cast<const h4*>(e), e_lo = *reinterpret_cast<const h4*>(e + a.p.plane);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float gram = static_cast<float>(e_hi[r]) + static_cast<float>(e_lo[r]);
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
            _Float16* t = a.ct.at(z, j, i);
            *reinterpret_cast<h4*>(t) = hi;
            *reinterpret_cast<h4*>(t + a.ct.plane) = lo;
            // a symmetric result's diagonal tile is complete with its transpose
            if (MODE == kNext || bi != bj) {
                _Float16* c = a.c.at(z, i, j);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    c[8 * r] = hi[r];
                    c[8 * r + a.c.plane] = lo[r];
                }
            }
        }
    };
    if constexpr (G == 1) {
#pragma unroll
        for (int x = 0; x < X; ++x)
#pragma unroll
            for (int y = 0; y < Y; ++y) finish(acc[x][y], bi * T + wr + 16 * x + 4 * lq, bj * T + wc + 16 * y + l16);
    } else {
        // every group's sums, a register after the other, then each group takes every G-th tile of 16 of a wavefront's part
        f4* sums = reinterpret_cast<f4*>(lds);
        __syncthreads();
#pragma unroll
        for (int x = 0; x < X; ++x)
#pragma unroll
            for (int y = 0; y < Y; ++y) sums[((group * kWaves + wave) * X * Y + x * Y + y) * kWave + lane] = acc[x][y];
        __syncthreads();
        for (int n = group; n < X * Y; n += G) {
            f4 v = sums[(wave * X * Y + n) * kWave + lane];
#pragma unroll
            for (int other = 1; other < G; ++other) v += sums[((other * kWaves + wave) * X * Y + n) * kWave + lane];
            finish(v, bi * T + wr + 16 * (n / Y) + 4 * lq, bj * T + wc + 16 * (n % Y) + l16);
        }
    }
}

template <int T, int WM, int WN, int G, int STAGES, int MODE, bool FINE = false>
void launch_tiles(const ProductArgs& a, unsigned count) {
    hipLaunchKernelGGL((ns_product_kernel<T, WM, WN, G, STAGES, MODE, FINE>), dim3(a.tiles * count), dim3(WM * WN * G * kWave), 0,
                       ctx().stream, a);
}

constexpr int kFineMost = 128;      // matrices with smaller sides up to it take the finer sums, in tiles of 64

// The tile side: what 32 entries of the summed axis cost with one tile on every compute unit, in hundredths of a
// microsecond, times the rounds that the tiles take. Measured (4096 x 4096: 256 against 192 and 128 for the full product
// 336, 440 and 412 us, for the symmetric ones 280, 208 and 315; 4 x 1000 x 1000: 128 against 64 for the full product 34.5
// and 38.7 us, for the symmetric ones 28.9 and 26.5); between the two a choice may be off, at a cost in time only. Tiles of 64
// share a compute unit, so their rounds need not be whole; where there is at most one for each, four groups share its summed
// axis (784 x 1200: 13 us, one group 20).
template <int MODE>
int launch_product(ProductArgs a, unsigned count) {
    const bool fine = a.used_p <= kFineMost;            // the smaller side
    const int64_t cus = ctx().num_cus;
    constexpr int kTiles[] = {256, 192, 128, 64}, kCost[] = {260, 160, 83, 30};
    int best = 0;                       // (a launch has fewer than 2^32 threads: up to 512 of them for a tile)
    double least = 0.0;
    for (int n = 0; n < 4; ++n) {
        const int64_t side = ceil_div(a.used_p, kTiles[n]), other = ceil_div(a.used_q, kTiles[n]);
        const int64_t tiles = MODE == kGram || MODE == kPoly ? side * (side + 1) / 2 : side * other;
        const int64_t all = tiles * count;
        const double rounds = kTiles[n] == 64 ? static_cast<double>(all > cus ? all : cus) / cus : static_cast<double>(ceil_div(all, cus));
        if (all > 0x7fffff || (fine && kTiles[n] != 64) || (best && rounds * kCost[n] >= least)) continue;
        least = rounds * kCost[n];
        best = kTiles[n];
        a.tiles_p = static_cast<int>(side);
        a.tiles = static_cast<unsigned>(tiles);
    }
    switch (best) {
        case 256: launch_tiles<256, 2, 4, 1, 2, MODE>(a, count); break;
        case 192: launch_tiles<192, 2, 4, 1, 3, MODE>(a, count); break;
        case 128: launch_tiles<128, 2, 2, 2, 2, MODE>(a, count); break;
        case 64:
            if (fine) {
                if (static_cast<int64_t>(a.tiles) * count > cus) launch_tiles<64, 2, 2, 1, 2, MODE, true>(a, count);
                else launch_tiles<64, 2, 2, 4, 2, MODE, true>(a, count);
            } else if (static_cast<int64_t>(a.tiles) * count > cus) launch_tiles<64, 2, 2, 1, 2, MODE>(a, count);
            else launch_tiles<64, 2, 2, 4, 2, MODE>(a, count);
            break;
        default: return set_error(BSHIP_ERR_BAD_DIMENSION, "orthogonalize: the matrices exceed one launch");
    }
    return check_launch("orthogonalize, product");
}

int orthogonal(UpdateArgs u, int64_t count, int steps) {
    const int tall = u.rows > u.cols;
    const int64_t m = ceil_div(tall ? u.cols : u.rows, kPad) * kPad, n = ceil_div(tall ? u.rows : u.cols, kPad) * kPad;
    const int small = static_cast<int>(tall ? u.cols : u.rows), large = static_cast<int>(tall ? u.rows : u.cols);
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
        Planes p = {at, count * rows * cols, rows * cols, static_cast<int>(rows), static_cast<int>(cols / 32)};
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
    for (int s = 0; s < steps && st == 0; ++s) {
        ProductArgs a = {};
        a.u = u;
        a.tall = tall;
        a.p = a.q = x;
        a.used_p = a.used_q = small;
        a.k = (large + 31) / 32 * 32;
        a.c = a.ct = gram;
        if ((st = launch_product<kGram>(a, z)) != 0) break;
        a.p = a.q = gram;
        a.k = (small + 31) / 32 * 32;
        a.c = a.ct = poly;
        if ((st = launch_product<kPoly>(a, z)) != 0) break;
        a.p = poly;
        a.q = xt;
        a.used_q = large;
        a.c = y;
        a.ct = yt;
        if (s + 1 < steps) st = launch_product<kNext>(a, z);
        else st = launch_product<kLast>(a, z);
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
