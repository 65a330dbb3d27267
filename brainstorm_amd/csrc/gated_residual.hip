// The norms around a block with its gate and residual scale, forward and backward, in one pass each:
//
//   y = residual_scale x + act(gate) * post * block / rms(block)        the norm behind the block, gate, residual
//   h = pre * y / rms(y)                                                the norm before the next block
//   rms(v) = sqrt(mean(v^2) + epsilon) over a row
//
// A row is read once, kept in registers and reduced there: 3 arrays in and 2 out forward, 5 in and 3 out
// backward (the row's two means are formed again, which costs two reductions and no memory). Memory bounds both: 10000 x
// 1000 forward 38 us (5.3 TB/s), backward 58 us (5.5 TB/s) and 7 us for the weights' sums, 2048 x 4096 forward 30 us (5.6
// TB/s; a large copy: 5.1). One vector of four columns per thread keeps enough rows under way: four per thread on a
// wavefront per row took 51 and 115 us. The gate, the second norm, and the block itself (only the norm: h = pre * x / rms(x),
// 10000 x 1000: 14 us, its gradients 22 and 6) can be left out.
#include "common.h"

#pragma clang fp contract(fast)

namespace bship {
namespace {

struct GateArgs {
    const float *block, *gate, *x, *post, *pre;    // gate NULL: 1; pre NULL: no norm behind; block NULL: y is x
    float *y, *h;
    const float *dy, *dh;                          // backward; y is read then
    float *dblock, *dgate, *dx;
    float* part;                                   // partial sums of the weights' gradients: (groups, 2, width)
    int64_t rows;
    int width;
    int act;
    float residual_scale, epsilon;
    int accumulate;
};

// Four columns of a row for one thread. Loads are made without conditions, so that all of a row's are under way at once:
// a thread without columns takes the row's last four, and the last thread of a row whose width is no multiple of four
// takes four that end with the row; `skip` of them are others' and count as zeros.
struct Columns {
    int at, skip;
    __device__ __forceinline__ Columns(int c, int width)
        : at(c + 4 <= width ? c : width - 4), skip(c + 4 <= width ? 0 : c < width ? 4 - (width - c) : 4) {}
    __device__ __forceinline__ f4 own(f4 x, bool ragged) const {
        if (ragged)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (r < skip) x[r] = 0.0f;
        return x;
    }
    __device__ __forceinline__ f4 load(const float* row, bool ragged) const {
        return own(*reinterpret_cast<const f4u*>(row + at), ragged);
    }
    __device__ __forceinline__ void store(float* row, f4 x, bool add) const {
        float* p = row + at;
        if (skip == 0) {
            if (add) x += *reinterpret_cast<const f4u*>(p);
            *reinterpret_cast<f4u*>(p) = x;
            return;
        }
#pragma unroll
        for (int r = 1; r < 4; ++r)
            if (r >= skip) p[r] = add ? p[r] + x[r] : x[r];
    }
};

// The rows of the kernels for long rows and for widths below four.
__device__ __forceinline__ f4 load_row4(const float* p, int left) {
    if (left >= 4) return *reinterpret_cast<const f4u*>(p);
    f4 r = {0.0f, 0.0f, 0.0f, 0.0f};
    if (left > 0) r[0] = p[0];
    if (left > 1) r[1] = p[1];
    if (left > 2) r[2] = p[2];
    return r;
}
__device__ __forceinline__ void store_row4(float* p, f4 v, int left, bool add) {
    if (left <= 0) return;
    if (add) v += load_row4(p, left);
    if (left >= 4) {
        *reinterpret_cast<f4u*>(p) = v;
        return;
    }
    p[0] = v[0];
    if (left > 1) p[1] = v[1];
    if (left > 2) p[2] = v[2];
}

__device__ __forceinline__ float logistic(float z) { return 1.0f / (1.0f + expf(-z)); }

// act(z), and its derivative by z
__device__ __forceinline__ float gate_value(int act, float z) {
    switch (act) {
        case BSHIP_ACT_SIGMOID: return logistic(z);
        case BSHIP_ACT_TANH:    return tanhf(z);
        case BSHIP_ACT_REL:     return z > 0.0f || z != z ? z : 0.0f;
        case BSHIP_ACT_EL:      return z > 0.0f ? z : expm1f(z);
        case BSHIP_ACT_SWISH:   return z * logistic(z);
        default:                return z;
    }
}
__device__ __forceinline__ float gate_slope(int act, float z, float value) {
    switch (act) {
        case BSHIP_ACT_SIGMOID: return value * (1.0f - value);
        case BSHIP_ACT_TANH:    return 1.0f - value * value;
        case BSHIP_ACT_REL:     return z > 0.0f ? 1.0f : 0.0f;
        case BSHIP_ACT_EL:      return z > 0.0f ? 1.0f : value + 1.0f;
        case BSHIP_ACT_SWISH: {
            const float s = logistic(z);
            return s + value * (1.0f - s);
        }
        default:                return 1.0f;
    }
}

// A workgroup is the threads of one row, or four wavefronts with a row each.
template <int TPR> constexpr int kThreadsFor = TPR == kWave ? kBlock : TPR;

// Sums over the TPR threads of a row. Two places in LDS in turn: who writes
// the next sums' does not disturb who still reads the last.
template <int TPR, int N>
struct RowSums {
    float lds[2][N][TPR / kWave];
    __device__ __forceinline__ void operator()(float (&v)[N], int& turn) {
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = wave_sum(v[n]);
        if constexpr (TPR > kWave) {
            const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
            if (lane == 0)
#pragma unroll
                for (int n = 0; n < N; ++n) lds[turn][n][wave] = v[n];
            __syncthreads();
#pragma unroll
            for (int n = 0; n < N; ++n) {
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < TPR / kWave; ++w) s += lds[turn][n][w];
                v[n] = s;
            }
            turn ^= 1;
        }
    }
};

// TPR threads per row, V vectors of four floats per thread: width <= 4 TPR V.
template <int TPR, int V>
__global__ __launch_bounds__(kThreadsFor<TPR>) void gate_fwd_kernel(GateArgs a) {
    constexpr int kThreads = kThreadsFor<TPR>, kRows = kThreads / TPR;
    __shared__ RowSums<TPR, 1> sums;
    const int t = threadIdx.x % TPR;
    const float inv_n = 1.0f / static_cast<float>(a.width);
    const bool ragged = a.width != 4 * TPR * V;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    int turn = 0;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR; row < a.rows; row += step) {
        const int64_t base = row * a.width;
        f4 y[V];
        if (a.block) {
            f4 o[V], z[V];
            float s[1] = {0.0f};
#pragma unroll
            for (int m = 0; m < V; ++m) {
                const Columns c((t + m * TPR) * 4, a.width);
                o[m] = c.load(a.block + base, ragged);
                y[m] = c.load(a.x + base, ragged);
                if (a.gate) z[m] = c.load(a.gate + base, ragged);
            }
#pragma unroll
            for (int m = 0; m < V; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[0] += o[m][r] * o[m][r];
            sums(s, turn);
            const float rb = 1.0f / sqrtf(s[0] * inv_n + a.epsilon);
#pragma unroll
            for (int m = 0; m < V; ++m) {
                const Columns c((t + m * TPR) * 4, a.width);
                const f4 w = c.load(a.post, ragged);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float u = w[r] * (o[m][r] * rb);
                    if (a.gate) u *= gate_value(a.act, z[m][r]);
                    y[m][r] = a.residual_scale * y[m][r] + (r >= c.skip ? u : 0.0f);
                }
                c.store(a.y + base, y[m], false);
            }
        } else {
#pragma unroll
            for (int m = 0; m < V; ++m) y[m] = Columns((t + m * TPR) * 4, a.width).load(a.x + base, ragged);
        }
        if (!a.pre) continue;
        float s[1] = {0.0f};
#pragma unroll
        for (int m = 0; m < V; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[0] += y[m][r] * y[m][r];
        sums(s, turn);
        const float ry = 1.0f / sqrtf(s[0] * inv_n + a.epsilon);
#pragma unroll
        for (int m = 0; m < V; ++m) {
            const Columns c((t + m * TPR) * 4, a.width);
            c.store(a.h + base, c.load(a.pre, ragged) * (y[m] * ry), false);
        }
    }
}

// Sums over a workgroup, for the kernels below.
template <int N>
__device__ __forceinline__ void block_sums(float (&v)[N], float* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = wave_sum(v[n]);
    if (lane == 0)
#pragma unroll
        for (int n = 0; n < N; ++n) lds[n * 4 + wave] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = (lds[n * 4] + lds[n * 4 + 1]) + (lds[n * 4 + 2] + lds[n * 4 + 3]);
    __syncthreads();
}

// Rows of any width, for those that do not fit registers and those below four columns: three passes over the row, the
// second and third mostly out of the caches.
__global__ __launch_bounds__(kBlock) void gate_fwd_long_kernel(GateArgs a) {
    __shared__ float lds[8];
    const float inv_n = 1.0f / static_cast<float>(a.width);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t base = row * a.width;
        const float* y = a.block ? a.y : a.x;
        float s[1] = {0.0f};
        if (a.block) {
            for (int c = threadIdx.x * 4; c < a.width; c += 4 * kBlock) {
                const f4 o = load_row4(a.block + base + c, a.width - c);
#pragma unroll
                for (int r = 0; r < 4; ++r) s[0] += o[r] * o[r];
            }
            block_sums(s, lds);
            const float rb = 1.0f / sqrtf(s[0] * inv_n + a.epsilon);
            s[0] = 0.0f;
            for (int c = threadIdx.x * 4; c < a.width; c += 4 * kBlock) {
                const int left = a.width - c;
                const f4 o = load_row4(a.block + base + c, left), w = load_row4(a.post + c, left);
                f4 v = load_row4(a.x + base + c, left), z = {0.0f, 0.0f, 0.0f, 0.0f};
                if (a.gate) z = load_row4(a.gate + base + c, left);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float u = w[r] * (o[r] * rb);
                    if (a.gate) u *= gate_value(a.act, z[r]);
                    v[r] = a.residual_scale * v[r] + (r < left ? u : 0.0f);
                    s[0] += v[r] * v[r];
                }
                store_row4(a.y + base + c, v, left, false);
            }
        } else {
            for (int c = threadIdx.x * 4; c < a.width; c += 4 * kBlock) {
                const f4 v = load_row4(y + base + c, a.width - c);
#pragma unroll
                for (int r = 0; r < 4; ++r) s[0] += v[r] * v[r];
            }
        }
        if (!a.pre) continue;
        block_sums(s, lds);
        const float ry = 1.0f / sqrtf(s[0] * inv_n + a.epsilon);
        for (int c = threadIdx.x * 4; c < a.width; c += 4 * kBlock) {       // every thread reads what it wrote
            const int left = a.width - c;
            store_row4(a.h + base + c, load_row4(a.pre + c, left) * (load_row4(y + base + c, left) * ry), left, false);
        }
    }
}

// With e = dh * pre, n = block / rms(block):
//   total = dy + (e - y mean(e y) / rms(y)^2) / rms(y)            what arrives at y
//   dx = residual_scale total;  dgate = total post n act'(gate);  d = total post act(gate)
//   dblock = (d - n mean(d n)) / rms(block);  dpost = sum total act(gate) n;  dpre = sum dh y / rms(y)
// A workgroup keeps the columns' sums over its rows in registers or, for long rows, in its own row of `part`; they are
// added over the workgroups in a fixed order afterwards.
template <int TPR, int V>
__global__ __launch_bounds__(kThreadsFor<TPR>) void gate_bwd_kernel(GateArgs a) {
    constexpr int kThreads = kThreadsFor<TPR>, kRows = kThreads / TPR;
    __shared__ RowSums<TPR, 3> sums;
    __shared__ RowSums<TPR, 1> sums_n;
    __shared__ f4 part_s[kRows > 1 ? 2 * V : 1][kRows > 1 ? kThreads : 1];
    const int t = threadIdx.x % TPR;
    const float inv_n = 1.0f / static_cast<float>(a.width);
    const bool ragged = a.width != 4 * TPR * V;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    const f4 nothing = {0.0f, 0.0f, 0.0f, 0.0f};
    int turn = 0, turn_n = 0;
    f4 wpost[V], wpre[V], spost[V], spre[V];
#pragma unroll
    for (int m = 0; m < V; ++m) {
        const Columns c((t + m * TPR) * 4, a.width);
        wpost[m] = a.block ? c.load(a.post, ragged) : nothing;
        wpre[m] = a.pre ? c.load(a.pre, ragged) : nothing;
        spost[m] = spre[m] = nothing;
    }
    // Rows on many wavefronts are fetched while the one before them is worked on (2048 x 4096: 68 us, without 78; on two
    // vectors per thread the registers cost more than that: 1000 x 8000 88 us, with 114; narrow rows gain nothing).
    constexpr bool kAhead = TPR >= 512 && V == 1;
    struct Row { f4 dy[V], y[V], e[V], o[V], z[V]; } next;
    auto fetch = [&](int64_t row) {
        const int64_t base = row * a.width;
#pragma unroll
        for (int m = 0; m < V; ++m) {
            const Columns c((t + m * TPR) * 4, a.width);
            next.dy[m] = a.dy ? c.load(a.dy + base, false) : nothing;
            next.y[m] = a.pre ? c.load(a.y + base, false) : nothing;
            next.e[m] = a.pre ? c.load(a.dh + base, false) : nothing;
            next.o[m] = a.block ? c.load(a.block + base, false) : nothing;
            next.z[m] = a.gate ? c.load(a.gate + base, false) : nothing;
        }
    };
    int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR;
    if (kAhead && row < a.rows) fetch(row);
    for (; row < a.rows; row += step) {
        if (!kAhead) fetch(row);
        const int64_t base = row * a.width;
        f4 total[V], y[V], e[V], o[V], z[V];
#pragma unroll
        for (int m = 0; m < V; ++m) {
            const Columns c((t + m * TPR) * 4, a.width);
            total[m] = c.own(next.dy[m], ragged);
            y[m] = c.own(next.y[m], ragged);
            e[m] = c.own(next.e[m], ragged);
            o[m] = c.own(next.o[m], ragged);
            z[m] = c.own(next.z[m], ragged);
        }
        if (kAhead && row + step < a.rows) fetch(row + step);
        float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int m = 0; m < V; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[0] += y[m][r] * y[m][r];
                s[1] += e[m][r] * wpre[m][r] * y[m][r];
                s[2] += o[m][r] * o[m][r];
            }
        sums(s, turn);
        if (a.pre) {
            const float ry = 1.0f / sqrtf(s[0] * inv_n + a.epsilon), back = s[1] * inv_n * ry * ry;
#pragma unroll
            for (int m = 0; m < V; ++m) {
                spre[m] += e[m] * (y[m] * ry);
                total[m] += ry * (e[m] * wpre[m] - y[m] * back);
            }
        }
#pragma unroll
        for (int m = 0; m < V; ++m)
            Columns((t + m * TPR) * 4, a.width).store(a.dx + base, a.residual_scale * total[m], a.accumulate);
        if (!a.block) continue;
        const float rb = 1.0f / sqrtf(s[2] * inv_n + a.epsilon);
        float dn[1] = {0.0f};
#pragma unroll
        for (int m = 0; m < V; ++m) {
            const Columns c((t + m * TPR) * 4, a.width);
            f4 dz;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float n = o[m][r] * rb, value = a.gate ? gate_value(a.act, z[m][r]) : 1.0f;
                const float tv = r >= c.skip ? total[m][r] * value : 0.0f;
                if (a.gate) dz[r] = total[m][r] * (wpost[m][r] * n) * gate_slope(a.act, z[m][r], value);
                spost[m][r] += tv * n;
                total[m][r] = tv * wpost[m][r];                 // d from here on
                dn[0] += total[m][r] * o[m][r];
            }
            if (a.gate) c.store(a.dgate + base, dz, a.accumulate);
        }
        sums_n(dn, turn_n);
        const float back = dn[0] * inv_n * rb * rb;
#pragma unroll
        for (int m = 0; m < V; ++m)
            Columns((t + m * TPR) * 4, a.width).store(a.dblock + base, rb * (total[m] - o[m] * back), a.accumulate);
    }
    // the sums of the workgroup's rows of threads, in their order
    if constexpr (kRows > 1) {
#pragma unroll
        for (int m = 0; m < V; ++m) {
            part_s[m][threadIdx.x] = spost[m];
            part_s[V + m][threadIdx.x] = spre[m];
        }
        __syncthreads();
        if (threadIdx.x >= TPR) return;
#pragma unroll
        for (int m = 0; m < V; ++m)
            for (int r = 1; r < kRows; ++r) {
                spost[m] += part_s[m][threadIdx.x + r * TPR];
                spre[m] += part_s[V + m][threadIdx.x + r * TPR];
            }
    }
    float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.width;
#pragma unroll
    for (int m = 0; m < V; ++m) {
        const Columns c((t + m * TPR) * 4, a.width);
        c.store(part, spost[m], false);
        c.store(part + a.width, spre[m], false);
    }
}

__global__ __launch_bounds__(kBlock) void gate_bwd_long_kernel(GateArgs a) {
    __shared__ float lds[12];
    const float inv_n = 1.0f / static_cast<float>(a.width);
    float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.width;
    for (int c = threadIdx.x * 4; c < a.width; c += 4 * kBlock) {
        store_row4(part + c, f4{0.0f, 0.0f, 0.0f, 0.0f}, a.width - c, false);
        store_row4(part + a.width + c, f4{0.0f, 0.0f, 0.0f, 0.0f}, a.width - c, false);
    }
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t base = row * a.width;
        float s[3] = {0.0f, 0.0f, 0.0f};
        for (int c = threadIdx.x * 4; c < a.width; c += 4 * kBlock) {
            const int left = a.width - c;
            if (a.pre) {
                const f4 y = load_row4(a.y + base + c, left);
                const f4 e = load_row4(a.dh + base + c, left) * load_row4(a.pre + c, left);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[0] += y[r] * y[r];
                    s[1] += e[r] * y[r];
                }
            }
            if (a.block) {
                const f4 o = load_row4(a.block + base + c, left);
#pragma unroll
                for (int r = 0; r < 4; ++r) s[2] += o[r] * o[r];
            }
        }
        block_sums(s, lds);
        const float ry = 1.0f / sqrtf(s[0] * inv_n + a.epsilon), back_y = s[1] * inv_n * ry * ry;
        const float rb = 1.0f / sqrtf(s[2] * inv_n + a.epsilon);
        // what arrives at y, formed where it is needed; dx and dgate may be arrays that are read here only by the
        // thread that writes them
        auto total_of = [&](int c, int left) {
            f4 v = a.dy ? load_row4(a.dy + base + c, left) : f4{0.0f, 0.0f, 0.0f, 0.0f};
            if (a.pre)
                v += ry * (load_row4(a.dh + base + c, left) * load_row4(a.pre + c, left) -
                           load_row4(a.y + base + c, left) * back_y);
            return v;
        };
        float dn[1] = {0.0f};
        if (a.block)
            for (int c = threadIdx.x * 4; c < a.width; c += 4 * kBlock) {
                const int left = a.width - c;
                const f4 v = total_of(c, left), o = load_row4(a.block + base + c, left), w = load_row4(a.post + c, left);
                f4 z = {0.0f, 0.0f, 0.0f, 0.0f};
                if (a.gate) z = load_row4(a.gate + base + c, left);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (r < left) dn[0] += v[r] * (a.gate ? gate_value(a.act, z[r]) : 1.0f) * w[r] * o[r];
            }
        block_sums(dn, lds);
        const float back_b = dn[0] * inv_n * rb * rb;
        for (int c = threadIdx.x * 4; c < a.width; c += 4 * kBlock) {
            const int left = a.width - c;
            const f4 v = total_of(c, left);
            if (a.pre)
                store_row4(part + a.width + c,
                           load_row4(a.dh + base + c, left) * (load_row4(a.y + base + c, left) * ry), left, true);
            if (a.block) {
                const f4 o = load_row4(a.block + base + c, left), w = load_row4(a.post + c, left);
                f4 z = {0.0f, 0.0f, 0.0f, 0.0f}, dz, db, dw;
                if (a.gate) z = load_row4(a.gate + base + c, left);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float n = o[r] * rb, value = a.gate ? gate_value(a.act, z[r]) : 1.0f;
                    dz[r] = v[r] * (w[r] * n) * (a.gate ? gate_slope(a.act, z[r], value) : 0.0f);
                    dw[r] = v[r] * value * n;
                    db[r] = rb * (v[r] * value * w[r] - o[r] * back_b);
                }
                store_row4(part + c, dw, left, true);
                if (a.gate) store_row4(a.dgate + base + c, dz, left, a.accumulate);
                store_row4(a.dblock + base + c, db, left, a.accumulate);
            }
            store_row4(a.dx + base + c, a.residual_scale * v, left, a.accumulate);
        }
    }
}

// dpost[c], dpre[c] = the sum of the groups' parts: 64 columns per workgroup, its 16 rows of threads take every
// 16th group.
__global__ __launch_bounds__(1024) void gate_weights_kernel(const float* __restrict__ part, int64_t groups, int width,
                                                            float* __restrict__ dpost, float* __restrict__ dpre) {
    __shared__ float s[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), r = threadIdx.x >> 6;
    float v = 0.0f;
    if (c < 2 * width) {
        int64_t g = r;
        for (; g + 7 * 16 < groups; g += 8 * 16) {
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = part[(g + 16 * k) * 2 * width + c];
#pragma unroll
            for (int k = 0; k < 8; ++k) v += x[k];
        }
        for (; g < groups; g += 16) v += part[g * 2 * width + c];
    }
    s[r][threadIdx.x & 63] = v;
    __syncthreads();
    if (r || c >= 2 * width) return;
    v = 0.0f;
#pragma unroll
    for (int x = 0; x < 16; ++x) v += s[x][threadIdx.x];
    if (c < width) {
        if (dpost) dpost[c] = v;
    } else if (dpre) {
        dpre[c - width] = v;
    }
}

// Wider rows do not stay in registers, and are read again behind each reduction (2048 x 8192: 87 and 151 us, 2048 x 8196: 86 and
// 279 us; 64 rows: 7 and 20, 16 and 46 us); nor are vectors of four loaded from rows of fewer.
constexpr int kLongWidth = 8192;
inline bool any_width(int64_t width) { return width < 4 || width > kLongWidth; }

struct LaunchForward {
    const GateArgs& a;
    template <int TPR, int V> int run() const {
        constexpr int kThreads = kThreadsFor<TPR>;
        const unsigned grid = stream_grid(ceil_div(a.rows, kThreads / TPR));
        hipLaunchKernelGGL((gate_fwd_kernel<TPR, V>), dim3(grid), dim3(kThreads), 0, ctx().stream, a);
        return check_launch("gated_residual_forward");
    }
    int operator()() const {
        if (a.width <= 256) return run<64, 1>();
        if (a.width <= 512) return run<128, 1>();
        if (a.width <= 1024) return run<256, 1>();
        if (a.width <= 2048) return run<512, 1>();
        if (a.width <= 4096) return run<1024, 1>();
        return run<1024, 2>();
    }
};
// Workgroups of the backward pass: each leaves its part of the weights' gradients, so there are no more than fill the
// device.
struct LaunchBackward {
    const GateArgs& a;
    int64_t* groups;
    template <int TPR, int V> int run(void** part) {
        constexpr int kThreads = kThreadsFor<TPR>;
        const int64_t all = ceil_div(a.rows, kThreads / TPR), most = 4 * static_cast<int64_t>(ctx().num_cus) * kBlock / kThreads;
        *groups = ceil_div(all, ceil_div(all, most));              // as many rows for each, but for the last
        int st = pool_alloc_raw(static_cast<size_t>(*groups) * 2 * a.width * sizeof(float), part);
        if (st != 0) return st;
        GateArgs b = a;
        b.part = static_cast<float*>(*part);
        hipLaunchKernelGGL((gate_bwd_kernel<TPR, V>), dim3(static_cast<unsigned>(*groups)), dim3(kThreads), 0, ctx().stream, b);
        return check_launch("gated_residual_backward");
    }
    int operator()(void** part) {
        if (a.width <= 256) return run<64, 1>(part);
        if (a.width <= 512) return run<128, 1>(part);
        if (a.width <= 1024) return run<256, 1>(part);
        if (a.width <= 2048) return run<512, 1>(part);
        if (a.width <= 4096) return run<1024, 1>(part);
        return run<1024, 2>(part);
    }
};

int check_arrays(const char* fn, const void* const* required, int count) {
    for (int n = 0; n < count; ++n) {
        if (!required[n]) return set_error(BSHIP_ERR_NULL_POINTER, "%s: a required array is NULL", fn);
        if (reinterpret_cast<uintptr_t>(required[n]) & 3u)
            return set_error(BSHIP_ERR_BAD_POINTER, "%s: an array is not 4-byte aligned", fn);
    }
    return 0;
}
int check_shape(const char* fn, int64_t rows, int64_t width, int act, bool gate) {
    if (rows < 0 || width < 0 || width > (int64_t(1) << 26))
        return set_error(BSHIP_ERR_BAD_DIMENSION, "%s: sizes out of range", fn);
    if (gate && (act < BSHIP_ACT_SIGMOID || act > BSHIP_ACT_SWISH))
        return set_error(BSHIP_ERR_BAD_OP, "%s: no activation has code %d", fn, act);
    return 0;
}

}  // namespace
}  // namespace bship

using namespace bship;

extern "C" {

int bship_gated_residual_fwd_f32(int act, const float* block, const float* gate, const float* x, const float* post,
                                 const float* pre, float* y, float* h, int64_t rows, int64_t width,
                                 float residual_scale, float epsilon) {
    BSHIP_REQUIRE_INIT();
    int st = check_shape(__func__, rows, width, act, gate != nullptr);
    if (st != 0) return st;
    if (rows == 0 || width == 0) return 0;
    GateArgs a = {};
    a.block = block; a.gate = gate; a.x = x; a.post = post; a.pre = pre;
    a.y = y; a.h = h;
    a.rows = rows; a.width = static_cast<int>(width);
    a.act = act; a.residual_scale = residual_scale; a.epsilon = epsilon;
    const void* need[] = {x, block ? static_cast<const void*>(block) : x, block ? static_cast<const void*>(post) : x,
                          block ? static_cast<const void*>(y) : x, pre ? static_cast<const void*>(h) : x,
                          pre ? static_cast<const void*>(pre) : x, gate ? static_cast<const void*>(gate) : x};
    if ((st = check_arrays(__func__, need, 7)) != 0) return st;
    if (!block && (gate || !pre))
        return set_error(BSHIP_ERR_NULL_POINTER, "%s: without a block there is only the norm before the next one", __func__);
    if (any_width(width)) {
        hipLaunchKernelGGL(gate_fwd_long_kernel, dim3(stream_grid(rows)), dim3(kBlock), 0, ctx().stream, a);
        return check_launch("gated_residual_forward");
    }
    return LaunchForward{a}();
}

int bship_gated_residual_bwd_f32(int act, const float* block, const float* gate, const float* post, const float* pre,
                                 const float* y, const float* dy, const float* dh, float* dblock, float* dgate,
                                 float* dx, float* dpost, float* dpre, int64_t rows, int64_t width,
                                 float residual_scale, float epsilon, int accumulate) {
    BSHIP_REQUIRE_INIT();
    int st = check_shape(__func__, rows, width, act, gate != nullptr);
    if (st != 0) return st;
    if (width == 0) return 0;
    if (rows == 0) {
        if (dpost && (st = launch_fill(dpost, 0.0f, static_cast<size_t>(width))) != 0) return st;
        return dpre ? launch_fill(dpre, 0.0f, static_cast<size_t>(width)) : 0;
    }
    if (!block && (gate || !pre))
        return set_error(BSHIP_ERR_NULL_POINTER, "%s: without a block there is only the norm before the next one", __func__);
    const void* need[] = {dx, block ? static_cast<const void*>(block) : dx, block ? static_cast<const void*>(post) : dx,
                          block ? static_cast<const void*>(dblock) : dx, block ? static_cast<const void*>(dpost) : dx,
                          gate ? static_cast<const void*>(gate) : dx, gate ? static_cast<const void*>(dgate) : dx,
                          pre ? static_cast<const void*>(pre) : dx, pre ? static_cast<const void*>(y) : dx,
                          pre ? static_cast<const void*>(dh) : dx, pre ? static_cast<const void*>(dpre) : dx,
                          pre ? dx : static_cast<const void*>(dy), dy ? static_cast<const void*>(dy) : dx};
    if ((st = check_arrays(__func__, need, 13)) != 0) return st;
    GateArgs a = {};
    a.block = block; a.gate = gate; a.post = post; a.pre = pre;
    a.y = const_cast<float*>(y); a.dy = dy; a.dh = dh;
    a.dblock = dblock; a.dgate = dgate; a.dx = dx;
    a.rows = rows; a.width = static_cast<int>(width);
    a.act = act; a.residual_scale = residual_scale; a.epsilon = epsilon;
    a.accumulate = accumulate != 0;
    void* part = nullptr;
    int64_t groups = 0;
    if (any_width(width)) {
        groups = rows < 2 * ctx().num_cus ? rows : 2 * ctx().num_cus;
        st = pool_alloc_raw(static_cast<size_t>(groups) * 2 * static_cast<size_t>(width) * sizeof(float), &part);
        if (st != 0) return st;
        a.part = static_cast<float*>(part);
        hipLaunchKernelGGL(gate_bwd_long_kernel, dim3(static_cast<unsigned>(groups)), dim3(kBlock), 0, ctx().stream, a);
        st = check_launch("gated_residual_backward");
    } else {
        st = LaunchBackward{a, &groups}(&part);
    }
    if (st == 0) {
        hipLaunchKernelGGL(gate_weights_kernel, dim3(static_cast<unsigned>(ceil_div(2 * width, 64))), dim3(1024), 0,
                           ctx().stream, static_cast<const float*>(part), groups, a.width, block ? dpost : nullptr,
                           pre ? dpre : nullptr);
        st = check_launch("gated_residual_backward, weights");
    }
    (void)pool_free_raw(part);
    return st;
}

}  // extern "C"
