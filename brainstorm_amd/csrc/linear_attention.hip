// Linear attention with a decay for each head: a whole sequence forward and backward, and one step.
//
//   S_t = g S_{t-1} + k_t^T v_t        o_t = scale q_t S_t        (S: dk x dv, g: the head's decay)
//
// All arrays are (time, batch, heads * d): the layout of the framework's recurrent layers, a head's row of
// d floats every batch * heads * d floats. Row addresses promise 4-byte alignment only.
//
// One pass kernel serves the forward pass and the three gradients, because each of them is the same sum with
// other operands (W_ts = g^(t-s), s <= t):
//   o_t  = scale sum_s W_ts (q_t . k_s) v_s
//   dq_t = scale sum_s W_ts (do_t . v_s) k_s            q, k, v := do, v, k
//   dk_s = scale sum_t W_ts (v_s . do_t) q_t            q, k, v := v, do, q, time running backwards
//   dv_s = scale sum_t W_ts (k_s . q_t) do_t            q, k, v := k, q, do, time running backwards
// In the comments below q, k, v, o are the operands of the pass, i counts the features of q and k, j those of
// v and o, and p the positions in the direction of the pass.
//
// The pass goes through a sequence in chunks of 32 positions with the carried state in registers. It keeps
// the state BEFORE a position's own term, already decayed (C_p = g S_{p-1}), so that the two directions
// differ only in their ends: forwards C_0 = g * state and the new state is S of the last position, undecayed;
// backwards C_0 = gradient of the new state and the result is C behind the last position. For a chunk of n
// positions (a, b local positions):
//   o_a    = out_scale (g^a q_a C + sum_{b<=a} g^(a-b) (q_a . k_b) v_b)
//   C_next = g^n C + sum_b g^(n-b) k_b^T v_b
// Powers come from a table made by repeated squaring in float64, so every decay is allowed whose powers float32 holds,
// 0 and 1 included.
//
// The gradient of the decay is the sum over (t, s) of (t-s) g^(t-s-1) scale (q_t.k_s)(do_t.v_s). It is taken
// in the dq pass by carrying the derivative C' of the state by g beside the state (C'_next = g^n C' +
// n g^(n-1) C + sum_b (n-b) g^(n-b-1) k_b^T v_b), because forming it as a difference of sums weighted with t
// and with s loses as many digits as the sequence is longer than the decay's memory.
//
// What bounds it and what it takes (a large copy moves 5.1 TB/s on this card, a float32 product reaches 152 TFLOP/s):
//   one step, 4096 sequences of 128 x 128: the state in and out, 537 MB: 106 us, 5.1 TB/s; 8 sequences: a launch, 3.7 us
//   16 sequences of 8192 steps of 64: 70 us in three launches (states of the segments 22, scan 6, pass 46); 134 MB would
//     take 26 us, but a segment's chunks wait for each other
//   128 sequences of 1024 steps of 128: forward 151 us, backward 484; 30 GFLOP that cannot be left out take 198 us; matrix
//     cores 44 % (one wavefront a SIMD) to 55 % (two) busy, a quarter of the work is the derivative by the decay
//   800 sequences of 100 steps of 125, all scores: forward 66 us, backward 168 us
#include "common.h"

#include <cfloat>
#include <limits>

#pragma clang fp contract(fast)

namespace bship {
namespace {

constexpr int kChunk = 32;
constexpr int64_t kStepFloats = int64_t(1) << 25;      // batch * heads * d of a pass: 31 rows within 4 GiB
// Up to so many segments a pass adds up what the ones before leave by itself; the scan of more is a launch of its own (1024
// steps, 160 sequences of 64 features, 4 segments: 83 us forwards, with the scan 90; 64 sequences, 8 segments: 47 and 44; 64
// sequences of 128 features, 4 segments: 116 and 106 forwards, 304 and 314 backwards).
constexpr int kAddedUp = 4;
// Sequences of at most this many positions go position by position; from the next on a pass is as fast or faster (with states;
// positions 3, 4, 5 one by one against a pass: 163, 193, 222 against 168, 170, 170 us for 4096 sequences of 128 features, 7.0, 8.1,
// 9.0 against 8.5 us for 256 of 64).
constexpr int kStepMost = 3;

struct PassArgs {
    const float *q, *k, *v;
    float* out;
    const float *decay, *lengths;      // lengths: NULL = every sequence has `time` steps
    const float* init;                 // (batch, heads, di, dj) with strides si, sj; NULL = zeros
    float* fin;                        // the same for the state behind the last position; NULL = not wanted
    const float* z;                    // TAN: the array of o's shape that the derivative of o by g is multiplied with
    const float* dfin;                 // TAN: gradient of the final state (strides si, sj), or NULL
    double* slope;                     // TAN: one partial sum per workgroup
    float* seg;                        // what each segment leaves, or starts from: (batch*heads, segs, 1 or 2, di, dj)
    int64_t time, batch, heads;
    int di, dj, si, sj;
    int segs, seg_len;                 // segments of seg_len positions (a multiple of kChunk)
    int scanned;                       // `seg` holds the states that segments start from, not what they leave
    int tiles_j;                       // single steps: workgroups that share the columns of one head
    float kv_scale, out_scale;
    int reverse;
};

__device__ __forceinline__ double power(double g, int64_t n) {
    double r = 1.0;
    for (; n > 0; n >>= 1) {
        if (n & 1) r *= g;
        g *= g;
    }
    return r;
}

// x = g^n, rounded to T but to 0 only for g = 0: what it weighs has vanished all the same (T's least number is as near as
// 0), but an infinite state stays infinite, as step by step.
template <class T>
__device__ __forceinline__ T not_vanished(double x, double g, int n) {
    const T r = static_cast<T>(x);
    constexpr T least = std::numeric_limits<T>::denorm_min();
    return r != 0 || g == 0 ? r : g < 0 && (n & 1) ? -least : least;
}

// Steps of sequence b: lengths are float32 like the framework's labels, truncated; NaN counts as 0.
__device__ __forceinline__ int64_t sequence_length(const float* lengths, int64_t b, int64_t time) {
    if (!lengths) return time;
    const float x = lengths[b];
    if (!(x >= 1.0f)) return 0;
    return x >= static_cast<float>(time) ? time : static_cast<int64_t>(x);
}

// Four floats at p of which the first `left` exist (the others 0); 4-byte alignment.
__device__ __forceinline__ f4 load4(const float* p, int left) {
    if (left >= 4) return *reinterpret_cast<const f4u*>(p);
    f4 r = {0.0f, 0.0f, 0.0f, 0.0f};
    if (left > 0) r[0] = p[0];
    if (left > 1) r[1] = p[1];
    if (left > 2) r[2] = p[2];
    return r;
}
__device__ __forceinline__ void store4(float* p, f4 x, int left) {
    if (left >= 4) {
        *reinterpret_cast<f4u*>(p) = x;
        return;
    }
    if (left > 0) p[0] = x[0];
    if (left > 1) p[1] = x[1];
    if (left > 2) p[2] = x[2];
}

// D (16 x 16) += A (16 x 4) B (4 x 16) in float32: lane l holds A[l % 16][l / 16], B[l / 16][l % 16] and the four
// D[4 (l / 16) + r][l % 16]. With the four products of a 16-deep step taken over k = 4 (l / 16) + r, r = 0..3, the
// register r of a D tile is at once the operand of product r, as A (transposed) or as B: the state and the
// scores never leave their layout.
__device__ __forceinline__ f4 mfma(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Keeps what is written before this point before it: the next step's LDS reads then are under way during this step's
// products, and not all of them at once, each in registers of its own.
__device__ __forceinline__ void one_step_ahead() { __builtin_amdgcn_sched_barrier(0); }

// x, but the compiler does not know: what is formed from it is formed where it is used, a few instructions each time,
// and does not stay in registers through the loop over the chunks.
__device__ __forceinline__ int form_again(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// Several passes over the same sequences in one launch (blockIdx.y): more workgroups at once, one tail.
struct Passes {
    PassArgs pass[2];
};

// NI: tiles of 16 features of q and k held (di <= 16 NI). NW: wavefronts, each with 16 features of v, blockIdx.z: from which
// 16 NW of them on (dj <= 16 NW gridDim.z). TAN:
// with the derivative by the decay. STATE: only the state behind a segment that starts from zero.
//
// q and k of a chunk are staged in LDS (every wavefront reads all of both, as operands of the scores, of q C and of
// the state's update), fetched into registers one chunk ahead; v, which a wavefront needs only its own columns of, goes
// from memory into the operand registers directly. Scores are shared through LDS in the layout that the product with
// v takes them in. Per chunk and wavefront 8 NI + 8 NI + 12 + 3 NI / 2 (NW = 8) matrix instructions: the float32
// matrix rate is what bounds the pass at 128 features, memory at 64 and below.
template <int NI, int NW, bool TAN, bool STATE, bool NARROW>
__global__ __launch_bounds__(NW * kWave, NW == 8 ? (TAN ? 2 : 4) : NI > 4 ? 2 : TAN ? 3 : 4) void la_pass_kernel(Passes passes) {
    constexpr int LD = 16 * NI + 4;        // rows in LDS are 4 floats longer: 16 lanes in 16 rows, and 64 lanes in 16
                                           // floats each of rows 4 apart, meet all 64 banks
    constexpr int kThreads = NW * kWave;
    constexpr int kRows = kChunk * LD;
    __shared__ __attribute__((aligned(16))) float q_all[STATE ? 4 : 2 * kRows];
    __shared__ __attribute__((aligned(16))) float k_all[2 * kRows];
    __shared__ f4 score_s[STATE ? 1 : (TAN ? 6 : 3) * kWave];
    __shared__ float pw[kChunk + 1], sl[kChunk + 1];                     // g^n, n g^(n-1)
    __shared__ float pt[kChunk + 1], pl[kChunk + 1];                     // g^n in two parts of the same sign
    __shared__ float pk[kChunk + 1], sk[kChunk + 1];                     // kv_scale times g^n and n g^(n-1)
    __shared__ double part_s[NW];

    const PassArgs& a = passes.pass[blockIdx.y];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, lq = lane >> 4;
    const int seg = static_cast<int>(blockIdx.x % a.segs);
    if (STATE && seg + 1 == a.segs) return;               // nothing starts behind the last segment
    const int64_t bh = blockIdx.x / a.segs, b = bh / a.heads, h = bh % a.heads;
    const int64_t len = sequence_length(a.lengths, b, a.time);
    const int64_t p0 = static_cast<int64_t>(seg) * a.seg_len;
    const int64_t p1 = p0 + a.seg_len < a.time ? p0 + a.seg_len : a.time;
    const int64_t pe = len < p1 ? (len > p0 ? len : p0) : p1;      // valid positions [p0, pe)
    const double g = a.decay[h];
    const float gf = a.decay[h];
    const int j0 = 16 * (NW * static_cast<int>(blockIdx.z) + wave);       // this wavefront's columns
    const bool mine = j0 < a.dj;

    // Position p is time p forwards, len - 1 - p backwards. Rows are addressed from a chunk's earliest time, which is
    // the same for all lanes, by a 32-bit byte offset (a chunk spans less than 4 GiB: run_passes). Loads are made
    // without conditions, so that the ones of a chunk are all under way at once: positions, pieces and columns that do
    // not exist are taken from ones that do, and replaced by zeros or left out further on.
    const int64_t step_i = a.batch * a.heads * a.di, step_j = a.batch * a.heads * a.dj;
    const int64_t t0 = a.reverse ? len - 1 - p0 - (kChunk - 1) : p0;
    const int64_t move_i = (a.reverse ? -kChunk : kChunk) * step_i, move_j = (a.reverse ? -kChunk : kChunk) * step_j;
    const float *q = a.q + t0 * step_i + bh * a.di, *k = a.k + t0 * step_i + bh * a.di;
    const float* v = a.v + t0 * step_j + bh * a.dj + (mine ? j0 : 0);
    float* out = a.out + t0 * step_j + bh * a.dj + j0;
    const float* z = TAN ? a.z + t0 * step_j + bh * a.dj + j0 : nullptr;
    const uint32_t step_i32 = static_cast<uint32_t>(step_i) * 4, step_j32 = static_cast<uint32_t>(step_j) * 4;
    auto row_offset = [&](int row, uint32_t step) { return static_cast<uint32_t>(a.reverse ? kChunk - 1 - row : row) * step; };
    auto at_offset = [](const float* p, uint32_t offset) {
        return reinterpret_cast<const float*>(reinterpret_cast<const char*>(p) + offset);
    };
    constexpr int kRowQ = 4 * NI, kPieces = kChunk * kRowQ;              // 16-byte pieces of a row, of a chunk
    constexpr int kLoads = (kPieces + kThreads - 1) / kThreads;
    // column of piece e: the last one of a row whose length is no multiple of 4 ends with the row
    auto piece_col = [&](int e) {
        const int col = e % kRowQ * 4;
        return NARROW || col >= a.di ? 0 : col + 4 > a.di ? a.di - 4 : col;
    };

    // ---- rows of the next chunk, on their way from memory
    f4 q_n[STATE ? 1 : kLoads], k_n[kLoads];
    float v_n[2][4];
    // Pieces of one thread that lie in one column differ by whole rows; so do the rows of v. Their distances are scalars.
    constexpr bool kColumn = kThreads % kRowQ == 0;
    const uint32_t turn_j = a.reverse ? 0u - step_j32 : step_j32;
    const uint32_t turn_i = (a.reverse ? 0u - step_i32 : step_i32) * (kThreads / kRowQ);
    const uint32_t first_q = row_offset(tid / kRowQ % kChunk, step_i32) + 4 * piece_col(tid);
    const uint32_t first_v = row_offset(4 * lq, step_j32) + 4 * (l16 < a.dj - j0 ? l16 : 0);
    auto fetch = [&](int n) {                                            // the n positions of the chunk at q, k, v
        uint32_t off_q[kLoads], off_v[2][4];
        if (n == kChunk && kColumn && kPieces >= kThreads) {
#pragma unroll
            for (int m = 0; m < kLoads; ++m) off_q[m] = first_q + m * turn_i;
#pragma unroll
            for (int bt = 0; bt < 2; ++bt)
#pragma unroll
                for (int r = 0; r < 4; ++r) off_v[bt][r] = first_v + (16 * bt + r) * turn_j;
        } else {
            const int tid = form_again(threadIdx.x), l16 = tid & 15, lq = tid >> 4 & 3;
#pragma unroll
            for (int m = 0; m < kLoads; ++m) {
                const int row = (tid + m * kThreads) / kRowQ % kChunk;
                off_q[m] = row_offset(row < n ? row : n - 1, step_i32) + 4 * piece_col(tid + m * kThreads);
            }
#pragma unroll
            for (int bt = 0; bt < 2; ++bt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * bt + 4 * lq + r;
                    off_v[bt][r] = row_offset(row < n ? row : n - 1, step_j32) + 4 * (l16 < a.dj - j0 ? l16 : 0);
                }
        }
#pragma unroll
        for (int m = 0; m < kLoads; ++m) {
            if constexpr (NARROW) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t at = off_q[m] + 4 * (r < a.di ? r : 0);
                    k_n[m][r] = *at_offset(k, at);
                    if (!STATE) q_n[m][r] = *at_offset(q, at);
                }
            } else {
                k_n[m] = *reinterpret_cast<const f4u*>(at_offset(k, off_q[m]));
                if (!STATE) q_n[m] = *reinterpret_cast<const f4u*>(at_offset(q, off_q[m]));
            }
        }
#pragma unroll
        for (int bt = 0; bt < 2; ++bt)
#pragma unroll
            for (int r = 0; r < 4; ++r) v_n[bt][r] = *at_offset(v, off_v[bt][r]);
    };
    const auto positions = [&](int64_t pc) {                             // of the chunk pc behind p0
        return pe - p0 - pc < kChunk ? static_cast<int>(pe - p0 - pc) : kChunk;
    };
    if (p0 < pe) fetch(positions(0));
    // columns that a row does not have: zeros, which nothing overwrites
    for (int e = tid * 4; e < 2 * kRows; e += kThreads * 4) {
        *reinterpret_cast<f4*>(k_all + e) = f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (!STATE) *reinterpret_cast<f4*>(q_all + e) = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    if (tid <= kChunk) {
        const double x = power(g, tid);
        pw[tid] = not_vanished<float>(x, g, tid);
        // The first part is one unit less than the rounded power, so that half a unit at least is left for the second and both
        // have one sign: an infinite state stays one, where inf - inf or 0 inf would be NaN.
        const bool normal = fabsf(pw[tid]) > FLT_MIN;
        pt[tid] = normal ? __uint_as_float(__float_as_uint(pw[tid]) - 1) : pw[tid];
        pl[tid] = not_vanished<float>(normal ? x - pt[tid] : 0.0, g, tid);
        sl[tid] = tid ? static_cast<float>(tid * power(g, tid - 1)) : 0.0f;
        pk[tid] = a.kv_scale * pw[tid];
        sk[tid] = a.kv_scale * sl[tid];
    }

    // ---- the state: rows 16 it + 4 lq + r, column j0 + l16
    f4 c[NI], dc[TAN ? NI : 1];
    const int64_t per_state = static_cast<int64_t>(a.di) * a.dj;
    {
        const float *from = nullptr, *dfrom = nullptr;
        int row = a.si, column = a.sj;
        const int64_t each = per_state * (TAN ? 2 : 1);
        const float* slots = a.seg + bh * a.segs * each;             // not used with one segment
        if (!STATE && a.scanned) {
            from = slots + seg * each;
            dfrom = from + per_state;
            row = a.dj;
            column = 1;
        } else if (!STATE && a.init) {
            from = dfrom = a.init + bh * per_state;
        }
        auto read = [&](f4 (&to)[NI], const float* p, int row, int column) {
#pragma unroll
            for (int it = 0; it < NI; ++it)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * it + 4 * lq + r, j = j0 + l16;
                    to[it][r] = 0.0f;
                    if (i < a.di && j < a.dj) to[it][r] = p[i * row + j * column];
                }
        };
#pragma unroll
        for (int it = 0; it < NI; ++it) c[it] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (from) read(c, from, row, column);
        if constexpr (TAN) {
#pragma unroll
            for (int it = 0; it < NI; ++it) dc[it] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            if (from && (a.scanned || len > 0)) read(dc, dfrom, row, column);
        }
        if (!a.scanned && len > 0 && !a.reverse)
#pragma unroll
            for (int it = 0; it < NI; ++it) c[it] *= gf;
        // few segments: what the ones before leave is added up here
        if (!STATE && !a.scanned)
            for (int s = 0; s < seg; ++s) {
                const int64_t rest = len - static_cast<int64_t>(s) * a.seg_len;
                const int64_t steps = rest < 0 ? 0 : rest < a.seg_len ? rest : a.seg_len;
                const float w = not_vanished<float>(power(g, steps), g, static_cast<int>(steps));
                f4 u[NI];
                if constexpr (TAN) {
                    const float dw = steps ? static_cast<float>(steps * power(g, steps - 1)) : 0.0f;
                    read(u, slots + s * each + per_state, a.dj, 1);
#pragma unroll
                    for (int it = 0; it < NI; ++it) dc[it] = w * dc[it] + (dw * c[it] + u[it]);
                }
                read(u, slots + s * each, a.dj, 1);
#pragma unroll
                for (int it = 0; it < NI; ++it) c[it] = w * c[it] + u[it];
            }
    }
    double slope = 0.0;
    __syncthreads();
    // One chunk, of which the first 16 `tiles` positions can be valid.
    auto chunk = [&](auto tiles, int64_t pc) {
        constexpr int kTiles = decltype(tiles)::value;
        const int tid = form_again(threadIdx.x), lane = tid & 63, l16 = tid & 15, lq = tid >> 4 & 3;
        const int n = positions(pc);
        // behind the sequence's last position a forward pass leaves S, not g S
        const int m = n - (!STATE && !a.reverse && p0 + pc + n == len ? 1 : 0);
        // two buffers in turn: a wavefront may still read the last chunk's rows here, the ones before that nobody does
        float* const q_s = q_all + (STATE ? 0 : (pc / kChunk & 1) * kRows);
        float* const k_s = k_all + (pc / kChunk & 1) * kRows;
        if (n < kChunk) {
#pragma unroll
            for (int x = 0; x < kLoads; ++x)
                if ((tid + x * kThreads) / kRowQ % kChunk >= n) {
                    k_n[x] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                    if (!STATE) q_n[x] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                }
#pragma unroll
            for (int bt = 0; bt < 2; ++bt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * bt + 4 * lq + r >= n) v_n[bt][r] = 0.0f;
        }
#pragma unroll
        for (int x = 0; x < kLoads; ++x) {
            const int e = tid + x * kThreads, at = e / kRowQ % kChunk * LD + piece_col(e);
            if ((kPieces % kThreads && e >= kPieces) || e % kRowQ * 4 >= a.di) continue;
            if (NARROW) {
#pragma unroll
                for (int r = 0; r < 3; ++r)
                    if (r < a.di) {
                        if (!STATE) q_s[at + r] = q_n[x][r];
                        k_s[at + r] = k_n[x][r];
                    }
            } else if (a.di & 3) {             // pieces that do not begin at multiples of 16 bytes
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (!STATE) q_s[at + r] = q_n[x][r];
                    k_s[at + r] = k_n[x][r];
                }
            } else {
                if (!STATE) *reinterpret_cast<f4*>(q_s + at) = q_n[x];
                *reinterpret_cast<f4*>(k_s + at) = k_n[x];
            }
        }
        // v[b][j] for b = 16 bt + 4 lq + r, j = own column: an operand of both products that use v. Taken over here,
        // before the next loads are under way: behind them it would wait for them too.
        float v_r[2][4];
#pragma unroll
        for (int bt = 0; bt < 2; ++bt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                v_r[bt][r] = v_n[bt][r];
                asm volatile("" : "+v"(v_r[bt][r]));
            }
        __syncthreads();
        q += move_i;
        k += move_i;
        v += move_j;
        if (pc + kChunk < pe - p0) fetch(positions(pc + kChunk));

        f4 o[2], dz[2];
        if constexpr (!STATE) {
            // scores k_b . q_a g^(a-b) of the tiles (b, a) = (0, 0), (0, 1), (1, 1), one wavefront each
            if (wave < (kTiles == 2 ? 3 : 1)) {
                const int bt = wave >> 1, at = (wave + 1) >> 1;
                const float* kp = k_s + (16 * bt + l16) * LD + 4 * lq;
                const float* qp = q_s + (16 * at + l16) * LD + 4 * lq;
                f4 s = {0.0f, 0.0f, 0.0f, 0.0f}, s2 = s, kf[2], qf[2];
                kf[0] = *reinterpret_cast<const f4*>(kp);
                qf[0] = *reinterpret_cast<const f4*>(qp);
#pragma unroll
                for (int it = 0; it < NI; ++it) {
                    if (it + 1 < NI) {
                        kf[(it + 1) & 1] = *reinterpret_cast<const f4*>(kp + 16 * (it + 1));
                        qf[(it + 1) & 1] = *reinterpret_cast<const f4*>(qp + 16 * (it + 1));
                    }
                    one_step_ahead();
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        s = mfma(kf[it & 1][r], qf[it & 1][r], s);
                        s2 = mfma(kf[it & 1][r + 1], qf[it & 1][r + 1], s2);
                    }
                }
                f4 w, dw;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int e = 16 * (at - bt) + l16 - 4 * lq - r;      // a - b; below 0: 0 whatever the score
                    const float x = s[r] + s2[r];
                    w[r] = e >= 0 ? x * pk[e] : 0.0f;
                    dw[r] = e >= 0 ? x * sk[e] : 0.0f;
                }
                score_s[wave * kWave + lane] = w;
                if (TAN) score_s[(3 + wave) * kWave + lane] = dw;
            }
            // q C
            if (mine) {
#pragma unroll
                for (int at = 0; at < 2; ++at) o[at] = dz[at] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                {
                    f4 qf[2][2];
                    auto read = [&](int it) {
#pragma unroll
                        for (int at = 0; at < kTiles; ++at)
                            qf[it & 1][at] = *reinterpret_cast<const f4*>(q_s + (16 * at + l16) * LD + 16 * it + 4 * lq);
                    };
                    read(0);
#pragma unroll
                    for (int it = 0; it < NI; ++it) {
                        if (it + 1 < NI) read(it + 1);
                        one_step_ahead();
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int at = 0; at < kTiles; ++at) {
                                o[at] = mfma(c[it][r], qf[it & 1][at][r], o[at]);
                                if (TAN) dz[at] = mfma(dc[it][r], qf[it & 1][at][r], dz[at]);
                            }
                    }
                }
#pragma unroll
                for (int at = 0; at < 2; ++at) {
                    const float w = pw[16 * at + l16], dw = sl[16 * at + l16];
                    if (TAN) dz[at] = w * dz[at] + dw * o[at];
                    o[at] = w * o[at];
                }
            }
        }
        // C = g^m C + sum_b g^(m-b) k_b^T v_b. A chunk's products are summed apart and added once: onto the state itself each would
        // round against its magnitude. The sum is added behind other products, which run while it comes. It begins with the
        // smaller part of the power, w + wl: the same factor every 32 positions.
        const float w = pt[m], wl = pl[m], dw = sl[m];
        f4 u[2], du[2];
        auto add = [&](int it) {
            if (TAN) dc[it] = w * dc[it] + (dw * c[it] + du[it & 1]);
            c[it] = w * c[it] + u[it & 1];
        };
        if (mine) {
            float vw[2][4], vs[2][4];
#pragma unroll
            for (int bt = 0; bt < 2; ++bt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int e = m - (16 * bt + 4 * lq + r);       // below 0 only where v is 0
                    vw[bt][r] = pk[e > 0 ? e : 0] * v_r[bt][r];
                    if (TAN) vs[bt][r] = sk[e > 0 ? e : 0] * v_r[bt][r];
                }
            {
                float kf[2][8];
                auto read = [&](int it) {
#pragma unroll
                    for (int x = 0; x < 4 * kTiles; ++x)
                        kf[it & 1][x] = k_s[(16 * (x >> 2) + 4 * lq + (x & 3)) * LD + 16 * it + l16];
                };
                read(0);
#pragma unroll
                for (int it = 0; it < NI; ++it) {
                    if (it + 1 < NI) read(it + 1);
                    one_step_ahead();
                    u[it & 1] = wl * c[it];
                    if (TAN) du[it & 1] = wl * dc[it];
#pragma unroll
                    for (int x = 0; x < 4 * kTiles; ++x) {
                        u[it & 1] = mfma(kf[it & 1][x], vw[x >> 2][x & 3], u[it & 1]);
                        if (TAN) du[it & 1] = mfma(kf[it & 1][x], vs[x >> 2][x & 3], du[it & 1]);
                    }
                    if (it > 0) add(it - 1);
                }
                if constexpr (STATE) add(NI - 1);
            }
        }
        if constexpr (!STATE) {
            __syncthreads();                   // the scores are there
            if (!mine) return;
            // A product with a score of 0 would carry a NaN or an infinity of v to positions before it: such values
            // are left out of the products and added to their own and later positions one by one.
            float nothing = 0.0f;                      // a NaN if one of the values is not finite
#pragma unroll
            for (int bt = 0; bt < kTiles; ++bt)
#pragma unroll
                for (int r = 0; r < 4; ++r) nothing += 0.0f * v_r[bt][r];
            const bool all_finite = __all(nothing == 0.0f);
            if (!all_finite)
#pragma unroll
                for (int bt = 0; bt < kTiles; ++bt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) v_r[bt][r] = __builtin_isfinite(v_r[bt][r]) ? v_r[bt][r] : 0.0f;
            f4 ws[3], dws[3];
#pragma unroll
            for (int tile = 0; tile < (kTiles == 2 ? 3 : 1); ++tile) {
                ws[tile] = score_s[tile * kWave + lane];
                if (TAN) dws[tile] = score_s[(3 + tile) * kWave + lane];
            }
#pragma unroll
            for (int bt = 0; bt < kTiles; ++bt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int at = bt; at < kTiles; ++at) {
                        o[at] = mfma(v_r[bt][r], ws[bt + at][r], o[at]);
                        if (TAN) dz[at] = mfma(v_r[bt][r], dws[bt + at][r], dz[at]);
                    }
            add(NI - 1);
            const int left = a.dj - j0 - 4 * lq;
            if (!all_finite) {
                const float* here = v - move_j;
                const float* score = reinterpret_cast<const float*>(score_s);
                for (int x = 0; x < n; ++x) {
                    const f4 vx = load4(at_offset(here, row_offset(x, step_j32) + 16 * lq), left);
#pragma unroll
                    for (int at = 0; at < kTiles; ++at) {
                        if (16 * at + l16 < x) continue;
                        const int from = (((x >> 4) + at) * kWave + (x >> 2 & 3) * 16 + l16) * 4 + (x & 3);
                        const float wx = score[from], dwx = TAN ? score[from + 12 * kWave] : 0.0f;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (__builtin_isfinite(vx[r])) continue;
                            o[at][r] += wx * vx[r];
                            if (TAN) dz[at][r] += dwx * vx[r];
                        }
                    }
                }
            }
            // lane: position 16 at + l16, columns j0 + 4 lq .. + 3
#pragma unroll
            for (int at = 0; at < kTiles; ++at) {
                if (16 * at + l16 >= n) continue;
                const uint32_t row = row_offset(16 * at + l16, step_j32) + 16 * lq;
                store4(const_cast<float*>(at_offset(out, row)), a.out_scale * o[at], left);
                if (TAN) {
                    const f4 zx = load4(at_offset(z, row), left);
                    float s = 0.0f;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (r < left) s += zx[r] * dz[at][r];
                    slope += static_cast<double>(a.out_scale * s);
                }
            }
        }
    };
    int64_t pc = 0;
    for (; pe - p0 - pc > 16; pc += kChunk, out += move_j, z += TAN ? move_j : 0) chunk(std::integral_constant<int, 2>{}, pc);
    for (; pc < pe - p0; pc += 16) chunk(std::integral_constant<int, 1>{}, pc);

    if constexpr (STATE) {
#pragma unroll
        for (int it = 0; it < NI; ++it)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * it + 4 * lq + r, j = j0 + l16;
                if (i >= a.di || j >= a.dj) continue;
                float* s = a.seg + (bh * a.segs + seg) * per_state * (TAN ? 2 : 1) + i * a.dj + j;
                s[0] = c[it][r];
                if (TAN) s[per_state] = dc[it][r];
            }
        return;
    }
    // rows behind the sequence's end: there position p is time p in both directions
    for (int64_t p = (len > p0 ? len : p0) + wave; p < p1; p += NW)
        for (int j = 16 * NW * static_cast<int>(blockIdx.z) + lane; j < a.dj && j < 16 * NW * static_cast<int>(blockIdx.z + 1); j += kWave)
            a.out[(p * a.batch * a.heads + bh) * a.dj + j] = 0.0f;
    // the workgroup of the segment with the last position has the final state
    const bool last = len > 0 ? (pe == len && pe > p0) : seg == 0;
    const bool moved = len > 0;            // an empty sequence's state is the one it had, whatever the decay
    if (last && (a.fin || (TAN && a.dfin && moved))) {
#pragma unroll
        for (int it = 0; it < NI; ++it)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * it + 4 * lq + r, j = j0 + l16;
                if (i >= a.di || j >= a.dj) continue;
                const int64_t at = bh * per_state + i * a.si + j * a.sj;
                if (a.fin) a.fin[at] = c[it][r];
                if (TAN && a.dfin && moved) slope += static_cast<double>(a.dfin[at]) * dc[it][r];
            }
    }
    if constexpr (TAN) {
        for (int d = 1; d < kWave; d <<= 1) slope += __shfl_xor(slope, d);
        if (lane == 0) part_s[wave] = slope;
        __syncthreads();
        if (tid == 0) {
            double s = 0.0;
            for (int x = 0; x < NW; ++x) s += part_s[x];
            a.slope[blockIdx.x * gridDim.z + blockIdx.z] = s;
        }
    }
}

// Short sequences without a state before or behind them: all scores are formed, none goes through a state. With d
// features a position costs 4 d (T / 2) operations instead of the 4 d^2 + 128 d of a pass in chunks.
constexpr int kAllScores = 128;        // positions that the kernels below cover

// 32 rows of d floats on their way from memory into LDS, a thread's pieces of 16 bytes. Loads are made without conditions:
// rows behind the last are taken from it, and become zeros in LDS.
template <int N, int THREADS>
struct Rows {
    static constexpr int kRow = 4 * N, kPieces = kChunk * kRow, kLoads = (kPieces + THREADS - 1) / THREADS, LD = 16 * N + 4;
    f4 x[kLoads];

    // column of piece e: the last one of a row whose length is no multiple of 4 ends with the row
    static __device__ __forceinline__ int column(int e, int d) {
        const int col = e % kRow * 4;
        return col >= d ? 0 : col + 4 > d ? d - 4 : col;
    }
    __device__ __forceinline__ void fetch(const float* p, int64_t step, int d, int first, int len) {
        const int tid = form_again(threadIdx.x);
#pragma unroll
        for (int m = 0; m < kLoads; ++m) {
            const int e = tid + m * THREADS, row = first + e / kRow % kChunk;
            x[m] = *reinterpret_cast<const f4u*>(p + (row < len ? row : len - 1) * step + column(e, d));
        }
    }
    __device__ __forceinline__ void put(float* to, int d, int first, int len) const {
        const int tid = threadIdx.x;
#pragma unroll
        for (int m = 0; m < kLoads; ++m) {
            const int e = tid + m * THREADS;
            if ((kPieces % THREADS && e >= kPieces) || e % kRow * 4 >= d) continue;
            const f4 y = first + e / kRow < len ? x[m] : f4{0.0f, 0.0f, 0.0f, 0.0f};
            float* at = to + e / kRow * LD + column(e, d);
            if (d & 3) {                           // pieces that do not begin at multiples of 16 bytes
#pragma unroll
                for (int r = 0; r < 4; ++r) at[r] = y[r];
            } else {
                *reinterpret_cast<f4*>(at) = y;
            }
        }
    }
};

// A row's pieces 16 it + 4 lq as operands; 0 behind its d floats.
template <int N>
__device__ __forceinline__ void read_operand(f4 (&to)[N], const float* row, int d, int lq) {
#pragma unroll
    for (int it = 0; it < N; ++it) {
        const int col = 16 * it + 4 * lq;
        to[it] = *reinterpret_cast<const f4u*>(row + (col + 4 <= d ? col : d - 4));
    }
    // the piece with the row's end was read up to it
#pragma unroll
    for (int it = 0; it < N; ++it) {
        const int over = 16 * it + 4 * lq + 4 - d;
        f4 x = to[it];
        if (over == 1) x = f4{x[1], x[2], x[3], 0.0f};
        if (over == 2) x = f4{x[2], x[3], 0.0f, 0.0f};
        if (over == 3) x = f4{x[3], 0.0f, 0.0f, 0.0f};
        if (over > 3) x = f4{0.0f, 0.0f, 0.0f, 0.0f};
        to[it] = x;
    }
}

// 16 rows in LDS times one column: D[16 rows][column] of lane (lq, l16): rows 4 lq + r, the own position as column l16.
template <int N>
__device__ __forceinline__ f4 scores(const float* rows, const f4 (&own)[N], int l16, int lq) {
    const float* p = rows + l16 * (16 * N + 4) + 4 * lq;
    f4 s = {0.0f, 0.0f, 0.0f, 0.0f}, s2 = s, x[2];
    x[0] = *reinterpret_cast<const f4*>(p);
#pragma unroll
    for (int it = 0; it < N; ++it) {
        if (it + 1 < N) x[(it + 1) & 1] = *reinterpret_cast<const f4*>(p + 16 * (it + 1));
        one_step_ahead();
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
            s = mfma(x[it & 1][r], own[it][r], s);
            s2 = mfma(x[it & 1][r + 1], own[it][r + 1], s2);
        }
    }
    return s + s2;
}

// acc[j] += sum over 16 rows y in LDS of rows[y][j] w[y], w as `scores` leaves it. On the diagonal a weight of 0 would carry a
// NaN or an infinity to positions that do not see it: such values are left out of the products and added one by one to the
// positions that do, which are those from y on (EARLIER = false), or up to y.
template <int N, int LD, bool EARLIER>
__device__ __forceinline__ void add_rows(f4 (&acc)[N], const float (&w)[4], const float* rows, bool diagonal, int l16, int lq) {
    const float* p = rows + 4 * lq * LD + l16;
    float x[2][4];
    auto read = [&](int jt) {
#pragma unroll
        for (int r = 0; r < 4; ++r) x[jt & 1][r] = p[r * LD + 16 * jt];
    };
    read(0);
    float nothing = 0.0f;                          // a NaN if a value is not finite
#pragma unroll
    for (int jt = 0; jt < N; ++jt) {
        if (jt + 1 < N) read(jt + 1);
        one_step_ahead();
        if (diagonal)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                nothing += 0.0f * x[jt & 1][r];
                x[jt & 1][r] = __builtin_isfinite(x[jt & 1][r]) ? x[jt & 1][r] : 0.0f;
            }
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[jt] = mfma(x[jt & 1][r], w[r], acc[jt]);
    }
    if (__all(nothing == 0.0f)) return;
    for (int y = 0; y < 16; ++y) {
        // the weight of row y and this lane's column: lane 16 (y / 4) + l16, element y % 4
        const int from = 16 * (y >> 2) + l16;
        float wy = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float w0 = __shfl(w[r], from);
            if ((y & 3) == r) wy = w0;
        }
        if (EARLIER ? l16 > y : l16 < y) continue;
#pragma unroll
        for (int jt = 0; jt < N; ++jt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float xy = rows[y * LD + 16 * jt + 4 * lq + r];
                if (!__builtin_isfinite(xy)) acc[jt][r] += wy * xy;
            }
    }
}

// Forwards. A wavefront has the 16 positions of one tile: q as operands in registers, the sums over v as accumulators. The
// rows of k and v come through LDS in steps of 32 positions; a tile of scores (b, a) is at once the operand of its
// product with v. Tile n has n + 1 tiles of scores: wavefronts s and s + 4, which share a SIMD, take tiles whose work adds
// up to the same.
template <int NI, int NJ>
__global__ __launch_bounds__(8 * kWave, 4) void la_scores_kernel(PassArgs a) {
    constexpr int kThreads = 8 * kWave;
    using RowsK = Rows<NI, kThreads>;
    using RowsV = Rows<NJ, kThreads>;
    constexpr int kRowsK = kChunk * RowsK::LD, kRowsV = kChunk * RowsV::LD;
    __shared__ __attribute__((aligned(16))) float k_all[2 * kRowsK], v_all[2 * kRowsV];
    __shared__ float pk[kAllScores];                                 // kv_scale times g^n

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, lq = lane >> 4;
    const int64_t bh = blockIdx.x, b = bh / a.heads, h = bh % a.heads;
    const int len = static_cast<int>(sequence_length(a.lengths, b, a.time));
    const int tiles = (len + 15) >> 4;
    const int mine = wave < 4 ? tiles - 1 - wave : wave - 4 - (8 - tiles);       // the tile of this wavefront, or < 0
    const int p = mine >= 0 ? 16 * mine + l16 : 0;                               // this lane's position as a column
    const int64_t step_i = a.batch * a.heads * a.di, step_j = a.batch * a.heads * a.dj;
    const float *k = a.k + bh * a.di, *v = a.v + bh * a.dj;
    RowsK k_n;
    RowsV v_n;
    f4 qf[NI];
    if (len > 0) {
        k_n.fetch(k, step_i, a.di, 0, len);
        v_n.fetch(v, step_j, a.dj, 0, len);
        read_operand(qf, a.q + (p < len ? p : len - 1) * step_i + bh * a.di, a.di, lq);
    }
    if (tid < kAllScores) pk[tid] = a.kv_scale * static_cast<float>(power(static_cast<double>(a.decay[h]), tid));
    // columns that a row does not have: zeros, which nothing overwrites
    for (int e = tid * 4; e < 2 * kRowsK; e += kThreads * 4) *reinterpret_cast<f4*>(k_all + e) = f4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int e = tid * 4; e < 2 * kRowsV; e += kThreads * 4) *reinterpret_cast<f4*>(v_all + e) = f4{0.0f, 0.0f, 0.0f, 0.0f};
    f4 o[NJ];
#pragma unroll
    for (int jt = 0; jt < NJ; ++jt) o[jt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    __syncthreads();

    for (int first = 0; first < len; first += kChunk) {
        float* const k_s = k_all + (first / kChunk & 1) * kRowsK;
        float* const v_s = v_all + (first / kChunk & 1) * kRowsV;
        k_n.put(k_s, a.di, first, len);
        v_n.put(v_s, a.dj, first, len);
        __syncthreads();                       // two buffers: nobody reads the ones before the last any more
        if (first + kChunk < len) {
            k_n.fetch(k, step_i, a.di, first + kChunk, len);
            v_n.fetch(v, step_j, a.dj, first + kChunk, len);
        }
        for (int x = first; x < first + kChunk && x <= 16 * mine; x += 16) {
            const f4 s = scores<NI>(k_s + (x - first) * RowsK::LD, qf, l16, lq);
            float w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int e = p - x - 4 * lq - r;                        // a - b; below 0: 0 whatever the score
                w[r] = e >= 0 ? s[r] * pk[e] : 0.0f;
            }
            add_rows<NJ, RowsV::LD, false>(o, w, v_s + (x - first) * RowsV::LD, x == 16 * mine, l16, lq);
        }
    }

    // lane: position p, columns 16 jt + 4 lq .. + 3
    if (mine >= 0 && p < len)
#pragma unroll
        for (int jt = 0; jt < NJ; ++jt) {
            const int col = 16 * jt + 4 * lq;
            store4(a.out + p * step_j + bh * a.dj + col, a.out_scale * o[jt], a.dj - col);
        }
    // rows behind the sequence's end
    for (int64_t x = len + wave; x < a.time; x += 8)
        for (int j = lane; j < a.dj; j += kWave) a.out[x * step_j + bh * a.dj + j] = 0.0f;
}

// Backwards: all gradients from each score formed once. s_ab = q_a . k_b and p_ab = do_a . v_b (b <= a, W_ab = g^(a-b)) give
//   dv_b = scale sum_a W s do_a,   dk_b = scale sum_a W p q_a,   dq_a = scale sum_b W p k_b,
//   ddecay = scale sum (a-b) g^(a-b-1) s p,
// five products of tiles where the passes one by one take seven and read ten arrays instead of five.
//
// First the keys' gradients: wavefronts 2 n and 2 n + 1 have the positions of tile n as columns, one with k and the sums of dv,
// one with v and the sums of dk, while the rows of q and do come through LDS; both leave their scores there. Then the
// queries': wavefronts 2 n and 2 n + 1 have half of the features of dq each, k comes through LDS, and the scores are
// read back with rows and columns exchanged. Consecutive tiles lie on different SIMDs, so that the tiles that a step of 32
// positions reaches are spread evenly over them, but for the last ones.
struct BackArgs {
    const float *q, *k, *v, *dout, *decay, *lengths;
    float *dq, *dk, *dv;
    double* slope;                     // one partial sum per sequence, or NULL
    int64_t time, batch, heads;
    int di, dj;
    float scale;
};

template <int N, int TILES>
__global__ __launch_bounds__(2 * TILES * kWave, TILES == 4 && N == 8 ? 2 : 4) void la_scores_bwd_kernel(BackArgs a) {
    constexpr int kThreads = 2 * TILES * kWave, kHalf = N / 2;
    using R = Rows<N, kThreads>;
    constexpr int LD = R::LD, kRows = kChunk * LD;
    constexpr int kLD = 20, kTile = 16 * kLD, kPairs = TILES * (TILES + 1) / 2;      // tiles of scores: rows a, columns b
    __shared__ __attribute__((aligned(16))) float q_all[2 * kRows], do_all[2 * kRows];
    __shared__ __attribute__((aligned(16))) float s_all[kPairs * kTile], p_all[kPairs * kTile];
    __shared__ float pk[16 * TILES], sk[16 * TILES];                                 // scale times g^n and n g^(n-1)
    __shared__ double part_s[2 * TILES];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, lq = lane >> 4;
    const int64_t bh = blockIdx.x, b = bh / a.heads, h = bh % a.heads;
    const int len = static_cast<int>(sequence_length(a.lengths, b, a.time));
    const int mine = 16 * (wave >> 1), role = wave & 1;              // first position of the tile; 0: k and dv, 1: v and dk
    const int pos = mine + l16;
    const int64_t step_i = a.batch * a.heads * a.di, step_j = a.batch * a.heads * a.dj;
    const float *q = a.q + bh * a.di, *dout = a.dout + bh * a.dj, *k = a.k + bh * a.di, *v = a.v + bh * a.dj;
    R q_n, do_n;
    f4 own[N];
    if (len > 0) {
        q_n.fetch(q, step_i, a.di, 0, len);
        do_n.fetch(dout, step_j, a.dj, 0, len);
        const int row = pos < len ? pos : len - 1;
        read_operand(own, role ? v + row * step_j : k + row * step_i, role ? a.dj : a.di, lq);
    }
    if (tid < 16 * TILES) {
        const double g = a.decay[h];
        pk[tid] = a.scale * static_cast<float>(power(g, tid));
        sk[tid] = tid ? a.scale * static_cast<float>(tid * power(g, tid - 1)) : 0.0f;
    }
    // columns that a row does not have: zeros, which nothing overwrites
    for (int e = tid * 4; e < 2 * kRows; e += kThreads * 4) {
        *reinterpret_cast<f4*>(q_all + e) = f4{0.0f, 0.0f, 0.0f, 0.0f};
        *reinterpret_cast<f4*>(do_all + e) = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    f4 acc[N];
#pragma unroll
    for (int it = 0; it < N; ++it) acc[it] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    __syncthreads();

    int turn = 0;
    for (int first = 0; first < len; first += kChunk, turn ^= 1) {
        float *const q_s = q_all + turn * kRows, *const do_s = do_all + turn * kRows;
        q_n.put(q_s, a.di, first, len);
        do_n.put(do_s, a.dj, first, len);
        __syncthreads();                       // two buffers: nobody reads the ones before the last any more
        const bool more = first + kChunk < len;
        q_n.fetch(more ? q : k, step_i, a.di, more ? first + kChunk : 0, len);      // k: for what follows the loop
        do_n.fetch(dout, step_j, a.dj, first + kChunk, len);
        for (int x = first; x < first + kChunk; x += 16) {
            if (x < mine || x >= len) continue;
            const f4 s = scores<N>((role ? do_s : q_s) + (x - first) * LD, own, l16, lq);
            float* to = (role ? p_all : s_all) + ((x >> 4) * ((x >> 4) + 1) / 2 + (mine >> 4)) * kTile + 4 * lq * kLD + l16;
            float w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = x + 4 * lq + r, e = row - pos;
                const bool seen = e >= 0 && row < len;                   // otherwise 0 whatever the score
                w[r] = seen ? s[r] * pk[e] : 0.0f;
                to[r * kLD] = seen ? (role ? s[r] : s[r] * sk[e]) : 0.0f;
            }
            add_rows<N, LD, true>(acc, w, (role ? q_s : do_s) + (x - first) * LD, x == mine, l16, lq);
        }
    }
    // lane: position pos, columns 16 it + 4 lq .. + 3
    if (pos < len) {
        float* to = role ? a.dk + pos * step_i + bh * a.di : a.dv + pos * step_j + bh * a.dj;
        const int d = role ? a.di : a.dj;
#pragma unroll
        for (int it = 0; it < N; ++it) store4(to + 16 * it + 4 * lq, acc[it], d - 16 * it - 4 * lq);
    }

    f4 dq[kHalf];
#pragma unroll
    for (int it = 0; it < kHalf; ++it) dq[it] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    double slope = 0.0;
    for (int first = 0; first < len; first += kChunk, turn ^= 1) {
        float* const k_s = q_all + turn * kRows;
        q_n.put(k_s, a.di, first, len);
        __syncthreads();
        if (first + kChunk < len) q_n.fetch(k, step_i, a.di, first + kChunk, len);
        for (int x = first; x < first + kChunk; x += 16) {
            if (x > mine || mine >= len) continue;
            const int at = ((mine >> 4) * ((mine >> 4) + 1) / 2 + (x >> 4)) * kTile + l16 * kLD + 4 * lq;
            const f4 p = *reinterpret_cast<const f4*>(p_all + at);
            if (a.slope && (x >> 4 & 1) == role) {
                const f4 s = *reinterpret_cast<const f4*>(s_all + at);
                slope += static_cast<double>((p[0] * s[0] + p[1] * s[1]) + (p[2] * s[2] + p[3] * s[3]));
            }
            float w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int e = pos - x - 4 * lq - r;
                w[r] = e >= 0 ? p[r] * pk[e] : 0.0f;
            }
            add_rows<kHalf, LD, false>(dq, w, k_s + (x - first) * LD + role * 16 * kHalf, x == mine, l16, lq);
        }
    }
    if (pos < len)
#pragma unroll
        for (int it = 0; it < kHalf; ++it) {
            const int col = 16 * (role * kHalf + it) + 4 * lq;
            store4(a.dq + pos * step_i + bh * a.di + col, dq[it], a.di - col);
        }
    // rows behind the sequence's end
    for (int64_t x = len + wave; x < a.time; x += 2 * TILES) {
        for (int i = lane; i < a.di; i += kWave) a.dq[x * step_i + bh * a.di + i] = a.dk[x * step_i + bh * a.di + i] = 0.0f;
        for (int j = lane; j < a.dj; j += kWave) a.dv[x * step_j + bh * a.dj + j] = 0.0f;
    }
    if (a.slope) {
        for (int d = 1; d < kWave; d <<= 1) slope += __shfl_xor(slope, d);
        if (lane == 0) part_s[wave] = slope;
        __syncthreads();
        if (tid == 0) {
            double s = 0.0;
            for (int x = 0; x < 2 * TILES; ++x) s += part_s[x];
            a.slope[bh] = s;
        }
    }
}

constexpr int kScanned = 32;
// Turns the states that the segments leave when they start from zero into the states they start from. The loads of
// kScanned segments at a time do not wait for each other nor for the first state's and the decay's: a chain of a few loads is
// what it takes.
template <bool TAN>
__global__ __launch_bounds__(kBlock) void la_scan_kernel(Passes passes) {
    const PassArgs& a = passes.pass[blockIdx.z];
    const int per_state = a.di * a.dj, e = blockIdx.x * kBlock + threadIdx.x;
    if (e >= per_state) return;
    const int64_t step = per_state * (TAN ? 2 : 1);
    for (int64_t bh = blockIdx.y; bh < a.batch * a.heads; bh += gridDim.y) {
        const float decay = a.decay[bh % a.heads];
        const float init = a.init ? a.init[bh * per_state + e / a.dj * a.si + e % a.dj * a.sj] : 0.0f;
        float* slot = a.seg + bh * a.segs * step + e;
        float u[kScanned], du[kScanned];
        auto fetch = [&](int first) {
#pragma unroll
            for (int x = 0; x < kScanned; ++x) {
                const int64_t from = first + x < a.segs - 1 ? x : a.segs - 2 - first;     // the last one's was not formed
                u[x] = slot[from * step];
                if (TAN) du[x] = slot[from * step + per_state];
            }
        };
        fetch(0);
        const int64_t len = sequence_length(a.lengths, bh / a.heads, a.time);
        // segments before `whole` have all their positions, that one `rest` of them, those behind it none
        const int whole = static_cast<int>(len) / a.seg_len, rest = static_cast<int>(len) % a.seg_len;
        const double g = decay, full = not_vanished<double>(power(g, a.seg_len), g, a.seg_len);
        const double part = not_vanished<double>(power(g, rest), g, rest);
        const double dfull = a.seg_len * power(g, a.seg_len - 1), dpart = rest ? rest * power(g, rest - 1) : 0.0;
        double c = len > 0 && !a.reverse ? decay * init : init, dc = len > 0 ? init : 0.0f;
        for (int first = 0;;) {
#pragma unroll
            for (int x = 0; x < kScanned; ++x) {
                if (first + x >= a.segs) break;
                slot[x * step] = static_cast<float>(c);
                if (TAN) slot[x * step + per_state] = static_cast<float>(dc);
                const double w = first + x < whole ? full : first + x == whole ? part : 1.0;
                const double dw = first + x < whole ? dfull : first + x == whole ? dpart : 0.0;
                if (TAN) dc = w * dc + dw * c + du[x];
                c = w * c + u[x];
            }
            first += kScanned;
            slot += kScanned * step;
            if (first >= a.segs) break;
            fetch(first);
        }
    }
}

// ddecay[h] = the sum of the partial sums of head h, in a fixed order.
__global__ __launch_bounds__(kBlock) void la_slope_kernel(const double* __restrict__ part, float* __restrict__ ddecay,
                                                          int64_t batch, int64_t heads, int64_t per_head) {
    __shared__ double s[kBlock];
    const int64_t h = blockIdx.x;
    double x = 0.0;
    for (int64_t e = threadIdx.x; e < batch * per_head; e += kBlock)
        x += part[(e / per_head * heads + h) * per_head + e % per_head];
    s[threadIdx.x] = x;
    for (int d = kBlock / 2; d > 0; d >>= 1) {
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < d) s[threadIdx.x] += s[threadIdx.x + d];
    }
    if (threadIdx.x == 0) ddecay[h] = static_cast<float>(s[0]);
}

// Few positions: the recurrence itself, position by position, the state read and written once. LC lanes side by side
// hold 4 LC columns of a row, the workgroup's 256 / LC groups of lanes every (256 / LC)-th row.
template <int LC>
__global__ __launch_bounds__(kBlock) void la_step_kernel(PassArgs a) {
    constexpr int kGroups = kBlock / LC, kRows = 128 / kGroups;
    __shared__ f4 part_s[2][4][LC];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int group = tid / LC, j = static_cast<int>(blockIdx.x % a.tiles_j) * 4 * LC + tid % LC * 4;
    const int left = a.dj - j;
    const int64_t bh = blockIdx.x / a.tiles_j, b = bh / a.heads, h = bh % a.heads;
    const int64_t len = sequence_length(a.lengths, b, a.time);
    const float g = a.decay[h];
    const int64_t state = bh * a.di * a.dj + j;
    f4 s[kRows];
#pragma unroll
    for (int m = 0; m < kRows; ++m) {
        const int i = group + m * kGroups;
        s[m] = a.init && i < a.di ? load4(a.init + state + static_cast<int64_t>(i) * a.dj, left) : f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (int64_t t = 0; t < a.time; ++t) {
        const int64_t row = (t * a.batch * a.heads + bh);
        if (t >= len) {                                        // rows behind the end (len is the workgroup's)
            if (group == 0) store4(a.out + row * a.dj + j, f4{0.0f, 0.0f, 0.0f, 0.0f}, left);
            continue;
        }
        const float* q = a.q + row * a.di;
        const float* k = a.k + row * a.di;
        const f4 v = load4(a.v + row * a.dj + j, left);
        f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int m = 0; m < kRows; ++m) {
            const int i = group + m * kGroups;
            if (i >= a.di) continue;
            s[m] = g * s[m] + k[i] * v;
            o += q[i] * s[m];
        }
#pragma unroll
        for (int d = LC; d < kWave; d <<= 1)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] += __shfl_xor(o[r], d);
        if (lane < LC) part_s[t & 1][wave][lane] = o;
        __syncthreads();           // two buffers: the next position's sums are written while these are read
        if (tid < LC) {
            o = (part_s[t & 1][0][tid] + part_s[t & 1][1][tid]) + (part_s[t & 1][2][tid] + part_s[t & 1][3][tid]);
            store4(a.out + row * a.dj + j, a.out_scale * o, left);
        }
    }
    if (a.fin)
#pragma unroll
        for (int m = 0; m < kRows; ++m) {
            const int i = group + m * kGroups;
            if (i < a.di) store4(a.fin + state + static_cast<int64_t>(i) * a.dj, s[m], left);
        }
}

struct Scratch {
    void* p = nullptr;
    ~Scratch() { (void)pool_free_raw(p); }
    int get(size_t n) { return pool_alloc_raw(n, &p); }
};

template <int NI, bool TAN, bool STATE, bool NARROW = false>
void launch_pass(const Passes& p, int dj, dim3 grid) {
    if (dj <= 64 * static_cast<int>(grid.z)) hipLaunchKernelGGL((la_pass_kernel<NI, 4, TAN, STATE, NARROW>), grid, dim3(4 * kWave), 0, ctx().stream, p);
    else hipLaunchKernelGGL((la_pass_kernel<NI, 8, TAN, STATE, NARROW>), grid, dim3(8 * kWave), 0, ctx().stream, p);
}
template <bool TAN, bool STATE>
void launch_pass(const Passes& p, int di, int dj, dim3 grid) {
    if (di < 4) launch_pass<2, TAN, STATE, true>(p, dj, grid);       // all passes of the launch, or none (bwd)
    else if (di <= 32) launch_pass<2, TAN, STATE>(p, dj, grid);
    else if (di <= 64) launch_pass<4, TAN, STATE>(p, dj, grid);
    else if (di <= 96) launch_pass<6, TAN, STATE>(p, dj, grid);
    else launch_pass<8, TAN, STATE>(p, dj, grid);
}

template <int NI>
void launch_scores(const PassArgs& a, dim3 grid) {
    if (a.dj <= 32) hipLaunchKernelGGL((la_scores_kernel<NI, 2>), grid, dim3(8 * kWave), 0, ctx().stream, a);
    else if (a.dj <= 64) hipLaunchKernelGGL((la_scores_kernel<NI, 4>), grid, dim3(8 * kWave), 0, ctx().stream, a);
    else hipLaunchKernelGGL((la_scores_kernel<NI, 8>), grid, dim3(8 * kWave), 0, ctx().stream, a);
}
// 64 steps need half of the wavefronts and a quarter of the tiles: two workgroups share a compute unit up to 64 features (800
// sequences of 64 steps of 64 features: 40 us, with room for 128 steps 59).
template <int N>
void launch_scores_bwd(const BackArgs& a, dim3 grid) {
    if (a.time <= kAllScores / 2) hipLaunchKernelGGL((la_scores_bwd_kernel<N, 4>), grid, dim3(8 * kWave), 0, ctx().stream, a);
    else if constexpr (N > 2) hipLaunchKernelGGL((la_scores_bwd_kernel<N, 8>), grid, dim3(16 * kWave), 0, ctx().stream, a);
}

int check_steps(int64_t sequences, int di, int dj) {
    if (sequences * (di > dj ? di : dj) > kStepFloats)
        return set_error(BSHIP_ERR_UNSUPPORTED, "linear attention: more than %lld features in a time step",
                         static_cast<long long>(kStepFloats));
    return 0;
}

// A launch has fewer than 2^32 threads.
int check_blocks(int64_t blocks, int threads) {
    if (blocks > 0xffffffffll / threads)
        return set_error(BSHIP_ERR_BAD_DIMENSION, "linear attention: %lld workgroups exceed one launch",
                         static_cast<long long>(blocks));
    return 0;
}

int sum_slopes(const Scratch& parts, float* ddecay, int64_t batch, int64_t heads, int64_t per_head) {
    hipLaunchKernelGGL(la_slope_kernel, dim3(static_cast<unsigned>(heads)), dim3(kBlock), 0, ctx().stream,
                       static_cast<const double*>(parts.p), ddecay, batch, heads, per_head);
    return check_launch("linear attention, decay gradient");
}

int run_scores(const PassArgs& a) {
    const int64_t sequences = a.batch * a.heads;
    int st = check_steps(sequences, a.di, a.dj);
    if (st != 0 || (st = check_blocks(sequences, 8 * kWave)) != 0) return st;
    const dim3 grid(static_cast<unsigned>(sequences));
    if (a.di <= 32) launch_scores<2>(a, grid);
    else if (a.di <= 64) launch_scores<4>(a, grid);
    else launch_scores<8>(a, grid);
    return check_launch("linear attention, all scores");
}

int run_scores_bwd(BackArgs a, float* ddecay) {
    const int64_t sequences = a.batch * a.heads;
    int st = check_steps(sequences, a.di, a.dj);
    if (st != 0 || (st = check_blocks(sequences, 16 * kWave)) != 0) return st;
    Scratch slope;
    if (ddecay && (st = slope.get(sequences * sizeof(double))) != 0) return st;
    a.slope = static_cast<double*>(slope.p);
    const int d = a.di > a.dj ? a.di : a.dj;
    const dim3 grid(static_cast<unsigned>(sequences));
    if (d <= 32) launch_scores_bwd<2>(a, grid);
    else if (d <= 64) launch_scores_bwd<4>(a, grid);
    else launch_scores_bwd<8>(a, grid);
    st = check_launch("linear attention, gradients from all scores");
    return st != 0 || !ddecay ? st : sum_slopes(slope, ddecay, a.batch, a.heads, 1);
}

// `count` passes over the same sequences side by side. ddecay: with the derivative by the decay (one pass).
int run_passes(Passes p, int count, float* ddecay) {
    const PassArgs& a = p.pass[0];
    const int64_t sequences = a.batch * a.heads;
    int st = check_steps(sequences, a.di, a.dj);
    if (st != 0) return st;
    int di = 0, dj = 0;
    for (int n = 0; n < count; ++n) {
        di = p.pass[n].di > di ? p.pass[n].di : di;
        dj = p.pass[n].dj > dj ? p.pass[n].dj : dj;
    }
    // Eight wavefronts for every compute unit (4, 8 and 16 of them: 94, 65 and 74 us forwards for 16 sequences of 2048 steps
    // of 128 features, 87, 78 and 93 for 16 of 8192 steps of 64): where there are fewer sequences, the time axis is cut, into
    // segments of 64 positions at least (37 us, with 128 positions 48, for 15 sequences of 777 steps of 72 features; 32
    // positions save nothing there and cost 10 % elsewhere). More than the scan loads at once, only of 128 (8 sequences of
    // 4000 steps of 64 features: 44 us, with 64 positions 54).
    const int64_t cus = ctx().num_cus, workgroups = sequences * count;
    int64_t segs = ceil_div(cus * (dj <= 64 ? 2 : 1), workgroups), parts = 1;
    int64_t most = ceil_div(a.time, 2 * kChunk);
    if (most > kScanned) most = kScanned;
    if (most < ceil_div(a.time, 4 * kChunk)) most = ceil_div(a.time, 4 * kChunk);
    if (segs > most) segs = most;
    if (segs < 1) segs = 1;
    if (dj > 64) {
        // Two workgroups with half of the columns each, instead of two segments, of which the second waits for the first's
        // state (1024 steps, 128 and 192 sequences of 128 features: 153 and 231 us forwards, with segments 175 and 297), and
        // where the time axis cannot be cut further (4 sequences of 300 steps: 30 us, whole 36).
        if (segs == 2) parts = 2, segs = 1;
        else if (2 * workgroups * segs <= cus) parts = 2;
    } else if (4 * workgroups >= 5 * cus) {
        segs = 1;      // (64 features, 320 and 448 sequences of 1024 steps: 142 and 146 us, with two segments 146 and 184; 160: 106, 84)
    }
    int64_t seg_len = ceil_div(ceil_div(a.time, segs), kChunk) * kChunk;
    if (seg_len < kChunk) seg_len = kChunk;
    segs = a.time > 0 ? ceil_div(a.time, seg_len) : 1;
    if ((st = check_blocks(sequences * segs, 8 * kWave)) != 0) return st;
    const size_t states = static_cast<size_t>(sequences) * segs * a.di * a.dj * (ddecay ? 2 : 1);
    Scratch seg, slope;
    if (segs > 1) {
        st = seg.get(states * count * sizeof(float));
        if (st != 0) return st;
    }
    if (ddecay) {
        st = slope.get(sequences * segs * parts * sizeof(double));
        if (st != 0) return st;
    }
    // A state that is replaced has been read by all segments before the last one writes it only if the scan has read it.
    bool scanned = segs > kAddedUp;
    for (int n = 0; n < count; ++n) scanned = scanned || (segs > 1 && p.pass[n].init && p.pass[n].init == p.pass[n].fin);
    for (int n = 0; n < count; ++n) {
        p.pass[n].segs = static_cast<int>(segs);
        p.pass[n].seg_len = static_cast<int>(seg_len);
        p.pass[n].scanned = scanned;
        p.pass[n].seg = segs > 1 ? static_cast<float*>(seg.p) + n * states : nullptr;
        p.pass[n].slope = static_cast<double*>(slope.p);
    }
    const dim3 grid(static_cast<unsigned>(sequences * segs), static_cast<unsigned>(count), static_cast<unsigned>(parts));
    if (segs > 1) {
        if (ddecay) launch_pass<true, true>(p, di, dj, grid);
        else launch_pass<false, true>(p, di, dj, grid);
        st = check_launch("linear attention, segment states");
        if (st != 0) return st;
    }
    if (scanned) {
        const int64_t rows = sequences < 32768 ? sequences : 32768;
        const dim3 elements(static_cast<unsigned>(ceil_div(a.di * a.dj, kBlock)), static_cast<unsigned>(rows),
                          static_cast<unsigned>(count));
        if (ddecay) hipLaunchKernelGGL((la_scan_kernel<true>), elements, dim3(kBlock), 0, ctx().stream, p);
        else hipLaunchKernelGGL((la_scan_kernel<false>), elements, dim3(kBlock), 0, ctx().stream, p);
        st = check_launch("linear attention, scan");
        if (st != 0) return st;
    }
    if (ddecay) launch_pass<true, false>(p, di, dj, grid);
    else launch_pass<false, false>(p, di, dj, grid);
    st = check_launch("linear attention");
    return st != 0 || !ddecay ? st : sum_slopes(slope, ddecay, a.batch, a.heads, segs * parts);
}

int run_steps(PassArgs a) {
    const int64_t sequences = a.batch * a.heads;
    // 64 columns for a workgroup where that still makes many of them, 16 otherwise (one step, heads of 64 features: 16.2 against
    // 18.0 us for 2048 sequences, 6.4 against 6.1 for 512; 112 us for 4096 sequences of 128 features)
    const bool wide = sequences * ceil_div(a.dj, 64) >= 4 * static_cast<int64_t>(ctx().num_cus);
    a.tiles_j = static_cast<int>(ceil_div(a.dj, wide ? 64 : 16));
    int st = check_blocks(sequences * a.tiles_j, kBlock);
    if (st != 0) return st;
    const dim3 grid(static_cast<unsigned>(sequences * a.tiles_j));
    if (wide) hipLaunchKernelGGL((la_step_kernel<16>), grid, dim3(kBlock), 0, ctx().stream, a);
    else hipLaunchKernelGGL((la_step_kernel<4>), grid, dim3(kBlock), 0, ctx().stream, a);
    return check_launch("linear attention, steps");
}

int check_all(const char* fn, const void* const* ptrs, int count) {
    for (int n = 0; n < count; ++n) {
        if (!ptrs[n]) return set_error(BSHIP_ERR_NULL_POINTER, "%s: a required array is NULL", fn);
        if (reinterpret_cast<uintptr_t>(ptrs[n]) & 3u)
            return set_error(BSHIP_ERR_BAD_POINTER, "%s: an array is not 4-byte aligned", fn);
    }
    return 0;
}
// Arrays that may be NULL.
int check_given(const char* fn, const void* const* ptrs, int count) {
    for (int n = 0; n < count; ++n)
        if (reinterpret_cast<uintptr_t>(ptrs[n]) & 3u)
            return set_error(BSHIP_ERR_BAD_POINTER, "%s: an array is not 4-byte aligned", fn);
    return 0;
}
int check_dims(const char* fn, int64_t time, int64_t batch, int64_t heads, int64_t dk, int64_t dv) {
    if (time < 0 || batch < 0 || heads < 0 || dk < 1 || dv < 1 || time > (int64_t(1) << 30) || batch > (int64_t(1) << 30) ||
        heads > (int64_t(1) << 16) || batch * heads > 0x7fffffff)
        return set_error(BSHIP_ERR_BAD_DIMENSION, "%s: sizes out of range", fn);
    if (dk > 128 || dv > 128)
        return set_error(BSHIP_ERR_UNSUPPORTED, "%s: heads of %lld and %lld features: 128 are the most", fn,
                         static_cast<long long>(dk), static_cast<long long>(dv));
    return 0;
}

}  // namespace
}  // namespace bship

using namespace bship;

extern "C" {

int bship_linear_attention_fwd_f32(const float* q, const float* k, const float* v, const float* decay,
                                   const float* lengths, const float* state, float* out, float* new_state, int64_t time,
                                   int64_t batch, int64_t heads, int64_t dk, int64_t dv, float scale) {
    BSHIP_REQUIRE_INIT();
    int st = check_dims(__func__, time, batch, heads, dk, dv);
    if (st != 0) return st;
    if (batch * heads == 0) return 0;
    const void* need[] = {q, k, v, out, decay};
    if (time > 0 && (st = check_all(__func__, need, 5)) != 0) return st;
    const void* given[] = {decay, lengths, state, new_state};
    if ((st = check_given(__func__, given, 4)) != 0) return st;
    PassArgs a = {};
    a.q = q; a.k = k; a.v = v; a.out = out;
    a.decay = decay; a.lengths = lengths;
    a.init = state; a.fin = new_state;
    a.time = time; a.batch = batch; a.heads = heads;
    a.di = static_cast<int>(dk); a.dj = static_cast<int>(dv);
    a.si = static_cast<int>(dv); a.sj = 1;
    a.kv_scale = 1.0f; a.out_scale = scale;
    if (time == 0 && !new_state) return 0;
    BSHIP_REQUIRE_PTR(decay);
    if (time <= kStepMost) return run_steps(a);
    // all scores where that is less work than a state: up to 1.5 d steps (800 sequences, chunks against scores: 64 features, 64, 96
    // and 128 steps, 22.4, 30.0, 37.4 against 19.6, 29.8, 42.0 us; 32 features, 32 and 64 steps, 8.2, 11.7 against 8.1, 12.6;
    // 125 features, 128 steps, 103 against 75)
    if (time <= kAllScores && !state && !new_state && dk >= 4 && dv >= 4 && time * (dk + dv) <= 3 * dk * dv)
        return run_scores(a);
    return run_passes(Passes{{a}}, 1, nullptr);
}

int bship_linear_attention_bwd_f32(const float* q, const float* k, const float* v, const float* decay,
                                   const float* lengths, const float* state, const float* dout, const float* dnew_state,
                                   float* dq, float* dk_out, float* dv_out, float* ddecay, float* dstate, int64_t time,
                                   int64_t batch, int64_t heads, int64_t dk, int64_t dv, float scale) {
    BSHIP_REQUIRE_INIT();
    int st = check_dims(__func__, time, batch, heads, dk, dv);
    if (st != 0) return st;
    if (heads == 0) return 0;
    if (batch == 0) return ddecay ? launch_fill(ddecay, 0.0f, static_cast<size_t>(heads)) : 0;
    BSHIP_REQUIRE_PTR(decay);
    const void* need[] = {q, k, v, dout, dq, dk_out, dv_out};
    if (time > 0 && (st = check_all(__func__, need, 7)) != 0) return st;
    const void* given[] = {decay, lengths, state, dnew_state, ddecay, dstate};
    if ((st = check_given(__func__, given, 6)) != 0) return st;
    // The gradients take more passes, so that all scores win up to 64 steps whatever the features (800 sequences of 16: 28.8
    // against 31.0 us) and up to 128 with more than 32 (64 and 125 features: 117 against 124, 196 against 392 us; 32: 84
    // against 61).
    if (time > 0 && time <= (dk > 32 || dv > 32 ? kAllScores : kAllScores / 2) && !state && !dnew_state && !dstate && dk >= 4 &&
        dv >= 4)
        return run_scores_bwd(BackArgs{q, k, v, dout, decay, lengths, dq, dk_out, dv_out, nullptr, time, batch, heads,
                                       static_cast<int>(dk), static_cast<int>(dv), scale}, ddecay);
    PassArgs a = {};
    a.decay = decay; a.lengths = lengths;
    a.time = time; a.batch = batch; a.heads = heads;
    // dq: q, k, v := do, v, k; the state is transposed
    a.q = dout; a.k = v; a.v = k; a.out = dq;
    a.init = state;
    a.di = static_cast<int>(dv); a.dj = static_cast<int>(dk);
    a.si = 1; a.sj = static_cast<int>(dv);
    a.kv_scale = 1.0f; a.out_scale = scale;
    a.z = q;
    a.dfin = dnew_state;
    if ((st = run_passes(Passes{{a}}, 1, ddecay)) != 0) return st;
    // dk: v, do, q backwards, from the transposed gradient of the new state
    Passes back = {{a, a}};
    PassArgs& pk = back.pass[0];
    pk.q = v; pk.k = dout; pk.v = q; pk.out = dk_out;
    pk.init = dnew_state;
    pk.dfin = nullptr;
    pk.kv_scale = scale; pk.out_scale = 1.0f;
    pk.reverse = 1;
    // dv: k, q, do backwards; what is left behind the first step is the gradient of the state
    PassArgs& pv = back.pass[1];
    pv = pk;
    pv.q = k; pv.k = q; pv.v = dout; pv.out = dv_out;
    pv.fin = dstate;
    pv.di = static_cast<int>(dk); pv.dj = static_cast<int>(dv);
    pv.si = static_cast<int>(dv); pv.sj = 1;
    // One after the other: if both passes read what the second overwrites, or only one of them has rows of fewer than
    // four floats, which another kernel takes.
    if ((dstate && dstate == dnew_state) || (dk < 4) != (dv < 4)) {
        if ((st = run_passes(Passes{{pk}}, 1, nullptr)) != 0) return st;
        return run_passes(Passes{{pv}}, 1, nullptr);
    }
    return run_passes(back, 2, nullptr);
}

}  // extern "C"
