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
// Powers come from a table made by repeated squaring in float64, so every decay is allowed, 0 and 1 included.
//
// The gradient of the decay is the sum over (t, s) of (t-s) g^(t-s-1) scale (q_t.k_s)(do_t.v_s). It is taken
// in the dq pass by carrying the derivative C' of the state by g beside the state (C'_next = g^n C' +
// n g^(n-1) C + sum_b (n-b) g^(n-b-1) k_b^T v_b), because forming it as a difference of sums weighted with t
// and with s loses as many digits as the sequence is longer than the decay's memory.
#include "common.h"

#pragma clang fp contract(fast)

namespace bship {
namespace {

constexpr int kChunk = 32;
constexpr int kStepMost = 4;      // sequences of at most this many positions go position by position

struct PassArgs {
    const float *q, *k, *v;
    float* out;
    const float *decay, *lengths;      // lengths: NULL = every sequence has `time` steps
    const float* init;                 // (batch, heads, di, dj) with strides si, sj; NULL = zeros
    float* fin;                        // the same for the state behind the last position; NULL = not wanted
    const float* z;                    // TAN: the array of o's shape that the derivative of o by g is multiplied with
    const float* dfin;                 // TAN: gradient of the final state (strides si, sj), or NULL
    double* slope;                     // TAN: one partial sum per workgroup
    float* seg;                        // states at the beginning of each segment: (batch*heads, segs, 1 or 2, di, dj)
    int64_t time, batch, heads;
    int di, dj, si, sj;
    int segs, seg_len;                 // segments of seg_len positions (a multiple of kChunk)
    int tiles_j;                       // workgroups that share the columns of one head
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

// NI: tiles of 16 features of q and k held (di <= 16 NI); NJ: tiles of 16 features of v per wavefront (a
// workgroup of four wavefronts has 64 NJ of them); TAN: with the derivative by the decay; STATE: only the
// state behind a segment that starts from zero.
template <int NI, int NJ, bool TAN, bool STATE>
__global__ __launch_bounds__(kBlock) void la_pass_kernel(PassArgs a) {
    constexpr int LD = 16 * NI + 4;        // rows of q and k in LDS: 4 floats longer, so that 16 lanes in 16 rows and
    constexpr int LDV = 64 * NJ + 4;       // 64 lanes in 4 x 16 floats of rows 4 apart each meet 64 banks
    __shared__ float q_s[STATE ? 4 : kChunk * LD];
    __shared__ float k_s[kChunk * LD];
    __shared__ float v_s[kChunk * LDV];
    __shared__ f4 score_s[STATE ? 1 : (TAN ? 6 : 3) * kWave];
    __shared__ float pw[kChunk + 1], sl[kChunk + 1];     // g^n and n g^(n-1)
    __shared__ double part_s[4];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int l16 = lane & 15, lq = lane >> 4;
    const int jt0 = static_cast<int>(blockIdx.x % a.tiles_j) * 64 * NJ;
    const int64_t rest = blockIdx.x / a.tiles_j;
    const int seg = static_cast<int>(rest % a.segs);
    if (STATE && seg + 1 == a.segs) return;               // nothing starts behind the last segment
    const int64_t bh = rest / a.segs, b = bh / a.heads, h = bh % a.heads;
    const int64_t len = sequence_length(a.lengths, b, a.time);
    const int64_t p0 = static_cast<int64_t>(seg) * a.seg_len;
    const int64_t p1 = p0 + a.seg_len < a.time ? p0 + a.seg_len : a.time;
    const int64_t pe = len < p1 ? (len > p0 ? len : p0) : p1;      // valid positions [p0, pe)
    const double g = a.decay[h];
    const float gf = a.decay[h];
    const int ni = (a.di + 15) >> 4;
    const int dj = a.dj - jt0;                                     // columns from this workgroup's first on

    const int64_t step_i = a.batch * a.heads * a.di, step_j = a.batch * a.heads * a.dj;
    const float* q = a.q + bh * a.di;
    const float* k = a.k + bh * a.di;
    const float* v = a.v + bh * a.dj + jt0;

    if (tid <= kChunk) {
        pw[tid] = static_cast<float>(power(g, tid));
        sl[tid] = tid ? static_cast<float>(tid * power(g, tid - 1)) : 0.0f;
    }

    // ---- the state: tile (it, jt) of this wavefront's columns 16 (4 jt + wave) .. + 15
    f4 c[NI][NJ], dc[TAN ? NI : 1][NJ];
    const int64_t per_state = static_cast<int64_t>(a.di) * a.dj;
#pragma unroll
    for (int it = 0; it < NI; ++it)
#pragma unroll
        for (int jt = 0; jt < NJ; ++jt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * it + 4 * lq + r, j = 16 * (4 * jt + wave) + l16;
                float x = 0.0f, dx = 0.0f;
                if (!STATE && i < a.di && j < dj) {
                    if (a.segs > 1) {
                        const float* s = a.seg + (bh * a.segs + seg) * per_state * (TAN ? 2 : 1) +
                                         static_cast<int64_t>(i) * a.dj + jt0 + j;
                        x = s[0];
                        if (TAN) dx = s[per_state];
                    } else if (a.init) {
                        const float s = a.init[bh * per_state + static_cast<int64_t>(i) * a.si +
                                               static_cast<int64_t>(jt0 + j) * a.sj];
                        x = len > 0 && !a.reverse ? gf * s : s;
                        if (TAN) dx = len > 0 ? s : 0.0f;
                    }
                }
                c[it][jt][r] = x;
                if (TAN) dc[it][jt][r] = dx;
            }
    double slope = 0.0;

    // ---- rows of the next chunk, on their way from memory
    constexpr int kRowQ = 4 * NI, kRowV = 16 * NJ;                       // 16-byte pieces of a row
    constexpr int kLoadQ = kChunk * kRowQ / kBlock, kLoadV = kChunk * kRowV / kBlock;
    static_assert(kChunk * kRowQ % kBlock == 0 && kChunk * kRowV % kBlock == 0, "whole pieces per thread");
    f4 q_n[STATE ? 1 : kLoadQ], k_n[kLoadQ], v_n[kLoadV];
    auto time_of = [&](int64_t p) { return a.reverse && p < len ? len - 1 - p : p; };
    auto fetch = [&](int64_t pc) {
#pragma unroll
        for (int m = 0; m < kLoadQ; ++m) {
            const int e = tid + m * kBlock, row = e / kRowQ, col = e % kRowQ * 4;
            const int64_t p = pc + row;
            const bool valid = p < pe && col < a.di;
            const int64_t at = valid ? time_of(p) * step_i + col : 0;
            const int left = valid ? a.di - col : 0;
            if (!STATE) q_n[m] = load4(q + at, left);
            k_n[m] = load4(k + at, left);
        }
#pragma unroll
        for (int m = 0; m < kLoadV; ++m) {
            const int e = tid + m * kBlock, row = e / kRowV, col = e % kRowV * 4;
            const int64_t p = pc + row;
            const bool valid = p < pe && col < dj;
            v_n[m] = load4(v + (valid ? time_of(p) * step_j + col : 0), valid ? dj - col : 0);
        }
    };
    fetch(p0);

    for (int64_t pc = p0; pc < pe; pc += kChunk) {
        const int n = pe - pc < kChunk ? static_cast<int>(pe - pc) : kChunk;
        // behind the sequence's last position a forward pass leaves S, not g S
        const int m = n - (!STATE && !a.reverse && pc + n == len ? 1 : 0);
        __syncthreads();                       // everybody is done with the rows of the last chunk
#pragma unroll
        for (int x = 0; x < kLoadQ; ++x) {
            const int e = tid + x * kBlock, at = e / kRowQ * LD + e % kRowQ * 4;
            if (!STATE) *reinterpret_cast<f4*>(q_s + at) = q_n[x];
            *reinterpret_cast<f4*>(k_s + at) = k_n[x];
        }
#pragma unroll
        for (int x = 0; x < kLoadV; ++x) {
            const int e = tid + x * kBlock;
            *reinterpret_cast<f4*>(v_s + e / kRowV * LDV + e % kRowV * 4) = v_n[x];
        }
        __syncthreads();
        if (pc + kChunk < pe) fetch(pc + kChunk);

        // v[b][j] for b = 16 bt + 4 lq + r, j = own column: an operand of both products that use v
        float v_r[NJ][2][4];
#pragma unroll
        for (int jt = 0; jt < NJ; ++jt)
#pragma unroll
            for (int bt = 0; bt < 2; ++bt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    v_r[jt][bt][r] = v_s[(16 * bt + 4 * lq + r) * LDV + 16 * (4 * jt + wave) + l16];

        f4 o[NJ][2], dz[TAN ? NJ : 1][2];
        if constexpr (!STATE) {
            // scores k_b . q_a of the tiles (b, a) = (0, 0), (0, 1), (1, 1), one wavefront each
            if (wave < 3) {
                const int bt = wave >> 1, at = (wave + 1) >> 1;
                f4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int it = 0; it < NI; ++it) {
                    if (it >= ni) break;
                    const f4 kf = *reinterpret_cast<const f4*>(k_s + (16 * bt + l16) * LD + 16 * it + 4 * lq);
                    const f4 qf = *reinterpret_cast<const f4*>(q_s + (16 * at + l16) * LD + 16 * it + 4 * lq);
#pragma unroll
                    for (int r = 0; r < 4; ++r) s = mfma(kf[r], qf[r], s);
                }
                f4 w, dw;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int e = 16 * (at - bt) + l16 - 4 * lq - r;
                    const float x = a.kv_scale * s[r];
                    w[r] = e >= 0 ? pw[e] * x : 0.0f;
                    dw[r] = e >= 0 ? sl[e] * x : 0.0f;
                }
                score_s[wave * kWave + lane] = w;
                if (TAN) score_s[(3 + wave) * kWave + lane] = dw;
            }
            // q C
#pragma unroll
            for (int at = 0; at < 2; ++at) {
#pragma unroll
                for (int jt = 0; jt < NJ; ++jt) {
                    o[jt][at] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                    if (TAN) dz[jt][at] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                }
#pragma unroll
                for (int it = 0; it < NI; ++it) {
                    if (it >= ni) break;
                    const f4 qf = *reinterpret_cast<const f4*>(q_s + (16 * at + l16) * LD + 16 * it + 4 * lq);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int jt = 0; jt < NJ; ++jt) {
                            o[jt][at] = mfma(c[it][jt][r], qf[r], o[jt][at]);
                            if (TAN) dz[jt][at] = mfma(dc[it][jt][r], qf[r], dz[jt][at]);
                        }
                }
            }
#pragma unroll
            for (int at = 0; at < 2; ++at) {
                const float w = pw[16 * at + l16], dw = sl[16 * at + l16];
#pragma unroll
                for (int jt = 0; jt < NJ; ++jt) {
                    if (TAN) dz[jt][at] = w * dz[jt][at] + dw * o[jt][at];
                    o[jt][at] = w * o[jt][at];
                }
            }
        }
        // C = g^m C + sum_b g^(m-b) k_b^T v_b
        {
            float vw[NJ][2][4], vs[TAN ? NJ : 1][2][4];
#pragma unroll
            for (int bt = 0; bt < 2; ++bt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int e = m - (16 * bt + 4 * lq + r);       // below 0 only where v is 0
                    const float w = a.kv_scale * pw[e > 0 ? e : 0], dw = a.kv_scale * sl[e > 0 ? e : 0];
#pragma unroll
                    for (int jt = 0; jt < NJ; ++jt) {
                        vw[jt][bt][r] = w * v_r[jt][bt][r];
                        if (TAN) vs[jt][bt][r] = dw * v_r[jt][bt][r];
                    }
                }
            const float w = pw[m], dw = sl[m];
#pragma unroll
            for (int it = 0; it < NI; ++it) {
                if (it >= ni) break;
#pragma unroll
                for (int jt = 0; jt < NJ; ++jt) {
                    if (TAN) dc[it][jt] = w * dc[it][jt] + dw * c[it][jt];
                    c[it][jt] = w * c[it][jt];
                }
#pragma unroll
                for (int bt = 0; bt < 2; ++bt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float kf = k_s[(16 * bt + 4 * lq + r) * LD + 16 * it + l16];
#pragma unroll
                        for (int jt = 0; jt < NJ; ++jt) {
                            c[it][jt] = mfma(kf, vw[jt][bt][r], c[it][jt]);
                            if (TAN) dc[it][jt] = mfma(kf, vs[jt][bt][r], dc[it][jt]);
                        }
                    }
            }
        }
        if constexpr (!STATE) {
            __syncthreads();                   // the scores are there
            // A product with a score of 0 would carry a NaN or an infinity of v to positions before it: such values
            // are left out of the products and added to their own and later positions one by one.
            bool finite = true;
#pragma unroll
            for (int jt = 0; jt < NJ; ++jt)
#pragma unroll
                for (int bt = 0; bt < 2; ++bt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) finite = finite && __builtin_isfinite(v_r[jt][bt][r]);
            const bool all_finite = __all(finite);
            if (!all_finite)
#pragma unroll
                for (int jt = 0; jt < NJ; ++jt)
#pragma unroll
                    for (int bt = 0; bt < 2; ++bt)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (!__builtin_isfinite(v_r[jt][bt][r])) v_r[jt][bt][r] = 0.0f;
#pragma unroll
            for (int at = 0; at < 2; ++at)
#pragma unroll
                for (int bt = 0; bt <= at; ++bt) {
                    const f4 w = score_s[(bt + at) * kWave + lane];
                    f4 dw;
                    if (TAN) dw = score_s[(3 + bt + at) * kWave + lane];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int jt = 0; jt < NJ; ++jt) {
                            o[jt][at] = mfma(v_r[jt][bt][r], w[r], o[jt][at]);
                            if (TAN) dz[jt][at] = mfma(v_r[jt][bt][r], dw[r], dz[jt][at]);
                        }
                }
            if (!all_finite) {
                const float* score = reinterpret_cast<const float*>(score_s);
#pragma unroll
                for (int at = 0; at < 2; ++at)
                    for (int x = 0; x <= 16 * at + l16; ++x) {
                        const int e = (((x >> 4) + at) * kWave + (x >> 2 & 3) * 16 + l16) * 4 + (x & 3);
                        const float w = score[e], dw = TAN ? score[e + 12 * kWave] : 0.0f;
#pragma unroll
                        for (int jt = 0; jt < NJ; ++jt) {
                            const f4 vx = *reinterpret_cast<const f4*>(v_s + x * LDV + 16 * (4 * jt + wave) + 4 * lq);
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                if (__builtin_isfinite(vx[r])) continue;
                                o[jt][at][r] += w * vx[r];
                                if (TAN) dz[jt][at][r] += dw * vx[r];
                            }
                        }
                    }
            }
            // lane: position 16 at + l16, columns 16 (4 jt + wave) + 4 lq .. + 3
#pragma unroll
            for (int at = 0; at < 2; ++at) {
                if (16 * at + l16 >= n) continue;
                const int64_t row = time_of(pc + 16 * at + l16) * step_j + bh * a.dj + jt0;
#pragma unroll
                for (int jt = 0; jt < NJ; ++jt) {
                    const int j = 16 * (4 * jt + wave) + 4 * lq;
                    if (j >= dj) continue;
                    store4(a.out + row + j, a.out_scale * o[jt][at], dj - j);
                    if (TAN) {
                        const f4 z = load4(a.z + row + j, dj - j);
                        float s = 0.0f;
#pragma unroll
                        for (int r = 0; r < 4; ++r) s += z[r] * dz[jt][at][r];
                        slope += static_cast<double>(a.out_scale * s);
                    }
                }
            }
        }
    }

    if constexpr (STATE) {
#pragma unroll
        for (int it = 0; it < NI; ++it)
#pragma unroll
            for (int jt = 0; jt < NJ; ++jt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * it + 4 * lq + r, j = 16 * (4 * jt + wave) + l16;
                    if (i >= a.di || j >= dj) continue;
                    float* s = a.seg + (bh * a.segs + seg) * per_state * (TAN ? 2 : 1) + static_cast<int64_t>(i) * a.dj +
                               jt0 + j;
                    s[0] = c[it][jt][r];
                    if (TAN) s[per_state] = dc[it][jt][r];
                }
        return;
    }
    // rows behind the sequence's end
    {
        const int64_t first = len > p0 ? len : p0;
        const int width = dj < 64 * NJ ? dj : 64 * NJ;
        for (int64_t p = first + wave; p < p1; p += 4)
            for (int j = lane; j < width; j += kWave) a.out[p * step_j + bh * a.dj + jt0 + j] = 0.0f;
    }
    // the workgroup of the segment with the last position has the final state
    const bool last = len > 0 ? (pe == len && pe > p0) : seg == 0;
    if (last && (a.fin || (TAN && a.dfin))) {
#pragma unroll
        for (int it = 0; it < NI; ++it)
#pragma unroll
            for (int jt = 0; jt < NJ; ++jt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * it + 4 * lq + r, j = 16 * (4 * jt + wave) + l16;
                    if (i >= a.di || j >= dj) continue;
                    const int64_t at = bh * per_state + static_cast<int64_t>(i) * a.si + static_cast<int64_t>(jt0 + j) * a.sj;
                    if (a.fin) a.fin[at] = c[it][jt][r];
                    if (TAN && a.dfin) slope += static_cast<double>(a.dfin[at]) * dc[it][jt][r];
                }
    }
    if constexpr (TAN) {
        for (int d = 1; d < kWave; d <<= 1) slope += __shfl_xor(slope, d);
        if (lane == 0) part_s[wave] = slope;
        __syncthreads();
        if (tid == 0) a.slope[blockIdx.x] = (part_s[0] + part_s[1]) + (part_s[2] + part_s[3]);
    }
}

// Turns the states that the segments leave when they start from zero into the states they start from.
__global__ __launch_bounds__(kBlock) void la_scan_kernel(PassArgs a, int tangent) {
    const int64_t per_state = static_cast<int64_t>(a.di) * a.dj;
    const int64_t e = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
    const int64_t bh = blockIdx.y + static_cast<int64_t>(blockIdx.z) * 65535;
    if (e >= per_state || bh >= a.batch * a.heads) return;
    const int64_t len = sequence_length(a.lengths, bh / a.heads, a.time);
    const double g = a.decay[bh % a.heads];
    const float full = static_cast<float>(power(g, a.seg_len));
    const float dfull = static_cast<float>(a.seg_len * power(g, a.seg_len - 1));
    float c = 0.0f, dc = 0.0f;
    if (a.init) {
        const float s = a.init[bh * per_state + e / a.dj * a.si + e % a.dj * a.sj];
        c = len > 0 && !a.reverse ? static_cast<float>(g) * s : s;
        dc = len > 0 ? s : 0.0f;
    }
    float* slot = a.seg + bh * a.segs * per_state * (1 + tangent) + e;
    for (int seg = 0; seg < a.segs; ++seg, slot += per_state * (1 + tangent)) {
        const bool more = seg + 1 < a.segs;
        const float u = more ? slot[0] : 0.0f;
        const float du = more && tangent ? slot[per_state] : 0.0f;
        slot[0] = c;
        if (tangent) slot[per_state] = dc;
        const int64_t left = len - static_cast<int64_t>(seg) * a.seg_len;
        float w = full, dw = dfull;
        if (left < a.seg_len) {
            w = static_cast<float>(power(g, left > 0 ? left : 0));
            dw = left > 0 ? static_cast<float>(left * power(g, left - 1)) : 0.0f;
        }
        dc = w * dc + dw * c + du;
        c = w * c + u;
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

template <int NI, bool TAN, bool STATE>
void launch_pass(const PassArgs& a, int nj, unsigned grid) {
    if (nj == 1)
        hipLaunchKernelGGL((la_pass_kernel<NI, 1, TAN, STATE>), dim3(grid), dim3(kBlock), 0, ctx().stream, a);
    else
        hipLaunchKernelGGL((la_pass_kernel<NI, 2, TAN, STATE>), dim3(grid), dim3(kBlock), 0, ctx().stream, a);
}
template <bool TAN, bool STATE>
void launch_pass(const PassArgs& a, int nj, unsigned grid) {
    if (a.di <= 32) launch_pass<2, TAN, STATE>(a, nj, grid);
    else if (a.di <= 64) launch_pass<4, TAN, STATE>(a, nj, grid);
    else launch_pass<8, TAN, STATE>(a, nj, grid);
}

// One pass. ddecay: with the derivative by the decay.
int run_pass(PassArgs a, float* ddecay) {
    const int64_t sequences = a.batch * a.heads;
    const int64_t want = 2 * static_cast<int64_t>(ctx().num_cus);
    const int nj = a.dj > 64 ? 2 : 1;
    a.tiles_j = static_cast<int>(ceil_div(a.dj, 64 * nj));
    // enough workgroups for the device: the time axis is cut, into segments of 128 positions at least
    int64_t segs = ceil_div(want, sequences * a.tiles_j);
    const int64_t most = ceil_div(a.time, 4 * kChunk);
    if (segs > most) segs = most;
    if (segs < 1) segs = 1;
    int64_t seg_len = ceil_div(ceil_div(a.time, segs), kChunk) * kChunk;
    if (seg_len < kChunk) seg_len = kChunk;
    segs = a.time > 0 ? ceil_div(a.time, seg_len) : 1;
    if (seg_len > 0x7fffffff || sequences * segs * a.tiles_j > 0x7fffffff)
        return set_error(BSHIP_ERR_BAD_DIMENSION, "linear attention: %lld sequences of %lld steps exceed one launch",
                         static_cast<long long>(sequences), static_cast<long long>(a.time));
    a.segs = static_cast<int>(segs);
    a.seg_len = static_cast<int>(seg_len);
    const unsigned grid = static_cast<unsigned>(sequences * segs * a.tiles_j);
    const size_t per_state = static_cast<size_t>(a.di) * a.dj;
    Scratch seg, slope;
    if (segs > 1) {
        int st = seg.get(sequences * segs * per_state * (ddecay ? 2 : 1) * sizeof(float));
        if (st != 0) return st;
        a.seg = static_cast<float*>(seg.p);
    }
    if (ddecay) {
        int st = slope.get(grid * sizeof(double));
        if (st != 0) return st;
        a.slope = static_cast<double*>(slope.p);
    }
    if (segs > 1) {
        if (ddecay) launch_pass<true, true>(a, nj, grid);
        else launch_pass<false, true>(a, nj, grid);
        int st = check_launch("linear attention, segment states");
        if (st != 0) return st;
        const unsigned y = static_cast<unsigned>(sequences < 65535 ? sequences : 65535);
        hipLaunchKernelGGL(la_scan_kernel, dim3(static_cast<unsigned>(ceil_div(per_state, kBlock)), y,
                                                static_cast<unsigned>(ceil_div(sequences, 65535))),
                           dim3(kBlock), 0, ctx().stream, a, ddecay ? 1 : 0);
        st = check_launch("linear attention, scan");
        if (st != 0) return st;
    }
    if (ddecay) launch_pass<true, false>(a, nj, grid);
    else launch_pass<false, false>(a, nj, grid);
    int st = check_launch("linear attention");
    if (st != 0 || !ddecay) return st;
    hipLaunchKernelGGL(la_slope_kernel, dim3(static_cast<unsigned>(a.heads)), dim3(kBlock), 0, ctx().stream, a.slope,
                       ddecay, a.batch, a.heads, segs * a.tiles_j);
    return check_launch("linear attention, decay gradient");
}

int run_steps(PassArgs a) {
    const int64_t sequences = a.batch * a.heads;
    const bool wide = sequences * ceil_div(a.dj, 64) >= ctx().num_cus;
    a.tiles_j = static_cast<int>(ceil_div(a.dj, wide ? 64 : 16));
    if (sequences * a.tiles_j > 0x7fffffff)
        return set_error(BSHIP_ERR_BAD_DIMENSION, "linear attention: %lld sequences exceed one launch",
                         static_cast<long long>(sequences));
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
    return time <= kStepMost ? run_steps(a) : run_pass(a, nullptr);
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
    if ((st = run_pass(a, ddecay)) != 0) return st;
    // dk: v, do, q backwards, from the transposed gradient of the new state
    a.q = v; a.k = dout; a.v = q; a.out = dk_out;
    a.init = dnew_state;
    a.dfin = nullptr;
    a.kv_scale = scale; a.out_scale = 1.0f;
    a.reverse = 1;
    if ((st = run_pass(a, nullptr)) != 0) return st;
    // dv: k, q, do backwards; what is left behind the first step is the gradient of the state. This pass comes
    // last: dstate may be dnew_state.
    a.q = k; a.k = q; a.v = dout; a.out = dv_out;
    a.fin = dstate;
    a.di = static_cast<int>(dk); a.dj = static_cast<int>(dv);
    a.si = static_cast<int>(dv); a.sj = 1;
    return run_pass(a, nullptr);
}

}  // extern "C"
