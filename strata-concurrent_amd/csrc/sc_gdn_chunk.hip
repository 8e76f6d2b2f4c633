// sc_gdn_chunk.hip - the gated delta rule over whole prompts (sc_gdn_chunk_async), 64 tokens at a time.
//
// With G the running sum of a chunk's log decays, M0 the state before it, and k, q of unit length (or as given):
//     (1 + A) U = X,   A_ij = beta_i e^(G_i - G_j) k_i . k_j  for j < i,   X = beta (V - e^G K M0)
//     O = scale (e^G Q M0 + P U),   P_ij = e^(G_i - G_j) q_i . k_j  for j <= i
//     M1 = e^(G_C) M0 + sum_j e^(G_C - G_j) k_j u_j^T
// Everything but M0 is known beforehand, so a first kernel forms T = (1 + A)^-1 and P of every chunk at once, and a second
// one takes the chunks of a sequence in order with products only.  Columns of the state (values) do not meet: a workgroup
// of the second kernel takes 16 or 32 of them.  Its four waves share the chunk's 64 tokens (16 rows each of K M0, X, U, O)
// and the state's keys (32 each, in registers); what the others need of a wave's result goes through LDS, three times a
// chunk.
//
// Accuracy: the products run as f16 matrix instructions with sums in 32 bits, and keep f32 accuracy: an f32 operand is
// two f16 parts (22 bits) after a scaling by a power of two that puts its largest values near f16's upper end, where small
// ones keep their digits too.  f16 keys and queries enter as they are, exactly, and f32 ones scaled by row; unit length,
// decays and write strengths are factors of rows in f32.  The scalings: the state by column and wave, X and U by column,
// from bounds: with beta |k|^2 <= 2 (where the rule does not diverge) X stays below 2^5 and U below 2^8 of the largest of
// beta |V| and beta |M0|.  Sums of log decays are in 64 bits: what counts is their differences.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sc_ops.hpp"

namespace sc {
namespace {

constexpr int kC = 64;                       // tokens of a chunk
constexpr int kWaves = 4, kThreadsC = kWaves * 64;
constexpr float kLeastG = -200.0f;           // a decay of e^-200 is 0 in f32
constexpr float kUpT = 0x1p10f, kUpX = 0x1p10f, kUpU = 0x1p6f;   // where operands lie in f16's range (T, P and X; U)

// Places of a v head's chunk in the workspace, in 16-byte words: T and P as matrix operands [wave][step][part][lane] (a
// wave's row tile w has steps 0 .. w / 2 of 32 tokens), then the factors of rows.
constexpr uint32_t kOperand = 6 * 2 * 64;
constexpr uint32_t operand_at(uint32_t wave, uint32_t step, uint32_t part) {
    return ((wave < 2 ? wave : wave == 2 ? 2 : 4) + step) * 128 + part * 64;
}
enum { kFState = 0, kFBeta = 64, kFWrite = 128, kFQuery = 192, kFRow = 256, kFDecay = 320, kFUp, kFBetaMost, kFactors = 384 };
constexpr uint32_t kChunkWords = 2 * kOperand + kFactors / 4;

__device__ __forceinline__ f32x4 mfma(ops_u32x4 a, ops_u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    return __builtin_bit_cast(uint32_t, f16x2{_Float16(a), _Float16(b)});
}
// Two values as two f16 parts: truncated, and what that left out.  The high part is taken by the instruction that packs
// two, so that what is subtracted is what is multiplied later (a conversion the compiler folds into the product before it
// may round another way).
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    const f16x2 h = __builtin_bit_cast(f16x2, hi);
    lo = pack_f16(a - float(h.x), b - float(h.y));
}
// 2^-e and 2^e for the exponent of x >= 0 (its largest power of two not above), within f32's normal range; 1 for 0.
__device__ __forceinline__ void power_of(float x, float& down, float& up) {
    int e = int(__float_as_uint(x) >> 23) - 127;
    e = x == 0 ? 0 : e > 126 ? 126 : e < -126 ? -126 : e;
    down = __uint_as_float(uint32_t(127 - e) << 23);
    up = __uint_as_float(uint32_t(127 + e) << 23);
}
template <class F>
__device__ __forceinline__ float over_rows(float x, F f) {   // over the four lanes that share lane % 16
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }

// A sequence's rows and chunks: rows [t0, t1), its first chunk of all.
struct Seq {
    uint32_t s, t0, t1, chunk0;
};
__device__ __forceinline__ uint32_t rows_from(const GdnArgs& a, uint32_t s) {
    const int64_t t = ld_global<int64_t>(a.cu + s);
    return t < 0 ? 0u : t > int64_t(a.tokens) ? a.tokens : uint32_t(t);
}
// The sequence that `find` (of a sequence and the range of its chunks) looks for; one load a lane and a scan for 64.
template <class Find>
__device__ __forceinline__ bool seq_of(const GdnArgs& a, uint32_t lane, Find find, Seq& q) {
    uint32_t chunks = 0;
    for (uint32_t base = 0; base < a.n_seqs; base += 64) {
        const bool in = base + lane < a.n_seqs;
        const uint32_t t0 = in ? rows_from(a, base + lane) : 0u, t1 = in ? rows_from(a, base + lane + 1) : 0u;
        const uint32_t n = t1 > t0 ? (t1 - t0 + kC - 1) / kC : 0u;
        const uint32_t sum = scan_add(n), lo = chunks + sum - n;
        const uint64_t here = __ballot(in && find(base + lane, lo, lo + n));
        if (here) {
            const int at = __builtin_ctzll(here);
            q.s = __builtin_amdgcn_readfirstlane(base + at);
            q.t0 = __builtin_amdgcn_readlane(t0, at);
            q.t1 = __builtin_amdgcn_readlane(t1, at);
            q.chunk0 = __builtin_amdgcn_readlane(lo, at);
            return true;
        }
        chunks += last_lane(sum);
    }
    return false;
}

// ---- every chunk's T and P ------------------------------------------------------------------------------------------------

// A workgroup takes one chunk of one key head, for each value head that shares it.  Wave w has the row tile of tokens
// 16 w .. 16 w + 15 of both products of K with K and Q with K.
template <int S, bool kF16>
__global__ void __launch_bounds__(kThreadsC) gdn_prepare_kernel(GdnArgs a, ChunkArgs c) {
    constexpr int kParts = kF16 ? 1 : 2, kSteps = S / 32;
    __shared__ ops_u32x4 s_k[kParts][4][kSteps][64];
    __shared__ __align__(16) float s_a[kC][kC + 4], s_t[kC][kC + 4];
    __shared__ double s_g[kC];
    __shared__ float s_beta[kC], s_fk[kC], s_fq[kC], s_kk[kC], s_qq[kC], s_up[2][kC];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 4, col = lane & 15;
    const uint32_t kh = blockIdx.x % c.k_heads, chunk = c.first + blockIdx.x / c.k_heads;
    Seq q;
    if (!seq_of(a, lane, [&](uint32_t, uint32_t lo, uint32_t hi) { return chunk >= lo && chunk < hi; }, q)) return;
    const uint32_t t0 = q.t0 + (chunk - q.chunk0) * kC, n = q.t1 - t0 < kC ? q.t1 - t0 : kC;
    const uint64_t slot = chunk - c.first;

    // this wave's rows: token 16 w + col, values 32 step + 8 g .. + 7
    const uint32_t mine = wave * 16 + col, row = mine < n ? mine : n - 1;
    ops_u32x4 kf[kParts][kSteps], qf[kParts][kSteps];
    if constexpr (kF16) {
        const uint8_t* kp = a.k + int64_t(t0 + row) * a.k_ld + (kh * S + g * 8) * 2;
        const uint8_t* qp = a.q + int64_t(t0 + row) * a.q_ld + (kh * S + g * 8) * 2;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) kf[0][i] = ld_global<ops_u32x4>(kp + i * 64), qf[0][i] = ld_global<ops_u32x4>(qp + i * 64);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
            if (mine >= n) kf[0][i] = ops_u32x4{}, qf[0][i] = ops_u32x4{};
        if (g == 0) s_up[0][mine] = 1.0f, s_up[1][mine] = 1.0f;
    } else {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const uint8_t* p = which ? a.q + int64_t(t0 + row) * a.q_ld : a.k + int64_t(t0 + row) * a.k_ld;
            f32x4 x[kSteps][2];
            float top = 0;
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) x[i][j] = ld_act4<false>(p, kh * S + i * 32 + g * 8 + j * 4);
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (mine >= n) x[i][j] = f32x4{};
#pragma unroll
                    for (int k = 0; k < 4; ++k) top = fmaxf(top, fabsf(x[i][j][k]));
                }
            top = over_rows(top, max_of);
            float down, up;
            power_of(top, down, up);
            if (g == 0) s_up[which][mine] = up;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                uint32_t h[4], l[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) split2(x[i][j / 2][j % 2 * 2] * down, x[i][j / 2][j % 2 * 2 + 1] * down, h[j], l[j]);
                (which ? qf : kf)[0][i] = ops_u32x4{h[0], h[1], h[2], h[3]};
                (which ? qf : kf)[kParts - 1][i] = ops_u32x4{l[0], l[1], l[2], l[3]};
            }
        }
        // the second kernel reads rows of f16 parts: [k, q][part][64][S]
        uint8_t* to = reinterpret_cast<uint8_t*>(c.rows + (slot * c.k_heads + kh) * (4 * kC * S / 8));
#pragma unroll
        for (int part = 0; part < kParts; ++part)
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                st_global<ops_u32x4>(to + ((part * kC + mine) * S + i * 32 + g * 8) * 2, kf[part][i]);
                st_global<ops_u32x4>(to + (((kParts + part) * kC + mine) * S + i * 32 + g * 8) * 2, qf[part][i]);
            }
    }
#pragma unroll
    for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int i = 0; i < kSteps; ++i) s_k[part][wave][i][lane] = kf[part][i];
    __syncthreads();

    // products of the row tile with the key tiles up to its own: element (4 g + i, col)
    f32x4 kk[4], qk[4], qq{};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        kk[j] = f32x4{}, qk[j] = f32x4{};
        if (uint32_t(j) > wave) continue;
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int x = 0; x < kParts; ++x)
#pragma unroll
                for (int y = 0; y < kParts; ++y) {
                    if (x + y > 1) continue;   // both low parts: below 2^-22
                    const ops_u32x4 b = s_k[y][j][i][lane];
                    kk[j] = mfma(kf[x][i], b, kk[j]);
                    qk[j] = mfma(qf[x][i], b, qk[j]);
                }
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int x = 0; x < kParts; ++x)
#pragma unroll
            for (int y = 0; y < kParts; ++y)
                if (x + y <= 1) qq = mfma(qf[x][i], qf[y][i], qq);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (uint32_t(j) == wave)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (g * 4 + i == col) s_kk[mine] = kk[j][i], s_qq[mine] = qq[i];
    __syncthreads();
    // factors that bring the rows as multiplied to their length: unit, or their own
    if (threadIdx.x < 2 * kC) {
        const uint32_t t = threadIdx.x % kC;
        const bool is_q = threadIdx.x >= kC;
        const float up = s_up[is_q][t], squares = is_q ? s_qq[t] : s_kk[t];
        const float f = t >= n ? 0.0f : a.l2norm ? 1.0f / sqrtf(squares + a.eps / up / up) : up;
        (is_q ? s_fq : s_fk)[t] = f;
        // lengths, for the bound of P's rows
        (is_q ? s_qq : s_kk)[t] = t >= n ? 0.0f : sqrtf(squares) * f;
    }

    for (uint32_t each = 0; each < a.share.d; ++each) {
        const uint32_t h = kh * a.share.d + each;
        __syncthreads();
        float k_most = s_kk[lane];
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) k_most = fmaxf(k_most, __shfl_xor(k_most, m));
        // sums of the log decays, lane = token
        const bool in = lane < n;
        const float* gates = a.g + int64_t(t0 + (in ? lane : 0)) * a.gate_ld + h;
        const float g1 = in ? ld_global<float>(gates) : 0.0f;
        const float beta = in ? ld_global<float>(a.beta + int64_t(t0 + (in ? lane : 0)) * a.gate_ld + h) : 0.0f;
        double G = double(g1 < kLeastG ? kLeastG : g1);
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const double o = __shfl_up(G, m);
            if (lane >= uint32_t(m)) G += o;
        }
        const double G_all = __shfl(G, 63);
        ops_u32x4* out = c.chunks + (slot * a.v_heads + h) * kChunkWords;
        if (wave == 0) {
            s_g[lane] = G;
            s_beta[lane] = beta;
            float* f = reinterpret_cast<float*>(out + 2 * kOperand);
            const float fk = s_fk[lane], e = expf(float(G)), write = expf(float(G_all - G)) * fk;
            float most = write, beta_most = fabsf(beta);
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                most = fmaxf(most, __shfl_xor(most, m));
                beta_most = fmaxf(beta_most, __shfl_xor(beta_most, m));
            }
            float down, up, row_down, row_up;
            power_of(most, down, up);
            power_of(fabsf(a.scale) * s_qq[lane] * k_most, row_down, row_up);
            s_up[0][lane] = row_down;
            f[kFState + lane] = beta * fk * e;
            f[kFBeta + lane] = beta;
            f[kFWrite + lane] = write * down;
            f[kFQuery + lane] = a.scale * s_fq[lane] * e;
            f[kFRow + lane] = row_up;
            if (lane == 0) f[kFDecay] = expf(float(G_all)), f[kFUp] = up, f[kFBetaMost] = beta_most;
        }
        __syncthreads();
        // A below the diagonal, and P
        f32x4 p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double Gj = s_g[j * 16 + col];
            const float fj = s_fk[j * 16 + col];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t r = wave * 16 + g * 4 + i, t = j * 16 + col;
                const float fade = r >= t ? expf(float(s_g[r] - Gj)) * fj : 0.0f;
                s_a[r][t] = r > t ? s_beta[r] * s_fk[r] * fade * kk[j][i] : 0.0f;
                p[j][i] = a.scale * s_fq[r] * fade * qk[j][i] * s_up[0][r] * kUpT;
            }
        }
        __syncthreads();
        // T: the diagonal tiles by substitution (lane = column of the inverse) ...
        {
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float sum = uint32_t(i) == col ? 1.0f : 0.0f;
#pragma unroll
                for (int k = 0; k < i; ++k) sum -= s_a[wave * 16 + i][wave * 16 + k] * x[k];
                x[i] = sum;
            }
            if (g == 0)
#pragma unroll
                for (int i = 0; i < 16; ++i) s_t[wave * 16 + i][wave * 16 + col] = x[i];
        }
        __syncthreads();
        // ... then T_21 = - T_22 (A_21 T_11) for tiles of 16 and of 32.  product(): 16 x 16 of rows r of X by columns c of Y
        auto product = [&](const float (&X)[kC][kC + 4], uint32_t r, uint32_t m, const float (&Y)[kC][kC + 4], uint32_t cc, f32x4 acc) {
#pragma unroll
            for (int k = 0; k < 4; ++k) acc = mfma_f32(X[r * 16 + col][m * 16 + k * 4 + g], Y[m * 16 + k * 4 + g][cc * 16 + col], acc);
            return acc;
        };
        auto store = [&](float (&X)[kC][kC + 4], uint32_t r, uint32_t cc, f32x4 v, float by) {
#pragma unroll
            for (int i = 0; i < 4; ++i) X[r * 16 + g * 4 + i][cc * 16 + col] = v[i] * by;
        };
        if (wave == 1 || wave == 3) store(s_a, wave, wave - 1, product(s_a, wave, wave - 1, s_t, wave - 1, f32x4{}), 1.0f);
        __syncthreads();
        if (wave == 1 || wave == 3) store(s_t, wave, wave - 1, product(s_t, wave, wave, s_a, wave - 1, f32x4{}), -1.0f);
        __syncthreads();
        const uint32_t tr = 2 + wave / 2, tc = wave % 2;
        f32x4 y = product(s_a, tr, 1, s_t, tc, f32x4{});   // T_01 is zero, as is A's part above
        if (tc == 0) y = product(s_a, tr, 0, s_t, 0, y);
        __syncthreads();
        store(s_a, tr, tc, y, 1.0f);
        __syncthreads();
        f32x4 z = product(s_t, tr, 2, s_a, tc, f32x4{});
        if (tr == 3) z = product(s_t, 3, 3, s_a, tc, z);
        store(s_t, tr, tc, z, -1.0f);
        __syncthreads();
        // both as the second kernel's operands: row 16 w + col, places 0 .. 3 tokens 32 step + 4 g, 4 .. 7 16 more
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            if (which) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s_t[wave * 16 + g * 4 + i][j * 16 + col] = p[j][i];
                __syncthreads();
            }
            for (uint32_t step = 0; step <= wave / 2; ++step) {
                // above the diagonal T's tiles were never written
                const bool upper = !which && step * 2 + 1 > wave;
                const f32x4 u = *reinterpret_cast<const f32x4*>(&s_t[wave * 16 + col][step * 32 + g * 4]) * (which ? 1.0f : kUpT);
                const f32x4 v = upper ? f32x4{} : *reinterpret_cast<const f32x4*>(&s_t[wave * 16 + col][step * 32 + 16 + g * 4]) * (which ? 1.0f : kUpT);
                uint32_t hi[4], lo[4];
                split2(u.x, u.y, hi[0], lo[0]);
                split2(u.z, u.w, hi[1], lo[1]);
                split2(v.x, v.y, hi[2], lo[2]);
                split2(v.z, v.w, hi[3], lo[3]);
                ops_u32x4* to = out + which * kOperand + lane;
                st_global<ops_u32x4>(to + operand_at(wave, step, 0), ops_u32x4{hi[0], hi[1], hi[2], hi[3]});
                st_global<ops_u32x4>(to + operand_at(wave, step, 1), ops_u32x4{lo[0], lo[1], lo[2], lo[3]});
            }
        }
    }
}

// ---- the chunks of a sequence in order ------------------------------------------------------------------------------------

// What a wave reads of a chunk before it can start on it.
template <int S, int kParts>
struct ChunkRows {
    static constexpr int kSteps = S / 32;
    ops_u32x4 k[kParts][kSteps], q[kParts][kSteps];   // its row tile
    uint32_t kt[kParts][2][8];                        // its 32 keys: pairs of keys of the eight tokens of a step
    ops_u32x4 t[2][2], p[2][2];                       // T and P: [step][part]
    float f_state[4], beta[4], write[4], f_query[4], f_row[4];
    float decay, up, beta_most;
};

template <int S, int kCols, bool kF16>
__global__ void __launch_bounds__(kThreadsC, 1) gdn_chunk_kernel(GdnArgs a, ChunkArgs c) {
    constexpr int kParts = kF16 ? 1 : 2, kSteps = S / 32, kN = kCols / 16;
    using R = ChunkRows<S, kParts>;
    __shared__ ops_u32x4 s_m[kN][kSteps][2][64];         // the state as an operand: [step][part][lane]
    __shared__ float s_scale[kN][kSteps][16];
    __shared__ ops_u32x2 s_x[kN][2][2][64][2], s_u[kN][2][2][64][2], s_w[kN][2][2][64][2];   // [step][part][lane][tile]
    __shared__ float s_v[2][kN][kWaves][16];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 4, col = lane & 15;
    // workgroups go to the eight XCDs in turn: the column blocks of a head are kept on one, whose L2 has its operands
    constexpr uint32_t kBlocks = S / kCols;
    const uint32_t within = blockIdx.x / 8, pair = within / kBlocks * 8 + blockIdx.x % 8, block = within % kBlocks;
    if (pair >= a.n_seqs * a.v_heads) return;
    const uint32_t seq = pair / a.v_heads, h = pair - seq * a.v_heads, kh = ops_div(h, a.share);
    Seq q;
    if (!seq_of(a, lane, [&](uint32_t s, uint32_t, uint32_t) { return s == seq; }, q)) return;
    // this launch's chunks of the sequence
    const uint32_t all = q.t1 > q.t0 ? (q.t1 - q.t0 + kC - 1) / kC : 0u;
    const uint32_t c0 = q.chunk0 > c.first ? q.chunk0 : c.first, c1 = q.chunk0 + all < c.first + c.count ? q.chunk0 + all : c.first + c.count;
    if (c0 >= c1) return;
    float* base = a.state[seq];
    if (!base) {
        const uint32_t from = q.t0 + (c0 - q.chunk0) * kC, to = q.t0 + (c1 - q.chunk0) * kC < q.t1 ? q.t0 + (c1 - q.chunk0) * kC : q.t1;
        for (uint32_t t = from + threadIdx.x / (kCols / 4); t < to; t += kThreadsC / (kCols / 4))
            st_act4<kF16>(a.out + int64_t(t) * a.out_ld, h * S + block * kCols + threadIdx.x % (kCols / 4) * 4, f32x4{});
        return;
    }
    // the state: keys 32 w + 8 g + 2 i + e in m[.][e][i], a column a lane; waves past the keys have none
    const bool keys = wave < uint32_t(kSteps);
    float* state = base + a.state_offset + h * a.head_ld + block * kCols + col + (wave * 32 + g * 8) * a.key_ld;
    f32x4 m[kN][2];
#pragma unroll
    for (int b = 0; b < kN; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) m[b][e][i] = keys ? ld_global<float>(state + (2 * i + e) * a.key_ld + b * 16) : 0.0f;

    auto put_state = [&] {
        if (!keys) return;
#pragma unroll
        for (int b = 0; b < kN; ++b) {
            float top = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(m[b][e][i]));
            top = over_rows(top, max_of);
            float down, up;
            power_of(top, down, up);
            if (g == 0) s_scale[b][wave][col] = top == 0 ? 0.0f : up;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) split2(m[b][0][i] * down, m[b][1][i] * down, hi[i], lo[i]);
            s_m[b][wave][0][lane] = ops_u32x4{hi[0], hi[1], hi[2], hi[3]};
            s_m[b][wave][1][lane] = ops_u32x4{lo[0], lo[1], lo[2], lo[3]};
        }
    };

    auto load = [&](R& r, uint32_t chunk) {
        const uint32_t t0 = q.t0 + (chunk - q.chunk0) * kC, n = q.t1 - t0 < kC ? q.t1 - t0 : kC;
        const uint64_t slot = chunk - c.first;
        const uint8_t* rows = reinterpret_cast<const uint8_t*>(c.rows + (slot * c.k_heads + kh) * (4 * kC * S / 8));
        const uint32_t mine = wave * 16 + col, at = mine < n ? mine : n - 1;
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            const uint8_t* kp = kF16 ? a.k + int64_t(t0 + at) * a.k_ld + kh * S * 2 : rows + (part * kC + mine) * S * 2;
            const uint8_t* qp = kF16 ? a.q + int64_t(t0 + at) * a.q_ld + kh * S * 2 : rows + ((kParts + part) * kC + mine) * S * 2;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                r.k[part][i] = ld_global<ops_u32x4>(kp + i * 64 + g * 16);
                r.q[part][i] = ld_global<ops_u32x4>(qp + i * 64 + g * 16);
            }
            if (keys)
#pragma unroll
                for (int step = 0; step < 2; ++step)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t t = step * 32 + (j / 4) * 16 + g * 4 + j % 4, u = t < n ? t : n - 1;
                        const uint8_t* p = kF16 ? a.k + int64_t(t0 + u) * a.k_ld + kh * S * 2 : rows + (part * kC + t) * S * 2;
                        r.kt[part][step][j] = ld_global<uint32_t>(p + (wave * 32 + col * 2) * 2);
                        if (kF16 && t >= n) r.kt[part][step][j] = 0;
                    }
        }
        const ops_u32x4* from = c.chunks + (slot * a.v_heads + h) * kChunkWords;
#pragma unroll
        for (int step = 0; step < 2; ++step)
            if (uint32_t(step) <= wave / 2)
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    r.t[step][part] = ld_global<ops_u32x4>(from + operand_at(wave, step, part) + lane);
                    r.p[step][part] = ld_global<ops_u32x4>(from + kOperand + operand_at(wave, step, part) + lane);
                }
        const float* f = reinterpret_cast<const float*>(from + 2 * kOperand);
        const uint32_t mine4 = wave * 16 + g * 4;
        const f32x4 fs = ld_global<f32x4>(f + kFState + mine4), fb = ld_global<f32x4>(f + kFBeta + mine4), fw = ld_global<f32x4>(f + kFWrite + mine4);
        const f32x4 fq = ld_global<f32x4>(f + kFQuery + mine4), fr = ld_global<f32x4>(f + kFRow + mine4);
        const f32x4 one = ld_global<f32x4>(f + kFDecay);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.f_state[i] = fs[i], r.beta[i] = fb[i], r.write[i] = fw[i], r.f_query[i] = fq[i], r.f_row[i] = fr[i];
        r.decay = one.x, r.up = one.y, r.beta_most = one.z;
    };
    // beta V of the wave's rows, and its largest value a column, for the scale of X
    auto load_v = [&](f32x4 (&v)[kN], uint32_t chunk, const float (&beta)[4]) {
        const uint32_t t0 = q.t0 + (chunk - q.chunk0) * kC, n = q.t1 - t0 < kC ? q.t1 - t0 : kC;
#pragma unroll
        for (int b = 0; b < kN; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t t = wave * 16 + g * 4 + i;
                const uint8_t* p = a.v + int64_t(t0 + (t < n ? t : n - 1)) * a.v_ld;
                const uint32_t at = h * S + block * kCols + b * 16 + col;
                float x;
                if constexpr (kF16) x = float(__builtin_bit_cast(_Float16, ld_global<uint16_t>(p + at * 2)));
                else x = ld_global<float>(p + at * 4);
                v[b][i] = t < n ? x * beta[i] : 0.0f;
            }
    };
    auto put_v = [&](const f32x4 (&v)[kN], uint32_t which) {
#pragma unroll
        for (int b = 0; b < kN; ++b) {
            float top = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(v[b][i]));
            top = over_rows(top, max_of);
            if (g == 0) s_v[which][b][wave][col] = top;
        }
    };
    // a tile of 16 tokens of X, U or the weighted U as an operand: the wave's half of a step
    auto put = [&](ops_u32x2 (&to)[2][2][64][2], f32x4 x) {
        uint32_t h0, l0, h1, l1;
        split2(x.x, x.y, h0, l0);
        split2(x.z, x.w, h1, l1);
        to[wave / 2][0][lane][wave % 2] = ops_u32x2{h0, h1};
        to[wave / 2][1][lane][wave % 2] = ops_u32x2{l0, l1};
    };
    auto get = [&](const ops_u32x2 (&from)[2][2][64][2], int step, int part) {
        return *reinterpret_cast<const ops_u32x4*>(&from[step][part][lane][0]);
    };

    R r;
    f32x4 v[kN];
    load(r, c0);
    load_v(v, c0, r.beta);
    put_state();
    put_v(v, 0);
    for (uint32_t chunk = c0; chunk < c1; ++chunk) {
        const uint32_t t0 = q.t0 + (chunk - q.chunk0) * kC, n = q.t1 - t0 < kC ? q.t1 - t0 : kC;
        __syncthreads();
        // K M0 and Q M0, a step's sum by its own scale
        f32x4 qm[kN];
        float x_down[kN], x_up[kN];
#pragma unroll
        for (int b = 0; b < kN; ++b) {
            f32x4 km{};
            qm[b] = f32x4{};
            float most = 0;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const ops_u32x4 hi = s_m[b][i][0][lane], lo = s_m[b][i][1][lane];
                const float scale = s_scale[b][i][col];
                f32x4 ks{}, qs{};
                ks = mfma(r.k[0][i], hi, ks);
                qs = mfma(r.q[0][i], hi, qs);
                ks = mfma(r.k[0][i], lo, ks);
                qs = mfma(r.q[0][i], lo, qs);
                if constexpr (!kF16) ks = mfma(r.k[kParts - 1][i], hi, ks), qs = mfma(r.q[kParts - 1][i], hi, qs);
                km += scale * ks;
                qm[b] += scale * qs;
                most = fmaxf(most, scale);
            }
            most *= r.beta_most;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) most = fmaxf(most, s_v[(chunk - c0) & 1][b][w][col]);
            power_of(most, x_down[b], x_up[b]);
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = wave * 16 + g * 4 + i < n ? (v[b][i] - r.f_state[i] * km[i]) * (x_down[b] * kUpX) : 0.0f;
            put(s_x[b], x);
        }
        __syncthreads();
        // U = T X, and the same weighted for the state
#pragma unroll
        for (int b = 0; b < kN; ++b) {
            f32x4 u{};
#pragma unroll
            for (int step = 0; step < 2; ++step)
                if (uint32_t(step) <= wave / 2) {
                    const ops_u32x4 hi = get(s_x[b], step, 0), lo = get(s_x[b], step, 1);
                    u = mfma(r.t[step][0], hi, u);
                    u = mfma(r.t[step][0], lo, u);
                    u = mfma(r.t[step][1], hi, u);
                }
            u *= kUpU / (kUpT * kUpX);
            put(s_u[b], u);
            f32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = u[i] * r.write[i];
            put(s_w[b], w);
        }
        __syncthreads();
        // the state after the chunk
        if (keys) {
#pragma unroll
            for (int b = 0; b < kN; ++b) {
                f32x4 add[2]{};
#pragma unroll
                for (int step = 0; step < 2; ++step) {
                    const ops_u32x4 hi = get(s_w[b], step, 0), lo = get(s_w[b], step, 1);
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int part = 0; part < kParts; ++part) {
                            const uint32_t sel = e ? 0x07060302u : 0x05040100u;
                            const uint32_t (&t)[8] = r.kt[part][step];
                            const ops_u32x4 key{__builtin_amdgcn_perm(t[1], t[0], sel), __builtin_amdgcn_perm(t[3], t[2], sel),
                                                __builtin_amdgcn_perm(t[5], t[4], sel), __builtin_amdgcn_perm(t[7], t[6], sel)};
                            add[e] = mfma(key, hi, add[e]);
                            if (part == 0) add[e] = mfma(key, lo, add[e]);
                        }
                }
                const float by = x_up[b] * r.up * (1.0f / kUpU);
#pragma unroll
                for (int e = 0; e < 2; ++e) m[b][e] = r.decay * m[b][e] + by * add[e];
            }
        }
        put_state();
        // outputs
#pragma unroll
        for (int b = 0; b < kN; ++b) {
            f32x4 pu{};
#pragma unroll
            for (int step = 0; step < 2; ++step)
                if (uint32_t(step) <= wave / 2) {
                    const ops_u32x4 hi = get(s_u[b], step, 0), lo = get(s_u[b], step, 1);
                    pu = mfma(r.p[step][0], hi, pu);
                    pu = mfma(r.p[step][0], lo, pu);
                    pu = mfma(r.p[step][1], hi, pu);
                }
            const float by = x_up[b] * (1.0f / (kUpU * kUpT));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t t = wave * 16 + g * 4 + i;
                if (t >= n) continue;
                const float o = r.f_query[i] * qm[b][i] + r.f_row[i] * by * pu[i];
                uint8_t* to = a.out + int64_t(t0 + t) * a.out_ld;
                const uint32_t at = h * S + block * kCols + b * 16 + col;
                if constexpr (kF16) st_global<uint16_t>(to + at * 2, __builtin_bit_cast(uint16_t, _Float16(o)));
                else st_global<float>(to + at * 4, o);
            }
        }
        if (chunk + 1 < c1) {
            load(r, chunk + 1);
            load_v(v, chunk + 1, r.beta);
            put_v(v, (chunk + 1 - c0) & 1);
        }
    }
    if (keys)
#pragma unroll
        for (int b = 0; b < kN; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i) st_global<float>(state + (2 * i + e) * a.key_ld + b * 16, m[b][e][i]);
}

template <int S, int kCols, bool kF16>
void launch_chunks(const GdnArgs& a, const ChunkArgs& c, hipStream_t stream) {
    const uint32_t pairs = (a.n_seqs * a.v_heads + 7) / 8 * 8;
    hipLaunchKernelGGL((gdn_prepare_kernel<S, kF16>), dim3(c.count * c.k_heads), dim3(kThreadsC), 0, stream, a, c);
    hipLaunchKernelGGL((gdn_chunk_kernel<S, kCols, kF16>), dim3(pairs * (S / kCols)), dim3(kThreadsC), 0, stream, a, c);
}
template <int S>
hipError_t launch_of(const GdnArgs& a, const ChunkArgs& plan, bool f16, hipStream_t stream) {
    for (ChunkArgs c = plan; c.first < plan.total; c.first += plan.count) {
        c.count = plan.total - c.first < plan.count ? plan.total - c.first : plan.count;
        if (f16) launch_chunks<S, 16, true>(a, c, stream);
        else launch_chunks<S, 16, false>(a, c, stream);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// Chunks of one pair of launches: a long prompt goes through the workspace in pieces.
constexpr uint32_t kMostChunks = 256;

}  // namespace

uint64_t plan_gdn_chunks(const GdnArgs& a, int size, bool f16, ChunkArgs& c) {
    // a sequence has at most one chunk that is not full
    c.total = a.tokens / kC + (a.n_seqs < a.tokens ? a.n_seqs : a.tokens);
    c.count = c.total < kMostChunks ? c.total : kMostChunks;
    c.first = 0;
    c.k_heads = a.v_heads / a.share.d;
    const uint64_t chunks = uint64_t(c.count) * a.v_heads * kChunkWords, rows = f16 ? 0 : uint64_t(c.count) * c.k_heads * (4 * kC * size / 8);
    c.rows_at = chunks;
    const uint64_t bytes = (chunks + rows) * 16;
    return bytes ? bytes : 256;
}

hipError_t launch_gdn_chunk(const GdnArgs& a, int size, bool f16, void* workspace, hipStream_t stream) {
    ChunkArgs c;
    plan_gdn_chunks(a, size, f16, c);
    c.chunks = static_cast<ops_u32x4*>(workspace);
    c.rows = c.chunks + c.rows_at;
    if (size == 32) return launch_of<32>(a, c, f16, stream);
    if (size == 64) return launch_of<64>(a, c, f16, stream);
    if (size == 128) return launch_of<128>(a, c, f16, stream);
    return hipErrorInvalidValue;
}

}  // namespace sc
