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
constexpr double kLog2e = 1.4426950408889634074;
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
// 2^x by the hardware's instruction, 1 unit in the last place
__device__ __forceinline__ float exp2_of(double x) { return __builtin_amdgcn_exp2f(float(x)); }
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

// The largest over the wave of values that are not negative, by row shifts and broadcasts.
__device__ __forceinline__ float wave_most(float v) {
    uint32_t x = __float_as_uint(v);
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x111, 0xF, 0xF, false)));   // row_shr 1, 2, 4, 8
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x112, 0xF, 0xF, false)));
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x114, 0xF, 0xF, false)));
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x118, 0xF, 0xF, false)));
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x142, 0xA, 0xF, false)));   // lane 15 of a row to the next one
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x143, 0xC, 0xF, false)));   // lane 31 to the upper half
    return __uint_as_float(last_lane(x));
}
template <int kCtrl, int kRows>
__device__ __forceinline__ double dpp_add(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(b)), kCtrl, kRows, 0xF, false));
    const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(b >> 32)), kCtrl, kRows, 0xF, false));
    return x + __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
// Inclusive sums over the lanes.
__device__ __forceinline__ double scan_add64(double x) {
    x = dpp_add<0x111, 0xF>(x);
    x = dpp_add<0x112, 0xF>(x);
    x = dpp_add<0x114, 0xF>(x);
    x = dpp_add<0x118, 0xF>(x);
    x = dpp_add<0x142, 0xA>(x);
    return dpp_add<0x143, 0xC>(x);
}

// What one wave writes to LDS the same wave reads in other lanes: its LDS operations stay in this order.
__device__ __forceinline__ void wave_sync() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

constexpr int kTileRow = 20, kTileFloats = 16 * kTileRow + 4;   // a 16 x 16 tile in LDS: 16-byte rows, tiles on banks of their own
constexpr int tile_of(int r, int c) { return r * (r + 1) / 2 + c; }

// A wave takes one chunk of one value head, alone: the products K K^T and Q K^T by tiles of 16 tokens up to the diagonal,
// A and P from them, and T = (1 + A)^-1: the four diagonal tiles by substitution, a column a lane, the rest by products
// of tiles, T_10 = - T_11 (A_10 T_00) for tiles of 16 and then of 32, with f32 matrix instructions.  A product's left tile
// comes from LDS as rows, its right one is a result in registers as it is: the four terms a lane adds are those whose rows
// it holds.
template <int S, bool kF16>
__global__ void __launch_bounds__(kThreadsC, 2) gdn_prepare_kernel(GdnArgs a, ChunkArgs c) {
    constexpr int kParts = kF16 ? 1 : 2, kSteps = S / 32;
    struct Mine {
        float tile[10 * kTileFloats];
        float p[4 * kTileFloats];
        double G[kC];
        float beta[kC], fk[kC], fq[kC], up[2][kC], row_down[kC], squares[kC];
    };
    __shared__ __align__(16) Mine s_all[kWaves];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 4, col = lane & 15;
    const uint32_t item = blockIdx.x * kWaves + wave;
    if (item >= c.count * a.v_heads) return;
    const uint32_t piece = item / a.v_heads, h = item - piece * a.v_heads, kh = ops_div(h, a.share), chunk = c.first + piece;
    Mine& s = s_all[wave];
    Seq q;
    if (!seq_of(a, lane, [&](uint32_t, uint32_t lo, uint32_t hi) { return chunk >= lo && chunk < hi; }, q)) return;
    const uint32_t t0 = q.t0 + (chunk - q.chunk0) * kC, n = q.t1 - t0 < kC ? q.t1 - t0 : kC;
    ops_u32x4* out = c.chunks + (uint64_t(piece) * a.v_heads + h) * kChunkWords;
    uint8_t* rows = reinterpret_cast<uint8_t*>(c.rows + (uint64_t(piece) * c.k_heads + kh) * (4 * kC * S / 8));
    const bool write_rows = !kF16 && h == kh * a.share.d;

    const bool in = lane < n;
    const int64_t gates = int64_t(t0 + (in ? lane : 0)) * a.gate_ld + h;
    const float g_in = ld_global<float>(a.g + gates), beta_in = ld_global<float>(a.beta + gates);

    // tile t of keys or queries: token 16 t + col, values 32 step + 8 g .. + 7: as they lie in memory, then as operands, rows
    // past the chunk zero
    auto load_raw = [&](const uint8_t* from, int64_t ld, int t, ops_u32x4 (&x)[kParts * kSteps]) {
        const uint32_t mine = t * 16 + col, row = mine < n ? mine : n - 1;
        const uint8_t* p = from + int64_t(t0 + row) * ld + (kh * S + g * 8) * (kF16 ? 2 : 4);
#pragma unroll
        for (int i = 0; i < kParts * kSteps; ++i) x[i] = ld_global<ops_u32x4>(p + (kF16 ? i * 64 : i / 2 * 128 + i % 2 * 16));
    };
    auto to_tile = [&](const ops_u32x4 (&raw)[kParts * kSteps], int t, ops_u32x4 (&x)[kParts][kSteps], float* up, uint32_t which) {
        const uint32_t mine = t * 16 + col;
        if constexpr (kF16) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) x[0][i] = raw[i];
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
                if (mine >= n) x[0][i] = ops_u32x4{};
        } else {
            // scaled by a power of two to a largest value of 1 .. 2, in two parts, which the second kernel reads
            f32x4 y[kSteps][2];
            float top = 0;
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    y[i][j] = mine < n ? __builtin_bit_cast(f32x4, raw[(i * 2 + j) % (kParts * kSteps)]) : f32x4{};
#pragma unroll
                    for (int k = 0; k < 4; ++k) top = fmaxf(top, fabsf(y[i][j][k]));
                }
            top = over_rows(top, max_of);
            float down, back;
            power_of(top, down, back);
            if (g == 0) up[mine] = back;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) split2(y[i][j / 2][j % 2 * 2] * down, y[i][j / 2][j % 2 * 2 + 1] * down, hi[j], lo[j]);
                x[0][i] = ops_u32x4{hi[0], hi[1], hi[2], hi[3]};
                x[kParts - 1][i] = ops_u32x4{lo[0], lo[1], lo[2], lo[3]};
                if (write_rows)
#pragma unroll
                    for (int part = 0; part < kParts; ++part)
                        st_global<ops_u32x4>(rows + (((which * kParts + part) * kC + mine) * S + i * 32 + g * 8) * 2, x[part][i]);
            }
        }
    };
    auto dot = [&](const ops_u32x4 (&x)[kParts][kSteps], const ops_u32x4 (&y)[kParts][kSteps], f32x4 acc) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            acc = mfma(x[0][i], y[0][i], acc);
            if constexpr (!kF16) acc = mfma(x[0][i], y[kParts - 1][i], acc), acc = mfma(x[kParts - 1][i], y[0][i], acc);
        }
        return acc;
    };
    // f16 queries are all asked for now, f32 ones a tile ahead (registers)
    constexpr int kAhead = kF16 ? 4 : 1;
    ops_u32x4 k_raw[4][kParts * kSteps], q_raw[kAhead][kParts * kSteps], kf[4][kParts][kSteps];
#pragma unroll
    for (int t = 0; t < 4; ++t) load_raw(a.k, a.k_ld, t, k_raw[t]);
#pragma unroll
    for (int t = 0; t < kAhead; ++t) load_raw(a.q, a.q_ld, t, q_raw[t]);
#pragma unroll
    for (int t = 0; t < 4; ++t) to_tile(k_raw[t], t, kf[t], s.up[0], 0);

    // sums of the log decays, to base 2, lane = token
    const double G = scan_add64(in ? double(g_in < kLeastG ? kLeastG : g_in) * kLog2e : 0.0);
    const float beta = in ? beta_in : 0.0f;
    s.G[lane] = G;
    s.beta[lane] = beta;
    const uint64_t G_bits = __builtin_bit_cast(uint64_t, G);
    const double G_all = __builtin_bit_cast(double, uint64_t(last_lane(uint32_t(G_bits >> 32))) << 32 | last_lane(uint32_t(G_bits)));

    // K K^T, element (4 g + i, col) of a tile; its diagonal has the squares of the lengths
    f32x4 kk[10];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int cc = 0; cc <= r; ++cc) kk[tile_of(r, cc)] = dot(kf[r], kf[cc], f32x4{});
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (g * 4 + i == col) s.squares[t * 16 + col] = kk[tile_of(t, t)][i];
    wave_sync();
    // the factor that brings a row as multiplied to its length, unit or its own, and that length
    auto factor = [&](float squares, const float* up, float& length) {
        const float by = kF16 ? 1.0f : up[lane];
        const float f = !in ? 0.0f : a.l2norm ? __builtin_amdgcn_rsqf(squares + a.eps / by / by) : by;
        length = in ? __builtin_amdgcn_sqrtf(squares) * f : 0.0f;
        return f;
    };
    float k_length;
    const float fk = factor(s.squares[lane], s.up[0], k_length), k_most = wave_most(k_length);
    s.fk[lane] = fk;
    const float e = exp2_of(G), write = exp2_of(G_all - G) * fk;
    float* f = reinterpret_cast<float*>(out + 2 * kOperand);
    {
        float down, up;
        power_of(wave_most(write), down, up);
        const float beta_most = wave_most(fabsf(beta));
        f[kFState + lane] = beta * fk * e;
        f[kFBeta + lane] = beta;
        f[kFWrite + lane] = write * down;
        if (lane == 0) f[kFDecay] = exp2_of(G_all), f[kFUp] = up, f[kFBetaMost] = beta_most;
    }
    wave_sync();

#pragma unroll
    for (int r = 0; r < 4; ++r) {
        ops_u32x4 qf[kParts][kSteps];
        to_tile(q_raw[r % kAhead], r, qf, s.up[1], 1);
        if (!kF16 && r < 3) load_raw(a.q, a.q_ld, r + 1, q_raw[0]);
        f32x4 qq = dot(qf, qf, f32x4{}), qk[4];
#pragma unroll
        for (int cc = 0; cc <= r; ++cc) qk[cc] = dot(qf, kf[cc], f32x4{});
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (g * 4 + i == col) s.squares[col] = qq[i];
        wave_sync();
        if (lane < 16) {
            // token 16 r + lane: this lane's own place in the chunk is another one
            const uint32_t t = r * 16 + lane;
            const float by = kF16 ? 1.0f : s.up[1][t], squares = s.squares[lane];
            const float fq = t >= n ? 0.0f : a.l2norm ? __builtin_amdgcn_rsqf(squares + a.eps / by / by) : by;
            float down, up;
            power_of(t >= n ? 0.0f : fabsf(a.scale) * __builtin_amdgcn_sqrtf(squares) * fq * k_most, down, up);
            s.fq[t] = fq * a.scale;
            s.row_down[t] = down * kUpT;
            f[kFQuery + t] = a.scale * fq * exp2_of(s.G[t]);
            f[kFRow + t] = up;
        }
        wave_sync();
        // A below the diagonal, and P
        double Gr[4];
        float br[4], qr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t t = r * 16 + g * 4 + i;
            Gr[i] = s.G[t];
            br[i] = s.beta[t] * s.fk[t];
            qr[i] = s.fq[t] * s.row_down[t];
        }
#pragma unroll
        for (int cc = 0; cc <= r; ++cc) {
            const double Gc = s.G[cc * 16 + col];
            const float fc = s.fk[cc * 16 + col];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t row = g * 4 + i;
                const float fade = cc < r || row >= col ? exp2_of(Gr[i] - Gc) * fc : 0.0f;
                s.tile[tile_of(r, cc) * kTileFloats + row * kTileRow + col] = cc < r || row > col ? br[i] * fade * kk[tile_of(r, cc)][i] : 0.0f;
                s.p[cc * kTileFloats + row * kTileRow + col] = qr[i] * fade * qk[cc][i];
            }
        }
        wave_sync();
        // P as the second kernel's operand: row 16 r + col, places 0 .. 3 tokens 32 step + 4 g, 4 .. 7 16 more
#pragma unroll
        for (int step = 0; step <= r / 2; ++step) {
            const f32x4 u = *reinterpret_cast<const f32x4*>(&s.p[step * 2 * kTileFloats + col * kTileRow + g * 4]);
            const f32x4 v = step * 2 + 1 <= r ? *reinterpret_cast<const f32x4*>(&s.p[(step * 2 + 1) * kTileFloats + col * kTileRow + g * 4]) : f32x4{};
            uint32_t hi[4], lo[4];
            split2(u.x, u.y, hi[0], lo[0]);
            split2(u.z, u.w, hi[1], lo[1]);
            split2(v.x, v.y, hi[2], lo[2]);
            split2(v.z, v.w, hi[3], lo[3]);
            st_global<ops_u32x4>(out + kOperand + operand_at(r, step, 0) + lane, ops_u32x4{hi[0], hi[1], hi[2], hi[3]});
            st_global<ops_u32x4>(out + kOperand + operand_at(r, step, 1) + lane, ops_u32x4{lo[0], lo[1], lo[2], lo[3]});
        }
        wave_sync();
    }

    // the diagonal tiles of T: column col of tile g
    auto tile_at = [&](int t) { return s.tile + t * kTileFloats; };
    {
        const float* d = s.tile + (g * (g + 1) / 2 + g) * kTileFloats;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            f32x4 sum{uint32_t(i) == col ? 1.0f : 0.0f, 0, 0, 0};   // four sums: a chain a quarter as long
#pragma unroll
            for (int k = 0; k < i; k += 4) {
                const f32x4 row = *reinterpret_cast<const f32x4*>(&d[i * kTileRow + k]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (k + j < i) sum[j] -= row[j] * x[k + j];
            }
            x[i] = (sum.x + sum.y) + (sum.z + sum.w);
        }
        wave_sync();
#pragma unroll
        for (int i = 0; i < 16; ++i) s.tile[(g * (g + 1) / 2 + g) * kTileFloats + i * kTileRow + col] = x[i];
        wave_sync();
    }
    auto left = [&](int t) { return *reinterpret_cast<const f32x4*>(tile_at(t) + col * kTileRow + g * 4); };
    auto right = [&](int t) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = tile_at(t)[(g * 4 + i) * kTileRow + col];
        return x;
    };
    auto product = [&](f32x4 x, f32x4 y, f32x4 acc) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = mfma_f32(x[i], y[i], acc);
        return acc;
    };
    auto put = [&](int t, f32x4 x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) tile_at(t)[(g * 4 + i) * kTileRow + col] = x[i];
    };
    {
        const f32x4 zero{}, t00 = right(tile_of(0, 0)), t11 = right(tile_of(1, 1)), t22 = right(tile_of(2, 2));
        const f32x4 y10 = product(left(tile_of(1, 0)), t00, zero), y32 = product(left(tile_of(3, 2)), t22, zero);
        const f32x4 t10 = -product(left(tile_of(1, 1)), y10, zero), t32 = -product(left(tile_of(3, 3)), y32, zero);
        wave_sync();
        put(tile_of(1, 0), t10);
        put(tile_of(3, 2), t32);
        const f32x4 y20 = product(left(tile_of(2, 1)), t10, product(left(tile_of(2, 0)), t00, zero)), y21 = product(left(tile_of(2, 1)), t11, zero);
        const f32x4 y30 = product(left(tile_of(3, 1)), t10, product(left(tile_of(3, 0)), t00, zero)), y31 = product(left(tile_of(3, 1)), t11, zero);
        wave_sync();
        const f32x4 l22 = left(tile_of(2, 2)), l32 = left(tile_of(3, 2)), l33 = left(tile_of(3, 3));
        put(tile_of(2, 0), -product(l22, y20, zero));
        put(tile_of(2, 1), -product(l22, y21, zero));
        put(tile_of(3, 0), -product(l33, y30, product(l32, y20, zero)));
        put(tile_of(3, 1), -product(l33, y31, product(l32, y21, zero)));
        wave_sync();
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int step = 0; step <= r / 2; ++step) {
            const f32x4 u = left(tile_of(r, step * 2)) * kUpT, v = step * 2 + 1 <= r ? left(tile_of(r, step * 2 + 1)) * kUpT : f32x4{};
            uint32_t hi[4], lo[4];
            split2(u.x, u.y, hi[0], lo[0]);
            split2(u.z, u.w, hi[1], lo[1]);
            split2(v.x, v.y, hi[2], lo[2]);
            split2(v.z, v.w, hi[3], lo[3]);
            st_global<ops_u32x4>(out + operand_at(r, step, 0) + lane, ops_u32x4{hi[0], hi[1], hi[2], hi[3]});
            st_global<ops_u32x4>(out + operand_at(r, step, 1) + lane, ops_u32x4{lo[0], lo[1], lo[2], lo[3]});
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
    f32x4 f_state, beta, write, f_query, f_row;
    f32x4 all;                                        // the chunk's decay, the scale of `write`, the largest beta
};

template <int S, int kCols, bool kF16>
__global__ void __launch_bounds__(kThreadsC, 1) gdn_chunk_kernel(GdnArgs a, ChunkArgs c) {
    constexpr int kParts = kF16 ? 1 : 2, kSteps = S / 32, kN = kCols / 16;
    using R = ChunkRows<S, kParts>;
    struct Values {
        f32x4 beta;
        uint32_t raw[kN][4];
        f32x4 by[kN];
    };
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
        r.f_state = ld_global<f32x4>(f + kFState + mine4);
        r.write = ld_global<f32x4>(f + kFWrite + mine4);
        r.f_query = ld_global<f32x4>(f + kFQuery + mine4);
        r.f_row = ld_global<f32x4>(f + kFRow + mine4);
        r.all = ld_global<f32x4>(f + kFDecay);
    };
    // the wave's rows of V, and their largest value a column times beta, for the scale of X
    auto load_v = [&](Values& v, uint32_t chunk) {
        const uint32_t t0 = q.t0 + (chunk - q.chunk0) * kC, n = q.t1 - t0 < kC ? q.t1 - t0 : kC;
        v.beta = ld_global<f32x4>(reinterpret_cast<const float*>(c.chunks + (uint64_t(chunk - c.first) * a.v_heads + h) * kChunkWords + 2 * kOperand) +
                                  kFBeta + wave * 16 + g * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t t = wave * 16 + g * 4 + i;
            const uint8_t* p = a.v + int64_t(t0 + (t < n ? t : n - 1)) * a.v_ld;
#pragma unroll
            for (int b = 0; b < kN; ++b) {
                const uint32_t at = h * S + block * kCols + b * 16 + col;
                if constexpr (kF16) v.raw[b][i] = ld_global<uint16_t>(p + at * 2);
                else v.raw[b][i] = ld_global<uint32_t>(p + at * 4);
            }
        }
    };
    auto put_v = [&](Values& v, uint32_t chunk) {
        const uint32_t t0 = q.t0 + (chunk - q.chunk0) * kC, n = q.t1 - t0 < kC ? q.t1 - t0 : kC;
#pragma unroll
        for (int b = 0; b < kN; ++b) {
            float top = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = kF16 ? float(__builtin_bit_cast(_Float16, uint16_t(v.raw[b][i]))) : __uint_as_float(v.raw[b][i]);
                v.by[b][i] = wave * 16 + g * 4 + i < n ? x * v.beta[i] : 0.0f;
                top = fmaxf(top, fabsf(v.by[b][i]));
            }
            top = over_rows(top, max_of);
            if (g == 0) s_v[(chunk - c0) & 1][b][wave][col] = top;
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

    // a chunk's rows are asked for a whole chunk before they are used
    R ra, rb;
    Values v;
    load_v(v, c0);
    load(ra, c0);
    put_state();
    put_v(v, c0);
    auto turn = [&](const uint32_t chunk, R& r, R& next) {
        const uint32_t t0 = q.t0 + (chunk - q.chunk0) * kC, n = q.t1 - t0 < kC ? q.t1 - t0 : kC;
        const bool more = chunk + 1 < c1;
        Values nv;
        if (more) {
            load_v(nv, chunk + 1);
            load(next, chunk + 1);
        }
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
            most *= r.all.z;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) most = fmaxf(most, s_v[(chunk - c0) & 1][b][w][col]);
            power_of(most, x_down[b], x_up[b]);
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = wave * 16 + g * 4 + i < n ? (v.by[b][i] - r.f_state[i] * km[i]) * (x_down[b] * kUpX) : 0.0f;
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
            if (kF16 && n < uint32_t(kC))   // the last, partial chunk: whatever lies in the rows past it stays out
#pragma unroll
                for (int step = 0; step < 2; ++step)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (step * 32 + (j / 4) * 16 + g * 4 + j % 4 >= n) r.kt[0][step][j] = 0;
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
                const float by = x_up[b] * r.all.y * (1.0f / kUpU);
#pragma unroll
                for (int e = 0; e < 2; ++e) m[b][e] = r.all.x * m[b][e] + by * add[e];
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
        if (more) {
            put_v(nv, chunk + 1);
            v = nv;
        }
    };
    for (uint32_t chunk = c0; chunk < c1; chunk += 2) {
        turn(chunk, ra, rb);
        if (chunk + 1 < c1) turn(chunk + 1, rb, ra);
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
    hipLaunchKernelGGL((gdn_prepare_kernel<S, kF16>), dim3((c.count * a.v_heads + kWaves - 1) / kWaves), dim3(kThreadsC), 0, stream, a, c);
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
