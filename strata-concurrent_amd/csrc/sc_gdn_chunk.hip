// sc_gdn_chunk.hip - the gated delta rule over whole prompts (sc_gdn_chunk_async), 64 tokens at a time.
//
// With G the running sum of a chunk's log decays, M0 the state before it, and k, q of unit length (or as given):
//     (1 + A) U = X,   A_ij = beta_i e^(G_i - G_j) k_i . k_j  for j < i,   X = beta (V - e^G K M0)
//     O = scale (e^G Q M0 + P U),   P_ij = e^(G_i - G_j) q_i . k_j  for j <= i
//     M1 = e^(G_C) M0 + sum_j e^(G_C - G_j) k_j u_j^T
// Everything but M0 is known beforehand, so a first kernel forms T = (1 + A)^-1 and P of every chunk at once, and a second
// one takes the chunks of a sequence in order with products only.  Columns of the state (values) do not meet: a workgroup
// of the second kernel takes 16 or 32 of them with two waves.  One carries the state, whole columns in its registers: a
// result of a product (column = lane % 16, rows in registers) is the right operand of the next one as it stands, so nothing
// it needs crosses lanes but a column's largest value.  The other is a chunk behind and forms the outputs from the state and
// U that the first left in LDS; it also brings V and the factors of rows.  They meet once a chunk.
//
// Accuracy: the products run as f16 matrix instructions with sums in 32 bits, and keep f32 accuracy: an f32 operand is
// two f16 parts (22 bits) after a scaling by a power of two that puts its largest values near f16's upper end, where small
// ones keep their digits too.  f16 keys and queries enter as they are, exactly, and f32 ones scaled by row; unit length,
// decays and write strengths are factors of rows in f32.  The scalings: the state by column, X and U by column
// too, from bounds: with beta |k|^2 <= 2 (where the rule does not diverge) X stays below 2^5 and U below 2^8 of the largest of
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
constexpr float kUpT = 0x1p3f, kUpX = 0x1p3f, kUpU = kUpT * kUpX;   // where operands lie in f16's range: T, P; X; U

// Places of a v head's chunk in the workspace, in 16-byte words: T and P as matrix operands [wave][step][part][lane] (a
// wave's row tile w has steps 0 .. w / 2 of 32 tokens), then the factors of rows.
constexpr uint32_t kOperand = 6 * 2 * 64;
constexpr uint32_t operand_at(uint32_t wave, uint32_t step, uint32_t part) {
    return ((wave < 2 ? wave : wave == 2 ? 2 : 4) + step) * 128 + part * 64;
}
enum { kFState = 0, kFBeta = 64, kFWrite = 128, kFQuery = 192, kFRow = 256, kFDecay = 320, kFUp, kFBetaMost, kFactors = 324 };
constexpr uint32_t kChunkWords = 2 * kOperand + kFactors / 4;

// Places of a key head's chunk in the workspace, in 16-byte words: its keys as the left operand of the state's update
// [part][step of 32 keys][odd keys][step of 32 tokens][lane], then, where keys and queries are f32, their f16 parts as left
// operands [keys, queries][part][tile of tokens][step][lane] (f16 ones are read from where they are).
template <int S, int kParts>
constexpr uint32_t key_operand(uint32_t part, uint32_t i, uint32_t e, uint32_t step) {
    return (((part * (S / 32) + i) * 2 + e) * 2 + step) * 64;
}
template <int S, int kParts>
constexpr uint32_t row_operand(uint32_t which, uint32_t part, uint32_t tile, uint32_t i) {
    return kParts * S * 8 + (((which * kParts + part) * 4 + tile) * (S / 32) + i) * 64;
}
template <int S, int kParts>
constexpr uint32_t kRowWords = kParts * S * 8 * (kParts == 1 ? 1 : 3);

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
    ops_u32x4* rows = c.rows + (uint64_t(piece) * c.k_heads + kh) * kRowWords<S, kParts>;
    const bool write_rows = h == kh * a.share.d;   // one of the value heads that share the keys

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
                        st_global<ops_u32x4>(rows + row_operand<S, kParts>(which, part, t, i) + lane, x[part][i]);
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

    // the keys as the left operand of the state's update: key 32 i + 2 col + e, tokens 32 step + 4 g + j and 16 more, by way
    // of LDS, where the tiles will be
    if (write_rows) {
        constexpr uint32_t kRow = S * 2 + 16;
        static_assert(kC * kRow <= sizeof(s.tile) + sizeof(s.p));
        uint8_t* lds = reinterpret_cast<uint8_t*>(s.tile);
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < kSteps; ++i) *reinterpret_cast<ops_u32x4*>(lds + (t * 16 + col) * kRow + i * 64 + g * 16) = kf[t][part][i];
            wave_sync();
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int step = 0; step < 2; ++step) {
                    uint32_t w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        w[j] = *reinterpret_cast<const uint32_t*>(lds + (step * 32 + (j / 4) * 16 + g * 4 + j % 4) * kRow + (i * 32 + col * 2) * 2);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t sel = e ? 0x07060302u : 0x05040100u;
                        st_global<ops_u32x4>(rows + key_operand<S, kParts>(part, i, e, step) + lane,
                                             ops_u32x4{__builtin_amdgcn_perm(w[1], w[0], sel), __builtin_amdgcn_perm(w[3], w[2], sel),
                                                       __builtin_amdgcn_perm(w[5], w[4], sel), __builtin_amdgcn_perm(w[7], w[6], sel)});
                    }
                }
            wave_sync();
        }
    }

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

// Eight values, four each of two tiles, as a right operand in two parts.
__device__ __forceinline__ void split_pair(f32x4 a, f32x4 b, ops_u32x4& hi, ops_u32x4& lo) {
    uint32_t h[4], l[4];
    split2(a.x, a.y, h[0], l[0]);
    split2(a.z, a.w, h[1], l[1]);
    split2(b.x, b.y, h[2], l[2]);
    split2(b.z, b.w, h[3], l[3]);
    hi = ops_u32x4{h[0], h[1], h[2], h[3]};
    lo = ops_u32x4{l[0], l[1], l[2], l[3]};
}

template <int S, int kCols, bool kF16>
__global__ void __launch_bounds__(128, 1) gdn_chunk_kernel(GdnArgs a, ChunkArgs c) {
    constexpr int kParts = kF16 ? 1 : 2, kSteps = S / 32, kN = kCols / 16;
    constexpr uint32_t kBytes = kF16 ? 2 : 4;                            // of an activation
    constexpr uint32_t kRowV = kCols * kBytes, kPieces = kRowV / 16;     // a row of V or O of this workgroup, in 16-byte pieces
    constexpr uint32_t kEach = kC * kPieces / 64;                        // pieces of a lane
    constexpr uint32_t kFLanes = (kFactors + 63) / 64;
    // what one wave leaves for the other, by the chunk's parity
    struct Left {
        ops_u32x4 m[kN][kSteps][2][64], u[kN][2][2][64];   // the state before the chunk and U as right operands: [step][part]
        float m_up[kN][16], x_up[kN][16];                  // what they were scaled down by, by column
    };
    __shared__ Left s_left[2];
    __shared__ __align__(16) uint8_t s_vin[2][kC * kRowV], s_out[kC * kRowV];
    __shared__ __align__(16) float s_f[3][kFLanes * 64];
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const bool carries = __builtin_amdgcn_readfirstlane(tid >> 6) == 0;
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
        for (uint32_t t = from + tid / (kCols / 4); t < to; t += 128 / (kCols / 4))
            st_act4<kF16>(a.out + int64_t(t) * a.out_ld, h * S + block * kCols + tid % (kCols / 4) * 4, f32x4{});
        return;
    }

    // Loads are asked for where the registers that they fill have been used, a chunk ahead.  What a lane reads past the
    // sequence's end is its last row again (a minimum of byte offsets, which row strides leave below 2^31), past the last
    // chunk that chunk again: no branch decides what is in flight.
    auto last_row = [&](uint32_t chunk) {
        const uint32_t t0 = (chunk - q.chunk0) * kC;
        return q.t1 - q.t0 - t0 < kC ? q.t1 - q.t0 - t0 - 1 : kC - 1;
    };
    auto clamped = [&](uint32_t chunk) { return chunk < c1 ? chunk : c1 - 1; };
    auto operands_of = [&](uint32_t chunk) { return c.chunks + (uint64_t(chunk - c.first) * a.v_heads + h) * kChunkWords; };
    auto rows_of = [&](uint32_t chunk) { return c.rows + (uint64_t(chunk - c.first) * c.k_heads + kh) * kRowWords<S, kParts>; };
    // keys or queries as left operands
    auto load_rows = [&](ops_u32x4 (&x)[4][kParts][kSteps], uint32_t chunk, uint32_t which) {
        if constexpr (kF16) {
            const uint32_t ld = uint32_t(which ? a.q_ld : a.k_ld), last = last_row(chunk) * ld;
            const uint8_t* p = (which ? a.q : a.k) + int64_t(q.t0 + (chunk - q.chunk0) * kC) * ld + kh * S * 2;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint32_t at = min((t * 16 + col) * ld, last) + g * 16;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) x[t][0][i] = ld_global<ops_u32x4>(p + at + i * 64);
            }
        } else {
            const ops_u32x4* p = rows_of(chunk) + lane;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int part = 0; part < kParts; ++part)
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) x[t][part][i] = ld_global<ops_u32x4>(p + row_operand<S, kParts>(which, part, t, i));
        }
    };
    // T or P: operand w of operand_at's six, in two parts
    auto load_operand = [&](ops_u32x4 (&x)[6][2], uint32_t chunk, uint32_t which) {
        const ops_u32x4* p = operands_of(chunk) + which * kOperand + lane;
#pragma unroll
        for (int i = 0; i < 6; ++i)
#pragma unroll
            for (int part = 0; part < 2; ++part) x[i][part] = ld_global<ops_u32x4>(p + i * 128 + part * 64);
    };
    // the product with T or P of a right operand [step][part]
    auto triangle = [&](const ops_u32x4 (&x)[6][2], const ops_u32x4 (&y)[2][2], int tile) {
        const int first = tile < 2 ? tile : tile == 2 ? 2 : 4;
        f32x4 hi{}, lo{};
#pragma unroll
        for (int step = 0; step <= tile / 2; ++step) {
            hi = mfma(x[first + step][0], y[step][0], hi);
            lo = mfma(x[first + step][0], y[step][1], lo);
            lo = mfma(x[first + step][1], y[step][0], lo);
        }
        return hi + lo;
    };

    if (carries) {
        // the state: keys 32 i + 8 g + 2 j + e in m[.][i][e][j], a column a lane
        float* state = base + a.state_offset + h * a.head_ld + block * kCols + col + g * 8 * a.key_ld;
        f32x4 m[kN][kSteps][2];
#pragma unroll
        for (int b = 0; b < kN; ++b)
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < 4; ++j) m[b][i][e][j] = ld_global<float>(state + (i * 32 + 2 * j + e) * a.key_ld + b * 16);
        ops_u32x4 k[4][kParts][kSteps], t[6][2], kt[kParts][kSteps][2][2];
        auto load_keys = [&](uint32_t chunk) {
            const ops_u32x4* p = rows_of(chunk) + lane;
#pragma unroll
            for (int part = 0; part < kParts; ++part)
#pragma unroll
                for (int i = 0; i < kSteps; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int step = 0; step < 2; ++step) kt[part][i][e][step] = ld_global<ops_u32x4>(p + key_operand<S, kParts>(part, i, e, step));
        };
        load_rows(k, c0, 0);
        load_operand(t, c0, 0);
        load_keys(c0);
        for (uint32_t chunk = c0; chunk < c1; ++chunk) {
            const uint32_t which = (chunk - c0) & 1, last = last_row(chunk), ahead = clamped(chunk + 1);
            Left& left = s_left[which];
            __syncthreads();   // V and the factors are here, and the outputs of the chunk before the last are done
            const float* f = s_f[(chunk - c0) % 3];
            // the state as a right operand, scaled by column
            ops_u32x4 mh[kN][kSteps], ml[kN][kSteps];
            float m_up[kN];
#pragma unroll
            for (int b = 0; b < kN; ++b) {
                float top = 0;
#pragma unroll
                for (int i = 0; i < kSteps; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(m[b][i][e][j]));
                top = over_rows(top, max_of);
                float down;
                power_of(top, down, m_up[b]);
                if (top == 0) m_up[b] = 0.0f;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    // keys 8 g .. 8 g + 7 in order: the even ones and the odd ones take turns
                    const f32x4 even = m[b][i][0] * down, odd = m[b][i][1] * down;
                    split_pair(f32x4{even.x, odd.x, even.y, odd.y}, f32x4{even.z, odd.z, even.w, odd.w}, mh[b][i], ml[b][i]);
                    left.m[b][i][0][lane] = mh[b][i];
                    left.m[b][i][1][lane] = ml[b][i];
                }
                if (g == 0) left.m_up[b][col] = m_up[b];
            }
            // K M0
            f32x4 km[kN][4];
#pragma unroll
            for (int b = 0; b < kN; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) km[b][r] = f32x4{};
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int x = 0; x < kParts + 1; ++x)   // high by high, high by low, low by high
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int b = 0; b < kN; ++b) km[b][r] = mfma(k[r][x == 2][i], x == 1 ? ml[b][i] : mh[b][i], km[b][r]);
            load_rows(k, ahead, 0);
            // X, scaled by column
            ops_u32x4 xs[kN][2][2];
            float x_up[kN];
#pragma unroll
            for (int b = 0; b < kN; ++b) {
                f32x4 v[4];
                float top = 0;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const f32x4 beta = *reinterpret_cast<const f32x4*>(&f[kFBeta + r * 16 + g * 4]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t row = r * 16 + g * 4 + j;
                        const uint8_t* p = &s_vin[which][row * kRowV + (b * 16 + col) * kBytes];
                        float x;
                        if constexpr (kF16) x = float(*reinterpret_cast<const _Float16*>(p));
                        else x = *reinterpret_cast<const float*>(p);
                        v[r][j] = row <= last ? x * beta[j] : 0.0f;
                        top = fmaxf(top, fabsf(v[r][j]));
                    }
                }
                top = over_rows(top, max_of);
                float down;
                power_of(fmaxf(top, m_up[b] * f[kFBetaMost]), down, x_up[b]);
                if (g == 0) left.x_up[b][col] = x_up[b];
                down *= kUpX;
                const float by = m_up[b] * down;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const f32x4 fs = *reinterpret_cast<const f32x4*>(&f[kFState + r * 16 + g * 4]);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v[r][j] = int(r * 16 + g * 4 + j) <= int(last) ? v[r][j] * down - fs[j] * by * km[b][r][j] : 0.0f;
                }
                split_pair(v[0], v[1], xs[b][0][0], xs[b][0][1]);
                split_pair(v[2], v[3], xs[b][1][0], xs[b][1][1]);
            }
            // U = T X, and the same weighted for the state
            ops_u32x4 ws[kN][2][2];
#pragma unroll
            for (int b = 0; b < kN; ++b) {
                f32x4 u[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) u[r] = triangle(t, xs[b], r);
                ops_u32x4 us[2][2];
                split_pair(u[0], u[1], us[0][0], us[0][1]);
                split_pair(u[2], u[3], us[1][0], us[1][1]);
#pragma unroll
                for (int step = 0; step < 2; ++step)
#pragma unroll
                    for (int part = 0; part < 2; ++part) left.u[b][step][part][lane] = us[step][part];
#pragma unroll
                for (int r = 0; r < 4; ++r) u[r] *= *reinterpret_cast<const f32x4*>(&f[kFWrite + r * 16 + g * 4]);
                split_pair(u[0], u[1], ws[b][0][0], ws[b][0][1]);
                split_pair(u[2], u[3], ws[b][1][0], ws[b][1][1]);
            }
            load_operand(t, ahead, 0);
            // the state after the chunk
            const float decay = f[kFDecay], up = f[kFUp] * (1.0f / kUpU);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                f32x4 add[kN][2];
#pragma unroll
                for (int b = 0; b < kN; ++b) add[b][0] = f32x4{}, add[b][1] = f32x4{};
#pragma unroll
                for (int step = 0; step < 2; ++step)
#pragma unroll
                    for (int x = 0; x < kParts + 1; ++x)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int b = 0; b < kN; ++b)
                                add[b][e] = mfma(kt[x == 2][i][e][step], ws[b][step][x == 1], add[b][e]);
#pragma unroll
                for (int b = 0; b < kN; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) m[b][i][e] = decay * m[b][i][e] + (x_up[b] * up) * add[b][e];
            }
            load_keys(ahead);
        }
        __syncthreads();   // the last chunk's outputs
#pragma unroll
        for (int b = 0; b < kN; ++b)
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < 4; ++j) st_global<float>(state + (i * 32 + 2 * j + e) * a.key_ld + b * 16, m[b][i][e][j]);
        return;
    }

    // the other wave: V and the factors of the chunk after the next, outputs of the chunk before
    const uint32_t v_ld = uint32_t(a.v_ld);
    ops_u32x4 v_in[kEach];
    float f_in[kFLanes];
    auto load_early = [&](uint32_t chunk) {
        const uint32_t last = last_row(chunk) * v_ld;
        const uint8_t* p = a.v + int64_t(q.t0 + (chunk - q.chunk0) * kC) * a.v_ld + (h * S + block * kCols) * kBytes;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t at = lane + i * 64;
            v_in[i] = ld_global<ops_u32x4>(p + min(at / kPieces * v_ld, last) + at % kPieces * 16);
        }
        const float* f = reinterpret_cast<const float*>(operands_of(chunk) + 2 * kOperand);
#pragma unroll
        for (uint32_t i = 0; i < kFLanes; ++i) f_in[i] = ld_global<float>(f + min(lane + i * 64, uint32_t(kFactors - 1)));
    };
    auto put_early = [&](uint32_t n) {
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) *reinterpret_cast<ops_u32x4*>(&s_vin[n & 1][(lane + i * 64) * 16]) = v_in[i];
#pragma unroll
        for (uint32_t i = 0; i < kFLanes; ++i) s_f[n % 3][lane + i * 64] = f_in[i];
    };
    ops_u32x4 qs[4][kParts][kSteps], p[6][2];
    load_early(c0);
    put_early(0);
    load_early(clamped(c0 + 1));
    load_rows(qs, c0, 1);
    load_operand(p, c0, 1);
    for (uint32_t chunk = c0; chunk <= c1; ++chunk) {
        const uint32_t n = chunk - c0;
        __syncthreads();
        // the first wave reads the places of chunk n now, and this one the factors of chunk n - 1
        if (chunk < c1) {
            put_early(n + 1);
            load_early(clamped(chunk + 2));
        }
        if (chunk == c0) continue;
        const uint32_t done = chunk - 1, last = last_row(done);
        const Left& left = s_left[(n - 1) & 1];
        const float* f = s_f[(n - 1) % 3];
#pragma unroll
        for (int b = 0; b < kN; ++b) {
            f32x4 qm[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) qm[r] = f32x4{};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const ops_u32x4 hi = left.m[b][i][0][lane], lo = left.m[b][i][1][lane];
#pragma unroll
                for (int x = 0; x < kParts + 1; ++x)
#pragma unroll
                    for (int r = 0; r < 4; ++r) qm[r] = mfma(qs[r][x == 2][i], x == 1 ? lo : hi, qm[r]);
            }
            ops_u32x4 us[2][2];
#pragma unroll
            for (int step = 0; step < 2; ++step)
#pragma unroll
                for (int part = 0; part < 2; ++part) us[step][part] = left.u[b][step][part][lane];
            const float m_up = left.m_up[b][col], by = left.x_up[b][col] * (1.0f / (kUpU * kUpT));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const f32x4 pu = triangle(p, us, r);
                const f32x4 fq = *reinterpret_cast<const f32x4*>(&f[kFQuery + r * 16 + g * 4]), fr = *reinterpret_cast<const f32x4*>(&f[kFRow + r * 16 + g * 4]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float o = fq[j] * m_up * qm[r][j] + fr[j] * by * pu[j];
                    uint8_t* to = &s_out[(r * 16 + g * 4 + j) * kRowV + (b * 16 + col) * kBytes];
                    if constexpr (kF16) *reinterpret_cast<_Float16*>(to) = _Float16(o);
                    else *reinterpret_cast<float*>(to) = o;
                }
            }
        }
        load_rows(qs, clamped(chunk), 1);
        load_operand(p, clamped(chunk), 1);
        wave_sync();
        uint8_t* to = a.out + int64_t(q.t0 + (done - q.chunk0) * kC) * a.out_ld + (h * S + block * kCols) * kBytes;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t at = lane + i * 64;
            if (at / kPieces <= last)
                st_global<ops_u32x4>(to + int64_t(at / kPieces) * a.out_ld + at % kPieces * 16, *reinterpret_cast<const ops_u32x4*>(&s_out[at * 16]));
        }
        wave_sync();
    }
}

template <int S, int kCols, bool kF16>
void launch_chunks(const GdnArgs& a, const ChunkArgs& c, hipStream_t stream) {
    const uint32_t pairs = (a.n_seqs * a.v_heads + 7) / 8 * 8;
    hipLaunchKernelGGL((gdn_prepare_kernel<S, kF16>), dim3((c.count * a.v_heads + kWaves - 1) / kWaves), dim3(kThreadsC), 0, stream, a, c);
    hipLaunchKernelGGL((gdn_chunk_kernel<S, kCols, kF16>), dim3(pairs * (S / kCols)), dim3(128), 0, stream, a, c);
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
    const uint64_t chunks = uint64_t(c.count) * a.v_heads * kChunkWords, rows = uint64_t(c.count) * c.k_heads * size * (f16 ? 8 : 48);
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
