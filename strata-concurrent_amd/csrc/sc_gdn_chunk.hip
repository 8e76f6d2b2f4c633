// sc_gdn_chunk.hip - the gated delta rule over whole prompts (sc_gdn_chunk_async), 64 tokens at a time.
//
// With G the running sum of a chunk's log decays, M0 the state before it, and k, q of unit length (or as given):
//     (1 + A) U = X,   A_ij = beta_i e^(G_i - G_j) k_i . k_j  for j < i,   X = beta (V - e^G K M0)
//     O = scale (e^G Q M0 + P U),   P_ij = e^(G_i - G_j) q_i . k_j  for j <= i
//     M1 = e^(G_C) M0 + sum_j e^(G_C - G_j) k_j u_j^T
// Everything but M0 is known beforehand, so a first kernel forms T = (1 + A)^-1 and P of every chunk at once, and a second
// one takes the chunks of a sequence in order with products only.  Columns of the state (values) do not meet: a workgroup
// of the second kernel takes 16 or 32 of them with four waves.  Two carry the state, half the keys each, in their registers: a
// result of a product (column = lane % 16, rows in registers) is the right operand of the next one as it stands, so nothing
// crosses lanes but a column's largest value, and the waves exchange parts of K M0 and U only.  The two others form the outputs
// from the state and U that the first left in LDS; they also bring V, T and the factors of rows.
//
// Accuracy: T X and P U are products of 32-bit numbers, since a chunk's rows differ by whatever its gates leave of them.  The
// other products run as f16 matrix instructions with sums in 32 bits, an f32 operand as two f16 parts: f16 keys and queries
// enter as they are, f32 ones, and all keys that the state takes, scaled by row with a power of two, so that no row's weight
// is larger for its key being short; unit length, decays and write strengths are factors of rows in f32.  The state before a
// chunk and the writes U that are added to it have a power of two a column each, from its largest, so that neither takes bits
// from the other.  A column of the state is held in the units that its last writes came in.  Sums of log decays are in 64 bits:
// what counts is their differences.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "sc_ops.hpp"

namespace sc {
namespace {

constexpr int kC = 64;                       // tokens of a chunk
constexpr int kWaves = 4, kThreadsC = kWaves * 64;
constexpr float kLeastG = -200.0f;           // a decay of e^-200 is 0 in f32
constexpr double kLog2e = 1.4426950408889634074;
// A column's largest lies at 2^kAim to twice that as an f16 operand; its state is kept below 2^kFar of its units.
constexpr int kAim = 14, kFar = 100;

constexpr int tile_of(int r, int c) { return r * (r + 1) / 2 + c; }   // of the tiles of 16 x 16 up to the diagonal
// Places of a v head's chunk in the workspace, in 16-byte words: T and P by tiles [tile][lane], then the factors of rows.
constexpr uint32_t kOperand = 10 * 64;
enum { kFState = 0, kFBeta = 64, kFWrite = 128, kFQuery = 192, kFDecay = 256, kFactors = 260 };
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
// The product of two tiles of 32-bit numbers: a lane has four values of its row of the left one and, as results lie, of its
// column of the right one.
__device__ __forceinline__ f32x4 product(f32x4 x, f32x4 y, f32x4 acc) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = mfma_f32(x[i], y[i], acc);
    return acc;
}
// n products of their own, side by side: one after the other, each instruction would wait for the one before.
template <int n>
__device__ __forceinline__ void products(f32x4 (&acc)[n], const f32x4 (&x)[n], const f32x4 (&y)[n]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < n; ++j) acc[j] = mfma_f32(x[j][i], y[j][i], acc[j]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Two values, each times `by`, as two f16 parts: the product rounded to nearest, and what that left out rounded likewise (a
// fused multiply-add a value).  What is subtracted is what is multiplied later, not a product that the compiler would round
// once more.
__device__ __forceinline__ void split2(float a, float b, float by_a, float by_b, uint32_t& hi, uint32_t& lo) {
    hi = __builtin_bit_cast(uint32_t, f16x2{_Float16(a * by_a), _Float16(b * by_b)});
    asm("" : "+v"(hi));
    const f16x2 h = __builtin_bit_cast(f16x2, hi);
    const f16x2 l{_Float16(__builtin_fmaf(a, by_a, -float(h.x))), _Float16(__builtin_fmaf(b, by_b, -float(h.y)))};
    lo = __builtin_bit_cast(uint32_t, l);
}
// 2^-e and 2^e for the exponent of x >= 0 (its largest power of two not above), within f32's normal range; 1 for 0.
__device__ __forceinline__ void power_of(float x, float& down, float& up) {
    int e = int(__float_as_uint(x) >> 23) - 127;
    e = x == 0 ? 0 : e > 126 ? 126 : e < -126 ? -126 : e;
    down = __uint_as_float(uint32_t(127 - e) << 23);
    up = __uint_as_float(uint32_t(127 + e) << 23);
}
// 2^x by the hardware's instruction, 1 unit in the last place
__device__ __forceinline__ float exp2_of(double x) { return __builtin_amdgcn_exp2f(float(x)); }

// A sequence's rows and chunks: rows [t0, t1), its first chunk of all.
struct Seq {
    uint32_t s, t0, t1, chunk0;
};
// The rows of sequence s, of the last one past it: two loads at once.
__device__ __forceinline__ void ends_of(const GdnArgs& a, uint32_t s, uint32_t& t0, uint32_t& t1) {
    const int64_t* p = a.cu + (s < a.n_seqs ? s : a.n_seqs - 1);
    const int64_t from = ld_global<int64_t>(p), to = ld_global<int64_t>(p + 1);
    auto bounded = [&](int64_t t) { return t < 0 ? 0u : t > int64_t(a.tokens) ? a.tokens : uint32_t(t); };
    t0 = bounded(from), t1 = bounded(to);
}
// The sequence that `find` (of a sequence and the range of its chunks) looks for; one load a lane and a scan for 64.
template <class Find>
__device__ __forceinline__ bool seq_of(const GdnArgs& a, uint32_t lane, Find find, Seq& q) {
    uint32_t chunks = 0;
    for (uint32_t base = 0; base < a.n_seqs; base += 64) {
        const bool in = base + lane < a.n_seqs;
        uint32_t t0, t1;
        ends_of(a, base + lane, t0, t1);
        const uint32_t n = in && t1 > t0 ? (t1 - t0 + kC - 1) / kC : 0u;
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
// The sequence that has the place `rank` by its chunks of [c0, c1), most first: the longest begin first, so that no long one
// is left to run alone at the end.  Batches of more than 64 are taken as they come.
__device__ __forceinline__ bool seq_of_rank(const GdnArgs& a, uint32_t lane, uint32_t rank, uint32_t c0, uint32_t c1, Seq& q) {
    if (a.n_seqs > 64) return seq_of(a, lane, [&](uint32_t s, uint32_t, uint32_t) { return s == rank; }, q);
    const bool in = lane < a.n_seqs;
    uint32_t t0, t1;
    ends_of(a, lane, t0, t1);
    const uint32_t n = in && t1 > t0 ? (t1 - t0 + kC - 1) / kC : 0u, hi = scan_add(n), lo = hi - n;
    const uint32_t from = lo > c0 ? lo : c0, to = hi < c1 ? hi : c1;
    const uint32_t key = in ? (from < to ? to - from : 0u) * 64 + 64 - lane : 0u;
    uint32_t before = 0;
    for (uint32_t i = 0; i < a.n_seqs; ++i) before += uint32_t(__builtin_amdgcn_readlane(int(key), int(i))) > key;
    const uint64_t here = __ballot(in && before == rank);
    if (!here) return false;
    const int at = __builtin_ctzll(here);
    q.s = uint32_t(at);
    q.t0 = __builtin_amdgcn_readlane(t0, at);
    q.t1 = __builtin_amdgcn_readlane(t1, at);
    q.chunk0 = __builtin_amdgcn_readlane(lo, at);
    return true;
}

// ---- every chunk's T and P ------------------------------------------------------------------------------------------------

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

// Eight values, four each of two tiles, times `by`, as a right operand in two parts.
__device__ __forceinline__ void split_pair(f32x4 a, f32x4 b, f32x4 by_a, f32x4 by_b, ops_u32x4& hi, ops_u32x4& lo) {
    uint32_t h[4], l[4];
    split2(a.x, a.y, by_a.x, by_a.y, h[0], l[0]);
    split2(a.z, a.w, by_a.z, by_a.w, h[1], l[1]);
    split2(b.x, b.y, by_b.x, by_b.y, h[2], l[2]);
    split2(b.z, b.w, by_b.z, by_b.w, h[3], l[3]);
    hi = ops_u32x4{h[0], h[1], h[2], h[3]};
    lo = ops_u32x4{l[0], l[1], l[2], l[3]};
}

// A workgroup takes one chunk of one value head; wave w has its row tile w, tokens 16 w .. 16 w + 15: K K^T and Q K^T by
// tiles up to the diagonal, A and P from them, and of T = (1 + A)^-1 the diagonal tile by substitution, a column a lane; the
// rest of T by products of tiles, T_10 = - T_11 (A_10 T_00) for tiles of 16 and then of 32, with f32 matrix instructions.  A
// product's left tile comes from LDS as rows, its right one is a result in registers as it is: the four terms a lane adds are
// those whose rows it holds.  A chunk of one head is a chain of small steps whose latency bounds a small call (11 us for one
// chunk of 32 heads of 128, f32; 20 by a single wave) and a large one (4096 of them in 55 us, f16, 3.7 TB/s; 50 by single waves,
// which is not worth a kernel more; 5568 in 123 to 147 us, f32, where it also writes the parts of keys and queries, 4 to
// 4.8 TB/s).
// So it keeps room for four workgroups a unit: A, T and P lie where the keys were, and the substitution asks for its rows a few
// at a time (by three workgroups, with all of them at once: 68 and 132 to 165 us).
template <int S, bool kF16>
__global__ void __launch_bounds__(kThreadsC, 4) gdn_prepare_kernel(GdnArgs a, ChunkArgs c) {
    constexpr int kParts = kF16 ? 1 : 2, kSteps = S / 32;
    __shared__ union {
        ops_u32x4 k[kParts][4][kSteps][64];   // keys as operands: [part][tile][step][lane]
        struct {
            float t[10 * kTileFloats], p[10 * kTileFloats];   // then A, which becomes T, and P, by tiles
        } f;
    } s_u;
    auto& s_k = s_u.k;
    float* s_tile = s_u.f.t;
    __shared__ double s_G[kC];
    __shared__ float s_beta[kC], s_fk[kC], s_kk[kC], s_up[kC], s_q[kWaves][2][16];
    __shared__ int s_short[kC];   // f16 keys: the power of two that they are scaled up by for the state's update
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 4, col = lane & 15;
    // workgroups go to the eight XCDs in turn: the value heads of a key head are kept on one, whose L2 then has its rows
    const uint32_t within = blockIdx.x / 8, group = ops_div(within, a.share) * 8 + blockIdx.x % 8;
    const uint32_t piece = group / c.k_heads, kh = group - piece * c.k_heads, h = kh * a.share.d + within % a.share.d;
    const uint32_t chunk = c.first + piece;
    if (piece >= c.count) return;
    Seq q;
    if (!seq_of(a, lane, [&](uint32_t, uint32_t lo, uint32_t hi) { return chunk >= lo && chunk < hi; }, q)) return;
    const uint32_t t0 = q.t0 + (chunk - q.chunk0) * kC, n = q.t1 - t0 < kC ? q.t1 - t0 : kC;
    ops_u32x4* out = c.chunks + (uint64_t(piece) * a.v_heads + h) * kChunkWords;
    ops_u32x4* rows = c.rows + (uint64_t(piece) * c.k_heads + kh) * kRowWords<S, kParts>;
    const bool write_rows = h == kh * a.share.d;   // one of the value heads that share the keys

    // the wave's rows of keys and queries as they lie in memory: token 16 w + col, values 32 step + 8 g .. + 7
    const uint32_t mine = wave * 16 + col, row = mine < n ? mine : n - 1;
    ops_u32x4 k_raw[kParts * kSteps], q_raw[kParts * kSteps], kf[kParts][kSteps], qf[kParts][kSteps];
    {
        const uint8_t* p = a.k + int64_t(t0 + row) * a.k_ld + (kh * S + g * 8) * (kF16 ? 2 : 4);
#pragma unroll
        for (int i = 0; i < kParts * kSteps; ++i) k_raw[i] = ld_global<ops_u32x4>(p + (kF16 ? i * 64 : i / 2 * 128 + i % 2 * 16));
        p = a.q + int64_t(t0 + row) * a.q_ld + (kh * S + g * 8) * (kF16 ? 2 : 4);
#pragma unroll
        for (int i = 0; i < kParts * kSteps; ++i) q_raw[i] = ld_global<ops_u32x4>(p + (kF16 ? i * 64 : i / 2 * 128 + i % 2 * 16));
    }
    // the gates, lane = token
    const bool in = lane < n;
    const int64_t gates = int64_t(t0 + (in ? lane : 0)) * a.gate_ld + h;
    const float g_in = ld_global<float>(a.g + gates), beta_in = ld_global<float>(a.beta + gates);

    // as operands, rows past the chunk zero; f32 ones scaled by a power of two to a largest value of 1 .. 2, in two parts,
    // which the second kernel reads.  The power of two is returned.
    auto to_operand = [&](const ops_u32x4 (&raw)[kParts * kSteps], ops_u32x4 (&x)[kParts][kSteps], uint32_t which) {
        float back = 1.0f;
        if constexpr (kF16) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) x[0][i] = mine < n ? raw[i] : ops_u32x4{};
        } else {
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
            float down;
            power_of(top, down, back);
            const f32x4 by{down, down, down, down};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                split_pair(y[i][0], y[i][1], by, by, x[0][i], x[kParts - 1][i]);
                if (write_rows)
#pragma unroll
                    for (int part = 0; part < kParts; ++part)
                        st_global<ops_u32x4>(rows + row_operand<S, kParts>(which, part, wave, i) + lane, x[part][i]);
            }
        }
        return back;
    };
    const float k_up = to_operand(k_raw, kf, 0);
    if (g == 0) s_up[mine] = k_up;
    if constexpr (kF16) {   // to a largest value of 2^14 .. 2^15, without loss; longer ones as they are
        u16x2 most{};
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, kf[0][i][j] & 0x7FFF7FFFu));
        const float top = over_rows(float(__builtin_bit_cast(_Float16, max(most.x, most.y))), max_of);
        if (g == 0) s_short[mine] = top > 0 ? max(14 + 127 - int(__float_as_uint(top) >> 23), 0) : 0;
    }
#pragma unroll
    for (int part = 0; part < kParts; ++part)
#pragma unroll
        for (int i = 0; i < kSteps; ++i) s_k[part][wave][i][lane] = kf[part][i];
    const float q_up = to_operand(q_raw, qf, 1);
    // sums of the log decays, to base 2
    const double G = scan_add64(in ? double(g_in < kLeastG ? kLeastG : g_in) * kLog2e : 0.0);
    const float beta = in ? beta_in : 0.0f;
    const uint64_t G_bits = __builtin_bit_cast(uint64_t, G);
    const double G_all = __builtin_bit_cast(double, uint64_t(last_lane(uint32_t(G_bits >> 32))) << 32 | last_lane(uint32_t(G_bits)));
    if (wave == 0) s_G[lane] = G, s_beta[lane] = beta;
    __syncthreads();

    // the row tile's products, element (4 g + i, col) of a tile; the diagonals have the squares of the lengths
    f32x4 kk[4], qk[4], qq{};
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        kk[t] = f32x4{}, qk[t] = f32x4{};
        if (uint32_t(t) > wave) continue;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const ops_u32x4 hi = s_k[0][t][i][lane];
            kk[t] = mfma(kf[0][i], hi, kk[t]);
            qk[t] = mfma(qf[0][i], hi, qk[t]);
            if constexpr (!kF16) {
                const ops_u32x4 lo = s_k[kParts - 1][t][i][lane];
                kk[t] = mfma(kf[0][i], lo, kk[t]);
                qk[t] = mfma(qf[0][i], lo, qk[t]);
                kk[t] = mfma(kf[kParts - 1][i], hi, kk[t]);
                qk[t] = mfma(qf[kParts - 1][i], hi, qk[t]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        qq = mfma(qf[0][i], qf[0][i], qq);
        if constexpr (!kF16) qq = mfma(qf[0][i], qf[kParts - 1][i], qq), qq = mfma(qf[kParts - 1][i], qf[0][i], qq);
    }
    f32x4 own{};
#pragma unroll
    for (int t = 0; t < 4; ++t)
        if (uint32_t(t) == wave) own = kk[t];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (g * 4 + i == col) s_kk[mine] = own[i], s_q[wave][0][col] = qq[i];
    // the keys as the left operand of the state's update: keys 32 w + 2 col + e, tokens 32 step + 4 g + j and 16 more
    if (write_rows && wave < uint32_t(kSteps)) {
#pragma unroll
        for (int part = 0; part < kParts; ++part)
#pragma unroll
            for (int step = 0; step < 2; ++step) {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    w[j] = reinterpret_cast<const uint32_t*>(&s_k[part][step * 2 + j / 4][wave][col / 4 * 16 + g * 4 + j % 4])[col % 4];
                    if constexpr (kF16) {
                        const float by = __builtin_amdgcn_ldexpf(1.0f, s_short[step * 32 + j / 4 * 16 + g * 4 + j % 4]);
                        const f16x2 k = __builtin_bit_cast(f16x2, w[j]);
                        w[j] = __builtin_bit_cast(uint32_t, f16x2{_Float16(float(k.x) * by), _Float16(float(k.y) * by)});
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t sel = e ? 0x07060302u : 0x05040100u;
                    st_global<ops_u32x4>(rows + key_operand<S, kParts>(part, wave, e, step) + lane,
                                         ops_u32x4{__builtin_amdgcn_perm(w[1], w[0], sel), __builtin_amdgcn_perm(w[3], w[2], sel),
                                                   __builtin_amdgcn_perm(w[5], w[4], sel), __builtin_amdgcn_perm(w[7], w[6], sel)});
                }
            }
    }
    __syncthreads();
    // the factor that brings a row as multiplied to its length, unit or its own, and that length
    auto factor = [&](float squares, float by, bool there) {
        return !there ? 0.0f : a.l2norm ? __builtin_amdgcn_rsqf(squares + a.eps / by / by) : by;
    };
    const float fk = factor(s_kk[lane], s_up[lane], in);
    float* f = reinterpret_cast<float*>(out + 2 * kOperand);
    if (wave == 0) {
        s_fk[lane] = fk;
        f[kFState + lane] = beta * fk * exp2_of(G);
        f[kFBeta + lane] = beta;
        // a key that is 0 writes nothing, whatever its factor
        const float write = s_kk[lane] == 0 ? 0.0f : exp2_of(G_all - G) * fk;
        f[kFWrite + lane] = kF16 ? __builtin_amdgcn_ldexpf(write, -s_short[lane]) : write;
        if (lane == 0) f[kFDecay] = exp2_of(G_all);
    }
    if (g == 0) {
        const float fq = factor(s_q[wave][0][col], q_up, mine < n) * a.scale;
        s_q[wave][1][col] = fq;
        f[kFQuery + mine] = fq * exp2_of(s_G[mine]);
    }
    __syncthreads();
    // A below the diagonal, and P, by way of LDS
    double Gr[4];
    float br[4], qr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t t = wave * 16 + g * 4 + i;
        Gr[i] = s_G[t];
        br[i] = s_beta[t] * s_fk[t];
        qr[i] = s_q[wave][1][g * 4 + i];
    }
    float* tiles = s_tile + wave * (wave + 1) / 2 * kTileFloats;   // the wave's row of them
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        if (uint32_t(t) > wave) continue;
        const double Gc = s_G[t * 16 + col];
        const float fc = s_fk[t * 16 + col];
        const bool below = uint32_t(t) < wave;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t r = g * 4 + i;
            const float fade = below || r >= col ? exp2_of(Gr[i] - Gc) * fc : 0.0f;
            tiles[t * kTileFloats + r * kTileRow + col] = below || r > col ? br[i] * fade * kk[t][i] : 0.0f;
            s_u.f.p[(wave * (wave + 1) / 2 + t) * kTileFloats + r * kTileRow + col] = qr[i] * fade * qk[t][i];
        }
    }
    wave_sync();
    // a row tile of P or T as the second kernel's left operands: row col, places 4 g .. + 3
    auto write_operand = [&](const float* from, uint32_t which) {
        for (uint32_t t = 0; t <= wave; ++t)
            st_global<ops_u32x4>(out + which * kOperand + (wave * (wave + 1) / 2 + t) * 64 + lane,
                                 *reinterpret_cast<const ops_u32x4*>(&from[t * kTileFloats + col * kTileRow + g * 4]));
    };
    write_operand(s_u.f.p + wave * (wave + 1) / 2 * kTileFloats, 1);
    // the diagonal tile of T, column col (the same in each group of lanes)
    auto tile_at = [&](int t) { return s_tile + t * kTileFloats; };
    {
        float* d = tiles + wave * kTileFloats;
        uint32_t row0 = 0;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            f32x4 sum{uint32_t(i) == col ? 1.0f : 0.0f, 0, 0, 0};   // four sums: a chain a quarter as long
#pragma unroll
            for (int k = 0; k < i; k += 4) {
                const f32x4 r = *reinterpret_cast<const f32x4*>(&d[row0 + i * kTileRow + k]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (k + j < i) sum[j] -= r[j] * x[k + j];
            }
            x[i] = (sum.x + sum.y) + (sum.z + sum.w);
            if (i == 3 || i == 7 || i == 11) asm volatile("" : "+v"(row0), "+v"(x[i]));   // not all rows at once
        }
        wave_sync();
        if (g == 0)
#pragma unroll
            for (int i = 0; i < 16; ++i) d[i * kTileRow + col] = x[i];
    }
    auto left = [&](int t) { return *reinterpret_cast<const f32x4*>(tile_at(t) + col * kTileRow + g * 4); };
    auto right = [&](int t) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = tile_at(t)[(g * 4 + i) * kTileRow + col];
        return x;
    };
    auto put = [&](int t, f32x4 x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) tile_at(t)[(g * 4 + i) * kTileRow + col] = x[i];
    };
    __syncthreads();
    const f32x4 zero{};
    if (wave & 1) {   // T_10 and T_32
        const int w = int(wave), at = tile_of(w, w - 1);
        const f32x4 x = product(left(at), right(tile_of(w - 1, w - 1)), zero);
        const f32x4 y = -product(left(tile_of(w, w)), x, zero);
        wave_sync();
        put(at, y);
    }
    __syncthreads();
    {
        // T_rc of the lower left half, r = 2, 3 and c = 0, 1, from the column y of A T there
        const int r = 2 + int(wave >> 1), cc = int(wave & 1);
        f32x4 y2 = product(left(tile_of(2, 1)), right(tile_of(1, cc)), zero), y3{};
        if (cc == 0) y2 = product(left(tile_of(2, 0)), right(tile_of(0, 0)), y2);
        f32x4 z;
        if (r == 2) {
            z = product(left(tile_of(2, 2)), y2, zero);
        } else {
            y3 = product(left(tile_of(3, 1)), right(tile_of(1, cc)), zero);
            if (cc == 0) y3 = product(left(tile_of(3, 0)), right(tile_of(0, 0)), y3);
            z = product(left(tile_of(3, 3)), y3, product(left(tile_of(3, 2)), y2, zero));
        }
        __syncthreads();   // everyone has read A there
        put(tile_of(r, cc), -z);
    }
    __syncthreads();
    write_operand(tiles, 0);
}

// ---- the chunks of a sequence in order ------------------------------------------------------------------------------------

// Waves of a workgroup of the second kernel: the state's keys are shared by two where there are 64 or more, two others form
// the outputs.
template <int S>
constexpr int kStateWaves = S >= 64 ? 2 : 1;
constexpr int kOutWaves = 2;

template <class T>
__device__ __forceinline__ T pick(bool first, T a, T b) { return first ? a : b; }

template <int kSteps>
__device__ __forceinline__ float most_of(const f32x4 (&m)[kSteps][2]) {
    float top = 0;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < 4; j += 2) top = fmaxf(fmaxf(top, fabsf(m[i][e][j])), fabsf(m[i][e][j + 1]));
    return over_rows(top, max_of);
}
// What a largest value is to be scaled down by to lie at 2^kAim, as an exponent whose power f32 holds either way.
__device__ __forceinline__ int exponent_of(float top) { return max(int(__float_as_uint(top) >> 23) - 127 - kAim, -126); }
// Keys 32 i + 8 g .. + 7 of the state as a right operand: the even ones and the odd ones take turns.
__device__ __forceinline__ void split_state(const f32x4 (&m)[2], float by, ops_u32x4& hi, ops_u32x4& lo) {
    const f32x4 four{by, by, by, by};
    split_pair(f32x4{m[0].x, m[1].x, m[0].y, m[1].y}, f32x4{m[0].z, m[1].z, m[0].w, m[1].w}, four, four, hi, lo);
}

// kN tiles of 16 columns.  With one, the state's two waves form half of U's rows each; with two, each forms U of its tile.  One
// sequence is bound by the chain of a chunk's products, splits and barriers, 1.9 us each (8192 tokens, 32 heads of 128, f16:
// 235 to 253 us, 4000 cycles a chunk).  Many are bound by that chain and by the operands that their workgroups read through
// their caches, 2.8 GB for 10 854 tokens of eight sequences in f32: 280 to 350 us, 8 to 10 TB/s of them, with the matrix units
// busy two fifths of the time.
template <int S, int kN, bool kF16>
__global__ void __launch_bounds__((kStateWaves<S> + kOutWaves) * 64, 2) gdn_chunk_kernel(GdnArgs a, ChunkArgs c) {
    constexpr int kParts = kF16 ? 1 : 2, kSteps = S / 32, kShares = kStateWaves<S>, kMine = kSteps / kShares;
    static_assert(kN == 1 || kShares == 2);
    constexpr uint32_t kCols = kN * 16, kThreads = (kShares + kOutWaves) * 64;
    constexpr uint32_t kBytes = kF16 ? 2 : 4;                            // of an activation
    constexpr uint32_t kRowV = kCols * kBytes, kPieces = kRowV / 16;     // a row of V or O of this workgroup, in 16-byte pieces
    constexpr uint32_t kEach = kC * kPieces / (kOutWaves * 64);          // pieces of a lane
    // where registers are few, the keys' second form is asked for within its chunk and the first one at its end
    constexpr bool kAhead = kF16, kOwnT = kF16 && kN == 1 && kShares == 2;
    // Right operands are [tile][step][part][lane], results [tile of columns][tile of rows][lane].  A chunk has three parts: a
    // barrier opens it, another comes where K M0 is known, the third where U is.  What lies here is written in one part and
    // read in later ones, before the next chunk's part that writes it again.
    __shared__ ops_u32x4 s_m[kN][kSteps][2][64];              // the state before the chunk: written in the first part, read in the second
    __shared__ f32x4 s_u[kN][4][64];                          // U: second, third
    __shared__ f32x4 s_v[kN][4][64];                          // beta V: first, second
    __shared__ f32x4 s_t[kOwnT ? 1 : 10][64];                 // T: first, second
    __shared__ f32x4 s_km[kShares][4][64];                    // K M0 by a wave's keys: first, second
    __shared__ __align__(16) uint8_t s_stage[kOutWaves][32 * kRowV];   // a wave's rows of V or O on their way
    __shared__ __align__(16) float s_f[2][(kFactors + 63) / 64 * 64];  // of rows: second; all of the next chunk, the first after it
    __shared__ float s_back[kN][16];                          // what brings a column's products with the state back: first, second
    __shared__ float s_top[kShares][kN][16];                  // the largest of a wave's state by column: third; the next first
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t g = lane >> 4, col = lane & 15;
    // workgroups go to the eight XCDs in turn: the column blocks of the value heads of a key head are kept on one
    constexpr uint32_t kBlocks = S / kCols;
    const uint32_t within = blockIdx.x / 8, heads8 = within / kBlocks, block = within % kBlocks;
    const uint32_t group = ops_div(heads8, a.share) * 8 + blockIdx.x % 8, rank = group / c.k_heads;
    if (rank >= a.n_seqs) return;
    const uint32_t kh = group - rank * c.k_heads, h = kh * a.share.d + heads8 % a.share.d;
    Seq q;
    if (!seq_of_rank(a, lane, rank, c.first, c.first + c.count, q)) return;
    // this launch's chunks of the sequence
    const uint32_t all = q.t1 > q.t0 ? (q.t1 - q.t0 + kC - 1) / kC : 0u;
    const uint32_t c0 = q.chunk0 > c.first ? q.chunk0 : c.first, c1 = q.chunk0 + all < c.first + c.count ? q.chunk0 + all : c.first + c.count;
    if (c0 >= c1) return;
    float* base = a.state[q.s];
    if (!base) {
        const uint32_t from = q.t0 + (c0 - q.chunk0) * kC, to = q.t0 + (c1 - q.chunk0) * kC < q.t1 ? q.t0 + (c1 - q.chunk0) * kC : q.t1;
        for (uint32_t t = from + tid / (kCols / 4); t < to; t += kThreads / (kCols / 4))
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
    // Operand `word / 64` of a key head's: the lane's offset holds what an instruction's own offset cannot, a scalar address
    // each would take more scalar registers than there are.
    auto row_word = [&](const ops_u32x4* from, uint32_t word) {
        uint32_t at = lane * 16 + (word / 512 * 8 + 4) * 1024;
        asm("" : "+v"(at));
        return reinterpret_cast<const uint8_t*>(from) + at + (int(word / 64 % 8) - 4) * 1024;
    };
    // a tile of keys or queries as left operands, N steps from `first` on
    auto load_rows = [&](auto& x, uint32_t chunk, uint32_t which, uint32_t tile, uint32_t first) {
        constexpr int N = sizeof(x[0]) / sizeof(x[0][0]);
        if constexpr (kF16) {
            const uint32_t ld = uint32_t(which ? a.q_ld : a.k_ld);
            const uint8_t* p = (which ? a.q : a.k) + int64_t(q.t0 + (chunk - q.chunk0) * kC) * ld + kh * S * 2 + first * 64;
            const uint32_t at = min((tile * 16 + col) * ld, last_row(chunk) * ld) + g * 16;
#pragma unroll
            for (int i = 0; i < N; ++i) x[0][i] = ld_global<ops_u32x4>(p + at + i * 64);
        } else {
            const ops_u32x4* p = rows_of(chunk) + (tile * kSteps + first) * 64;
#pragma unroll
            for (int part = 0; part < kParts; ++part)
#pragma unroll
                for (int i = 0; i < N; ++i) x[part][i] = ld_global<ops_u32x4>(row_word(p, row_operand<S, kParts>(which, part, 0, i)));
        }
    };
    // The five tiles up to the diagonal of rows w and then of rows 3 - w.
    auto row_and_other = [](uint32_t w, uint32_t i) { return i <= w ? w * (w + 1) / 2 + i : (3 - w) * (4 - w) / 2 + i - w - 1; };

    if (wave < kShares) {
        // the state: keys 32 (first + i) + 8 g + 2 j + e in m[b][i][e][j], a column a lane
        const uint32_t first = wave * kMine;
        float* state = base + a.state_offset + h * a.head_ld + block * kCols + col + (first * 32 + g * 8) * a.key_ld;
        f32x4 m[kN][kMine][2];
#pragma unroll
        for (int b = 0; b < kN; ++b)
#pragma unroll
            for (int i = 0; i < kMine; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < 4; ++j) m[b][i][e][j] = ld_global<float>(state + (i * 32 + 2 * j + e) * a.key_ld + b * 16);
        // waited for here: the loop would wait for it every time around
#pragma unroll
        for (int b = 0; b < kN; ++b)
#pragma unroll
            for (int i = 0; i < kMine; ++i) asm volatile("" : "+v"(m[b][i][0]), "+v"(m[b][i][1]));
        ops_u32x4 k[4][kParts][kMine], kt[kParts][kMine][2][2];
        f32x4 t_own[kOwnT ? 5 : 1];   // a wave's two rows of T's tiles
        auto load_t = [&](uint32_t chunk) {
            const ops_u32x4* from = operands_of(chunk) + lane;
#pragma unroll
            for (uint32_t i = 0; i < 5; ++i) t_own[kOwnT ? i : 0] = ld_global<f32x4>(from + row_and_other(wave, i) * 64);
        };
        auto load_keys = [&](uint32_t chunk) {
#pragma unroll
            for (int r = 0; r < 4; ++r) load_rows(k[r], chunk, 0, r, first);
        };
        auto load_turned = [&](uint32_t chunk) {
            const ops_u32x4* p = rows_of(chunk) + first * 256;
#pragma unroll
            for (int part = 0; part < kParts; ++part)
#pragma unroll
                for (int i = 0; i < kMine; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int step = 0; step < 2; ++step) kt[part][i][e][step] = ld_global<ops_u32x4>(row_word(p, key_operand<S, kParts>(part, i, e, step)));
        };
        load_keys(c0);
        if (kOwnT) load_t(c0);
        if (kAhead) load_turned(c0);
        int up[kN];   // a column's state is m times 2^up
#pragma unroll
        for (int b = 0; b < kN; ++b) {
            up[b] = 0;
            const float top = most_of<kMine>(m[b]);
            if (g == 0) s_top[wave][b][col] = top;
        }
        for (uint32_t chunk = c0; chunk < c1; ++chunk) {
            const uint32_t ahead = clamped(chunk + 1);
            __syncthreads();
            const float* f = s_f[(chunk - c0) & 1];
            // the state as a right operand, its column's largest at 2^kAim
            ops_u32x4 mh[kN][kMine], ml[kN][kMine];
            float back[kN];
            int reach[kN];   // the exponent of the column's largest, in all
#pragma unroll
            for (int b = 0; b < kN; ++b) {
                const float top = fmaxf(s_top[0][b][col], s_top[kShares - 1][b][col]);
                const int e = top > 0 ? exponent_of(top) : 0;
                const float by = __builtin_amdgcn_ldexpf(1.0f, -e);
                reach[b] = top > 0 ? e + up[b] + kAim : INT_MIN;
                back[b] = __builtin_amdgcn_ldexpf(1.0f, e + up[b]);
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    split_state(m[b][i], by, mh[b][i], ml[b][i]);
                    s_m[b][first + i][0][lane] = mh[b][i];
                    s_m[b][first + i][1][lane] = ml[b][i];
                }
                if (wave == 0 && g == 0) s_back[b][col] = back[b];
            }
            // K M0
            f32x4 km[kN][4];
#pragma unroll
            for (int b = 0; b < kN; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) km[b][r] = f32x4{};
#pragma unroll
            for (int i = 0; i < kMine; ++i)
#pragma unroll
                for (int x = 0; x < kParts + 1; ++x)   // high by high, high by low, low by high
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int b = 0; b < kN; ++b) km[b][r] = mfma(k[r][x == 2][i], x == 1 ? ml[b][i] : mh[b][i], km[b][r]);
            if (kAhead) load_keys(ahead);
            else load_turned(chunk);
            // the factors of K M0's rows, with what brings it back; asked for now where there are registers
            auto factors_of = [&](int r) {
                return *reinterpret_cast<const f32x4*>(&f[kFState + r * 16 + g * 4]) * (kN == 1 ? float(back[0]) : pick(wave, back[kN - 1], back[0]));
            };
            f32x4 fs[4];
            if constexpr (kN == 1)
#pragma unroll
                for (int r = 0; r < 4; ++r) fs[r] = factors_of(r);
            // with one tile each wave's part goes to the other, with two the part of the other's tile
            const uint32_t tile = kN == 1 ? 0 : wave;
            if constexpr (kShares > 1) {
#pragma unroll
                for (int r = 0; r < 4; ++r) s_km[wave][r][lane] = kN == 1 ? f32x4(km[0][r]) : pick(wave, km[0][r], km[kN - 1][r]);
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (kN > 1) km[0][r] = pick(wave, km[kN - 1][r], km[0][r]);
                if constexpr (kShares > 1) km[0][r] += s_km[wave ^ 1][r][lane];   // the same sum in both waves
            }
            // X; rows past the sequence's end are zero, as their V and factors are
            f32x4 x[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (kN > 1) fs[r] = factors_of(r);
                const f32x4 v = s_v[tile][r][lane];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[r][j] = __builtin_fmaf(-fs[r][j], km[0][r][j], v[j]);
            }
            // U = T X; weighted, it is what the state takes, its column's largest at 2^kAim.  With one tile of columns the state's
            // waves have two row tiles each, five of T's ten tiles; with two, each has its columns'.
            ops_u32x4 ws[kN][2][2];
            int to[kN];
            {
                f32x4 fw[4];
                if constexpr (kN == 1)
#pragma unroll
                    for (int r = 0; r < 4; ++r) fw[r] = *reinterpret_cast<const f32x4*>(&f[kFWrite + r * 16 + g * 4]);
                if constexpr (kN == 1 && kShares == 2) {
                    f32x4 t[5];
#pragma unroll
                    for (uint32_t i = 0; i < 5; ++i) t[i] = kOwnT ? t_own[i] : s_t[row_and_other(wave, i)][lane];
                    // row `wave` in y[0], row 3 - wave in y[1] and y[2]
                    f32x4 y[3]{};
                    if (wave) {
                        products(y, {t[0], t[2], t[3]}, {x[0], x[0], x[1]});
                        f32x4 z[2]{y[0], y[1]};
                        products(z, {t[1], t[4]}, {x[1], x[2]});
                        y[0] = z[0], y[1] = z[1];
                    } else {
                        products(y, {t[0], t[1], t[2]}, {x[0], x[0], x[1]});
                        f32x4 z[2]{y[1], y[2]};
                        products(z, {t[3], t[4]}, {x[2], x[3]});
                        y[1] = z[0], y[2] = z[1];
                    }
                    if (kOwnT) load_t(ahead);
                    s_u[0][wave][lane] = y[0];
                    s_u[0][3 - wave][lane] = y[1] + y[2];
                } else {
                    auto t = [&](int r, int c) { return s_t[tile_of(r, c)][lane]; };
                    f32x4 y[4]{};
                    products(y, {t(0, 0), t(1, 0), t(2, 0), t(3, 0)}, {x[0], x[0], x[0], x[0]});
                    f32x4 z[3]{y[1], y[2], {}};   // row 3 in two sums
                    products(z, {t(1, 1), t(2, 1), t(3, 1)}, {x[1], x[1], x[1]});
                    f32x4 last[3]{z[1], y[3], z[2]};
                    products(last, {t(2, 2), t(3, 2), t(3, 3)}, {x[2], x[2], x[3]});
                    s_u[tile][0][lane] = y[0];
                    s_u[tile][1][lane] = z[0];
                    s_u[tile][2][lane] = last[0];
                    s_u[tile][3][lane] = last[1] + last[2];
                }
                __syncthreads();
#pragma unroll
                for (int b = 0; b < kN; ++b) {
                    float top = 0;
                    f32x4 w[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const f32x4 u = s_u[b][r][lane];
                        if constexpr (kN > 1) fw[r] = *reinterpret_cast<const f32x4*>(&f[kFWrite + r * 16 + g * 4]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            w[r][j] = u[j] * fw[r][j];
                            top = fmaxf(top, fabsf(w[r][j]));
                        }
                    }
                    top = over_rows(top, max_of);
                    to[b] = top > 0 ? max(max(exponent_of(top), reach[b] == INT_MIN ? INT_MIN : reach[b] - kFar), up[b] - 126) : up[b];
                    const float by = __builtin_amdgcn_ldexpf(1.0f, -to[b]);
                    const f32x4 four{by, by, by, by};
#pragma unroll
                    for (int step = 0; step < 2; ++step) split_pair(w[step * 2], w[step * 2 + 1], four, four, ws[b][step][0], ws[b][step][1]);
                }
            }
            // the state after the chunk, in the units of what is added
#pragma unroll
            for (int b = 0; b < kN; ++b) {
                const float decay = __builtin_amdgcn_ldexpf(f[kFDecay], up[b] - to[b]);
                up[b] = to[b];
#pragma unroll
                for (int i = 0; i < kMine; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) m[b][i][e] *= decay;
            }
#pragma unroll
            for (int step = 0; step < 2; ++step)
#pragma unroll
                for (int x = 0; x < kParts + 1; ++x)
#pragma unroll
                    for (int i = 0; i < kMine; ++i)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
#pragma unroll
                            for (int b = 0; b < kN; ++b) m[b][i][e] = mfma(kt[x == 2][i][e][step], ws[b][step][x == 1], m[b][i][e]);
            if (kAhead) load_turned(ahead);
            else load_keys(ahead);
#pragma unroll
            for (int b = 0; b < kN; ++b) {
                const float top = most_of<kMine>(m[b]);
                if (g == 0) s_top[wave][b][col] = top;
            }
        }
        __syncthreads();   // the last chunk's outputs
#pragma unroll
        for (int b = 0; b < kN; ++b)
#pragma unroll
            for (int i = 0; i < kMine; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        st_global<float>(state + (i * 32 + 2 * j + e) * a.key_ld + b * 16, __builtin_amdgcn_ldexpf(m[b][i][e][j], up[b]));
        return;
    }

    // The other waves: V, T and the factors, and the outputs, whose part from U is formed where U is known.  Wave w of the two
    // takes the row tiles w and 3 - w, which have five of P's ten.
    const uint32_t w = wave - kShares, v_ld = uint32_t(a.v_ld);
    uint8_t* stage = s_stage[w];
    auto row_tile = [&](uint32_t i) { return i ? 3 - w : w; };
    auto row_at = [&](uint32_t at) { return row_tile(at / (16 * kPieces)) * 16 + at / kPieces % 16; };   // of piece `at` of the wave's rows
    ops_u32x4 v_in[kEach];
    f32x4 t_in[5];
    float f_in[3];
    f32x4 v[kN][2];
    auto factor_at = [&](uint32_t i) { return (i == 0 ? 1 : w ? i + 2 : (i - 1) * 2) * 64 + lane; };   // both have kFBeta's
    auto load_early = [&](uint32_t chunk) {
        const uint32_t last = last_row(chunk) * v_ld;
        const uint8_t* p = a.v + int64_t(q.t0 + (chunk - q.chunk0) * kC) * a.v_ld + (h * S + block * kCols) * kBytes;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t at = lane + i * 64;
            v_in[i] = ld_global<ops_u32x4>(p + min(row_at(at) * v_ld, last) + at % kPieces * 16);
        }
        const float* f = reinterpret_cast<const float*>(operands_of(chunk) + 2 * kOperand);
#pragma unroll
        for (uint32_t i = 0; i < 3; ++i) f_in[i] = ld_global<float>(f + min(factor_at(i), uint32_t(kFactors - 1)));
    };
    // V as the state's waves take it, by way of LDS: times beta, rows past the sequence's end zero, a lane's four rows together
    auto put_early = [&](uint32_t chunk, uint32_t n) {
        const uint32_t last = last_row(chunk);
        float* f = s_f[n & 1];
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t at = lane + i * 64;
            *reinterpret_cast<ops_u32x4*>(&stage[at * 16]) = row_at(at) <= last ? v_in[i] : ops_u32x4{};
        }
#pragma unroll
        for (uint32_t i = 0; i < 3; ++i) f[factor_at(i)] = f_in[i];
        wave_sync();
#pragma unroll
        for (int b = 0; b < kN; ++b) {
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                f32x4 x = *reinterpret_cast<const f32x4*>(&f[kFBeta + row_tile(i) * 16 + g * 4]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint8_t* p = &stage[(i * 16 + g * 4 + j) * kRowV + (b * 16 + col) * kBytes];
                    if constexpr (kF16) x[j] *= float(*reinterpret_cast<const _Float16*>(p));
                    else x[j] *= *reinterpret_cast<const float*>(p);
                }
                v[b][i] = x;
            }
        }
        wave_sync();
    };
    auto load_t = [&](uint32_t chunk) {
#pragma unroll
        for (int i = 0; i < 5; ++i) t_in[i] = ld_global<f32x4>(operands_of(chunk) + (w * 5 + i) * 64 + lane);
    };
    ops_u32x4 qs[2][kParts][kSteps];
    f32x4 p[5];
    auto load_queries = [&](uint32_t chunk) {
        load_rows(qs[0], chunk, 1, w, 0);
        load_rows(qs[1], chunk, 1, 3 - w, 0);
    };
    // P's tiles of rows w, then those of rows 3 - w
    auto load_p = [&](uint32_t chunk) {
        const ops_u32x4* from = operands_of(chunk) + kOperand + lane;
#pragma unroll
        for (uint32_t i = 0; i < 5; ++i) p[i] = ld_global<f32x4>(from + row_and_other(w, i) * 64);
    };
    f32x4 qm[kN][2], sum[kN][2];
    float back[kN];
    // P U: a wave's second tile is of rows w or 3 - w
    auto outputs_of_u = [&] {
#pragma unroll
        for (int b = 0; b < kN; ++b) {
            auto u = [&](uint32_t r) { return s_u[b][r][lane]; };
            f32x4 near = product(p[0], u(0), f32x4{}), far{}, odd = product(p[3], u(2 - w), f32x4{});   // rows 3 - w in two sums
            const f32x4 x = product(p[1], u(w), w ? near : far);
            near = w ? x : near;
            far = product(p[2], u(1 - w), w ? far : x);
            odd = product(p[4], u(3 - w), odd);
            sum[b][0] = near, sum[b][1] = far + odd;
        }
    };
    auto first_part = [&](uint32_t chunk) {
#pragma unroll
        for (int b = 0; b < kN; ++b)
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) s_v[b][row_tile(i)][lane] = v[b][i];
#pragma unroll
        for (uint32_t i = 0; i < 5 && !kOwnT; ++i) s_t[w * 5 + i][lane] = t_in[i];
        if (!kOwnT) load_t(clamped(chunk + 1));
    };
    auto rest = [&](uint32_t chunk) {
        __syncthreads();
#pragma unroll
        for (int b = 0; b < kN; ++b)
#pragma unroll
            for (int r = 0; r < 2; ++r) qm[b][r] = f32x4{};
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int b = 0; b < kN; ++b) {
                const ops_u32x4 hi = s_m[b][i][0][lane], lo = s_m[b][i][1][lane];
#pragma unroll
                for (int x = 0; x < kParts + 1; ++x)
#pragma unroll
                    for (int r = 0; r < 2; ++r) qm[b][r] = mfma(qs[r][x == 2][i], x == 1 ? lo : hi, qm[b][r]);
            }
#pragma unroll
        for (int b = 0; b < kN; ++b) back[b] = s_back[b][col];
        load_queries(clamped(chunk + 1));
        // the next chunk's V, while the state's waves form U
        put_early(clamped(chunk + 1), chunk + 1 - c0);
        load_early(clamped(chunk + 2));
        __syncthreads();
        outputs_of_u();
        load_p(clamped(chunk + 1));
    };
    auto outputs = [&](uint32_t done) {
        const uint32_t last = last_row(done);
        const float* f = s_f[(done - c0) & 1];
#pragma unroll
        for (int b = 0; b < kN; ++b) {
#pragma unroll
            for (uint32_t r = 0; r < 2; ++r) {
                const uint32_t row = row_tile(r) * 16 + g * 4;
                const f32x4 fq = *reinterpret_cast<const f32x4*>(&f[kFQuery + row]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float o = __builtin_fmaf(fq[j], qm[b][r][j] * back[b], sum[b][r][j]);
                    uint8_t* to = &stage[(r * 16 + g * 4 + j) * kRowV + (b * 16 + col) * kBytes];
                    if constexpr (kF16) *reinterpret_cast<_Float16*>(to) = _Float16(o);
                    else *reinterpret_cast<float*>(to) = o;
                }
            }
        }
        wave_sync();
        uint8_t* to = a.out + int64_t(q.t0 + (done - q.chunk0) * kC) * a.out_ld + (h * S + block * kCols) * kBytes;
        uint32_t o_ld = __builtin_amdgcn_readfirstlane(uint32_t(a.out_ld));
        asm volatile("" : "+s"(o_ld));   // the rows' offsets formed here: kept, they would have to be read from memory
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t at = lane + i * 64, row = row_at(at);
            if (row <= last) st_global<ops_u32x4>(to + (row * o_ld + at % kPieces * 16), *reinterpret_cast<const ops_u32x4*>(&stage[at * 16]));
        }
        wave_sync();
    };
    load_early(c0);
    if (!kOwnT) load_t(c0);
    put_early(c0, 0);
    load_queries(c0);
    load_early(clamped(c0 + 1));
    __syncthreads();
    first_part(c0);
    load_p(c0);
    rest(c0);
    for (uint32_t chunk = c0 + 1; chunk < c1; ++chunk) {
        __syncthreads();
        first_part(chunk);
        outputs(chunk - 1);
        rest(chunk);
    }
    __syncthreads();
    outputs(c1 - 1);
}

// Two tiles of columns a workgroup halve what a chunk's operands cost in reads (126 KB for f32, 68 for f16), one gives twice
// as many workgroups, each with less to do between its barriers.  Measured in us for both kernels, sequences of 32 heads of
// 128 and up to 1024 tokens, two tiles against one: f16 59 : 42 for one sequence, 64 : 58 for two, 74 : 68, 92 : 104 for four,
// 112 : 136 for eight; f32 72 : 51, 86 : 78, 96 : 90, 120 : 136, 149 : 178.  So two where that leaves the chip's 256 units two
// workgroups each, if all sequences of the call were in one piece.
constexpr uint32_t kWideFrom = 512;

template <int S, bool kF16>
void launch_chunks(const GdnArgs& a, const ChunkArgs& c, hipStream_t stream) {
    auto by_eight = [&](uint32_t rows) { return (rows * c.k_heads + 7) / 8 * 8 * a.share.d; };   // value heads, key heads by eights
    const uint32_t heads = by_eight(a.n_seqs);
    const dim3 threads((kStateWaves<S> + kOutWaves) * 64);
    hipLaunchKernelGGL((gdn_prepare_kernel<S, kF16>), dim3(by_eight(c.count)), dim3(kThreadsC), 0, stream, a, c);
    if constexpr (S >= 64)
        if (a.n_seqs * a.v_heads * (S / 32) >= kWideFrom) {
            hipLaunchKernelGGL((gdn_chunk_kernel<S, 2, kF16>), dim3(heads * (S / 32)), threads, 0, stream, a, c);
            return;
        }
    hipLaunchKernelGGL((gdn_chunk_kernel<S, 1, kF16>), dim3(heads * (S / 16)), threads, 0, stream, a, c);
}
template <int S>
hipError_t launch_of(const GdnArgs& a, const ChunkArgs& plan, bool f16, hipStream_t stream) {
    for (ChunkArgs c = plan; c.first < plan.total; c.first += plan.count) {
        c.count = plan.total - c.first < plan.count ? plan.total - c.first : plan.count;
        if (f16) launch_chunks<S, true>(a, c, stream);
        else launch_chunks<S, false>(a, c, stream);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// Chunks of one pair of launches: a long prompt goes through the workspace in pieces, which bounds it (1.2 GB at most for 32
// heads of 128 in f32).  A piece of one sequence stays in the memory's own cache, 256 MB, until it has been read: 32 768 tokens
// of 32 heads of 128 take 1104, 1077, 1125 and 1115 us by pieces of 64, 128, 256 and 512 chunks in f16, 1426, 1666, 1611 and
// 1576 in f32, whose pieces are twice as large.  The numbers are for such heads: fewer or smaller ones have pieces that are a
// fraction of what fits.  Each further sequence adds as many chunks, up to 512; but a piece is a run of the chunks of all sequences
// in order, so that it holds many short sequences, or one or two of several long ones.
constexpr uint32_t kMostChunks = 512;

}  // namespace

uint64_t plan_gdn_chunks(const GdnArgs& a, int size, bool f16, ChunkArgs& c) {
    // a sequence has at most one chunk that is not full, of one token at least
    c.total = uint32_t((a.tokens + uint64_t(kC - 1) * (a.n_seqs < a.tokens ? a.n_seqs : a.tokens)) / kC);
    const uint32_t each = f16 ? 128 : 64, most = a.n_seqs < kMostChunks / each ? a.n_seqs * each : kMostChunks;
    c.count = c.total < most ? c.total : most;
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
