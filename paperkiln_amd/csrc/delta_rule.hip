// Gated delta rule, forward: over a sequence in chunks of 64 tokens, and token by token.
//
//   S_t = e^{g_t} S_{t-1} + k_t u_t^T,   u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t),   o_t = scale S_t^T q_t
//
// In chunks (delta_rule.h) one launch forms what does not depend on a state, T and A of every chunk, and a second one walks down the chunks, a workgroup for 16 or 32 columns of a
// head's state: the columns do not know of one another. What bounds the walk is its own chain: three products and three exchanges through LDS a chunk, 3.4 us of it. (One of the three, U = T R,
// is there because T is kept by itself: U = T beta V - (T beta gamma K) S has its products with T outside of the chain, for as many more of them beside the chunks' matrices.)
// 4 x 4096 tokens, 16 heads of 128 in bf16: the chunks' matrices 77 us (3.7 TB/s of 134 MB read and 154 written), the walk 216 us, 203 if it leaves the states for the backward in place of O.
// Token by token, the state in registers, memory bounds one token: the state read and written once. One token of 256 sequences, 16 heads of 128: 119 us, 4.5 TB/s; of one sequence 5 us.
// Of several tokens each one's k, q, v and decay are asked for in its own turn, behind the barrier of the one before: 8 tokens of those 256 sequences 345 us, 217 in fp32.
#include "delta_rule.h"

namespace pk {
namespace delta {
namespace {

// e^x, x from differences in 64 bits; a decay below e^-1000 is none.
__device__ inline float decay_of(double x) { return __builtin_amdgcn_exp2f(static_cast<float>(x * 1.4426950408889634074)); }
__device__ inline double held(float g) { return g < -1000.0f ? -1000.0 : static_cast<double>(g); }

// ---- what does not depend on a state ----
// A workgroup for a unit's chunk. T by 16 x 16 blocks: those of the diagonal by forward substitution, a lane for each column and a wavefront for each block, the others by
// T_ij = -T_ii sum_k M_ik T_kj, one diagonal after the other on the matrix cores. (All 64 rows by substitution are 2016 additions
// one behind the other: 32 us however few the chunks.) Three wavefronts to a SIMD: of four the registers would be spilled (99 us in place of 78).
constexpr int MP = C + 4, XP = 20;
template <typename T, int DK, bool BACKWARD, Rows BY>
__global__ __launch_bounds__(256, PARTS<T> == 1 ? 3 : 2) void chunk_matrices(Rule a) {
    constexpr int N = PARTS<T>, MOST = N == 1 ? 0 : 2, KS = DK / 32;
    __shared__ float m[C * MP], tt[C * MP];  // M; T transposed
    __shared__ float xs[3][16 * XP];
    __shared__ double total[C];
    __shared__ float betas[C];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c16 = lane & 15;
    const int64_t unit = blockIdx.x / static_cast<unsigned>(a.chunks);
    const int chunk = blockIdx.x % static_cast<unsigned>(a.chunks), b = static_cast<int>(unit / a.Hv), h = static_cast<int>(unit % a.Hv);
    const int t0 = chunk * C, n = min(C, a.T - t0);
    const int64_t place = unit * a.chunks + chunk;
    const int hk = h / (a.Hv / a.Hk);
    const T *q = head<const T>(a.q, b, hk) + static_cast<int64_t>(t0) * a.q.st, *k = head<const T>(a.k, b, hk) + static_cast<int64_t>(t0) * a.k.st;
    uint16_t *attn = a.attn + place * 3 * (BLOCKS * BLOCK), *attn_t = BACKWARD ? a.attn_t + place * 3 * (BLOCKS * BLOCK) : nullptr;
    // wavefront w: rows 16w .. 16w+15 of both products, so the first one, with one tile of them, has time for the sum of the log-decays
    const int it = wave, i = 16 * it + c16;
    Eight<BY, T> ki[KS], qi[KS], kj[3][KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        ki[s].load(k, a.k.st, min(i, n - 1), 32 * s + 8 * g, a.dk), qi[s].load(q, a.q.st, min(i, n - 1), 32 * s + 8 * g, a.dk);
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < it) kj[j][s].load(k, a.k.st, min(16 * j + c16, n - 1), 32 * s + 8 * g, a.dk);
    }
    if (wave == 0) {
        const int64_t at = (static_cast<int64_t>(b) * a.T + t0 + min(lane, n - 1)) * a.Hv + h;
        double sum = lane < n ? held(a.g[at]) : 0.0;
        const float beta = lane < n ? a.beta[at] : 0.0f;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double up = __shfl_up(sum, o);
            if (lane >= o) sum += up;
        }
        float* scalars = a.scalars + place * 3 * C;
        total[lane] = sum, betas[lane] = beta;
        scalars[lane] = decay_of(sum), scalars[C + lane] = decay_of(__shfl(sum, 63) - sum), scalars[2 * C + lane] = beta;
    }
    f32x4 kk[4] = {}, qk[4] = {};  // rows j, column i; transposed, qk: rows i, column j
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j <= it) {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const Operand<N> x = j < 3 && j < it ? kj[j < 3 ? j : 0][s].operand() : ki[s].operand(), y = qi[s].operand();
                product<MOST>(x, ki[s].operand(), kk[j]);
                if (BACKWARD)
                    product<MOST>(y, x, qk[j]);
                else
                    product<MOST>(x, y, qk[j]);
            }
        }
    __syncthreads();
    {
        const float beta = betas[i];
        const double own = total[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int j4 = 16 * j + 4 * g;
            if (j <= it) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float d = j4 + r <= i ? decay_of(own - total[j4 + r]) : 0.0f;
                    kk[j][r] = j4 + r < i ? beta * d * kk[j][r] : 0.0f;
                    if (BACKWARD) {
                        const int row = 16 * it + 4 * g + r, col = 16 * j + c16;
                        qk[j][r] = col <= row ? a.scale * decay_of(total[row] - total[col]) * qk[j][r] : 0.0f;
                    } else {
                        qk[j][r] = j4 + r <= i ? a.scale * d * qk[j][r] : 0.0f;
                    }
                }
                *reinterpret_cast<f32x4*>(m + i * MP + j4) = kk[j];
            }
            if (j <= it || (j & 1)) {  // a tile of zeros completes a block
                if (BACKWARD && (j <= it || j == it + 1))
                    put_block4<3, true>(attn_t, 16 * j + c16, 16 * it + 4 * g, qk[j]);
                else if (!BACKWARD && (j <= it || j == it + 1))
                    put_block4<3, false>(attn, i, j4, qk[j]);
            }
        }
    }
    __syncthreads();
    {
        const float* block = m + 16 * wave * MP + 16 * wave;
        f32x4 row[16][4];
        float t[16];
        const auto read = [&](auto from, auto to) {  // rows one behind the other would each be waited for
#pragma unroll
            for (int i = decltype(from)::value; i < decltype(to)::value; ++i)
#pragma unroll
                for (int j = 0; j < i; j += 4) row[i][j / 4] = *reinterpret_cast<const f32x4*>(block + i * MP + j);
            __builtin_amdgcn_sched_barrier(0);
        };
        const auto solve = [&](auto from, auto to) {
#pragma unroll
            for (int i = decltype(from)::value; i < decltype(to)::value; ++i) {
                float s[2] = {i == c16 ? 1.0f : 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < i; ++j) s[j & 1] = fmaf(-row[i][j / 4][j & 3], t[j], s[j & 1]);
                t[i] = s[0] + s[1];
            }
        };
        using std::integral_constant;
        read(integral_constant<int, 1>{}, integral_constant<int, 9>{});
        solve(integral_constant<int, 0>{}, integral_constant<int, 5>{});
        read(integral_constant<int, 9>{}, integral_constant<int, 13>{});
        solve(integral_constant<int, 5>{}, integral_constant<int, 9>{});
        read(integral_constant<int, 13>{}, integral_constant<int, 16>{});
        solve(integral_constant<int, 9>{}, integral_constant<int, 16>{});
        if (g == 0) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) *reinterpret_cast<f32x4*>(tt + (16 * wave + c16) * MP + 16 * wave + i) = f32x4{t[i], t[i + 1], t[i + 2], t[i + 3]};
        }
    }
    __syncthreads();
    const Operand<3> zeros = split8<3>(f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0});
    const auto eight = [](const float* p) { return split8<3>(*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 4)); };
    const auto down = [](const float* p) { return split8<3>(f32x4{p[0], p[MP], p[2 * MP], p[3 * MP]}, f32x4{p[4 * MP], p[5 * MP], p[6 * MP], p[7 * MP]}); };
#pragma unroll
    for (int d = 1; d < 4; ++d) {
        if (wave >= d) {
            const int it = wave, jt = wave - d;
            f32x4 sums[3] = {};
#pragma unroll
            for (int k0 = 0; k0 < 16 * d; k0 += 32) {
                const bool in = k0 + 8 * g < 16 * d;  // half of the last step's values of k may be past the sum
                const int at = 16 * jt + (in ? k0 + 8 * g : 0);
                const Operand<3> x = eight(m + (16 * it + c16) * MP + at), y = eight(tt + (16 * jt + c16) * MP + at);
                spread<2>(in ? x : zeros, in ? y : zeros, sums);
            }
            float* mine = xs[wave - 1];
            *reinterpret_cast<f32x4*>(mine + c16 * XP + 4 * g) = gather(sums);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_wave_barrier();
            f32x4 more[3] = {};
            const int at = g < 2 ? 8 * g : 0;
            const Operand<3> x = down(tt + (16 * it + at) * MP + 16 * it + c16), y = eight(mine + c16 * XP + at);
            spread<2>(g < 2 ? x : zeros, g < 2 ? y : zeros, more);
            *reinterpret_cast<f32x4*>(tt + (16 * jt + c16) * MP + 16 * it + 4 * g) = -gather(more);
        }
        __syncthreads();
    }
    // T, and transposed, a block to a wavefront at a time; what lies past the diagonal's blocks is zero
    uint16_t* out = a.inverse + place * 3 * (BLOCKS * BLOCK);
    for (int e = wave; e < BLOCKS; e += 4) {
        const int it = e < 2 ? e : e < 4 ? 2 : 3, kk = e < 2 ? 0 : (e & 1);
        const bool in = 2 * kk + (g >> 1) <= it;
        const Operand<3> o = down(tt + (in ? 32 * kk + 8 * g : 0) * MP + 16 * it + c16);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(out + (p * BLOCKS + e) * BLOCK + 8 * lane) = in ? o.part[p] : zeros.part[p];
    }
    if (!BACKWARD) return;
    out = a.inverse_t + place * 3 * (BLOCKS * BLOCK);
    for (int e = wave ^ 2; e < BLOCKS; e += 4) {
        const int it = e < 4 ? e / 2 : e - 2, kk = e < 4 ? (e & 1) : 1;
        const bool in = 2 * kk + (g >> 1) >= it;
        const Operand<3> o = eight(tt + (16 * it + c16) * MP + (in ? 32 * kk + 8 * g : 16 * it));
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(out + (p * BLOCKS + e) * BLOCK + 8 * lane) = in ? o.part[p] : zeros.part[p];
    }
}
static_assert(block_of<false>(1, 0) == 1 && block_of<false>(2, 0) == 2 && block_of<false>(2, 1) == 3 && block_of<false>(3, 0) == 4 && block_of<false>(3, 1) == 5, "the order that T is written in");
static_assert(block_of<true>(0, 1) == 1 && block_of<true>(1, 0) == 2 && block_of<true>(1, 1) == 3 && block_of<true>(2, 1) == 5 - 1 && block_of<true>(3, 1) == 5, "and transposed");

// ---- the walk down the chunks ----
// Four wavefronts for each 16 columns: one has 16 of a chunk's tokens, and of the state a quarter of its rows.
// Everything that a chunk needs from memory is asked for a chunk ahead, each as soon as the registers that hold the one before are free.
// STATES: for the backward, the states and U go to memory and there is no O.
template <typename T, int DK>
constexpr bool TWO_K = PARTS<T> == 1 || DK < 128;  // two of K's tiles in LDS: the next one is written while this one is still read

template <typename T, int DK, int VB, bool STATES, Rows BY>
__global__ __launch_bounds__(16 * VB) void walk(Rule a) {
    constexpr int N = PARTS<T>, KP = DK + 16, SP = DK + 8, KS = DK / 32, KT = (DK + 63) / 64;
    extern __shared__ uint16_t lds[];
    uint16_t *kt = lds, *st = kt + (TWO_K<T, DK> ? 2 : 1) * N * C * KP, *rt = st + 3 * VB * SP, *dt = rt + 3 * VB * CP, *ut = dt + 3 * VB * CP;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c16 = lane & 15;
    int unit, blk;
    if (!unit_of(blockIdx.x, a.B * a.Hv, (a.dv + VB - 1) / VB, unit, blk)) return;
    const int b = unit / a.Hv, h = unit - b * a.Hv, hk = h / (a.Hv / a.Hk);
    const int tile = wave >> (VB / 32), vt = VB == 32 ? 16 * (wave & 1) : 0;
    const int column = vt + c16, vc = VB * blk + column, tokens = 16 * tile + 4 * g;  // the state's column and the four tokens of this lane,
    const int token = 16 * tile + c16, vo = VB * blk + vt + 4 * g;                     // of O the token and the four columns
    const bool low = tile < 2;                         // rows of T and A with nothing past their first 32 columns
    const bool rows_here = DK > 32 || tile < DK / 16;  // a state of 32 rows is two tiles
    const T *q = head<const T>(a.q, b, hk), *k = head<const T>(a.k, b, hk), *v = head<const T>(a.v, b, h);
    T* out = STATES ? nullptr : head<T>(a.o, b, h);
    const int64_t state_at = static_cast<int64_t>(unit) * a.dk * a.dv + vc, first = static_cast<int64_t>(unit) * a.chunks;
    const auto row_of = [&](int i) { return 16 * (tile * KT + i) + 4 * g; };
    // this lane's part of a state in memory
    const auto each_row = [&](auto&& f) {
        if (!rows_here || vc >= a.dv) return;
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (row_of(i) + r < a.dk) f(i, r, static_cast<int64_t>(row_of(i) + r) * a.dv);
    };
    f32x4 S[KT] = {};
    if (a.state_in) each_row([&](int i, int r, int64_t at) { S[i][r] = a.state_in[state_at + at]; });
    Tile<BY, T, DK, 16 * VB> K;
    Eight<BY, T> Q[KS];
    Tokens<BY, T> V;
    Operand<3> inverse[2];
    Operand<3> attn[2];
    f32x4 gamma, delta, beta;
    float whole, gamma_o;
    const auto load_k = [&](int chunk) { K.load(k + static_cast<int64_t>(chunk) * C * a.k.st, a.k.st, min(C, a.T - chunk * C), a.dk); };
    const auto load_rows = [&](int chunk) {
        const int n = min(C, a.T - chunk * C);
        const float* d = a.scalars + (first + chunk) * 3 * C;
        gamma = *reinterpret_cast<const f32x4*>(d + tokens), delta = *reinterpret_cast<const f32x4*>(d + C + tokens), beta = *reinterpret_cast<const f32x4*>(d + 2 * C + tokens);
        whole = d[C - 1];
        V.load(v + static_cast<int64_t>(chunk) * C * a.v.st, a.v.st, tokens, n, vc, a.dv);
        if (!STATES) {
            gamma_o = d[token];
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) Q[kk].load(q + static_cast<int64_t>(chunk) * C * a.q.st, a.q.st, min(token, n - 1), 32 * kk + 8 * g, a.dk);
        }
    };
    const auto load_inverse = [&](int chunk) {
        const uint16_t* m = a.inverse + (first + chunk) * 3 * (BLOCKS * BLOCK);
        inverse[0] = matrix_block<3, false>(m, tile, 0, lane);
        if (!low) inverse[1] = matrix_block<3, false>(m, tile, 1, lane);
    };
    const auto load_attn = [&](int chunk) {
        const uint16_t* m = a.attn + (first + chunk) * 3 * (BLOCKS * BLOCK);
        attn[0] = matrix_block<3, false>(m, tile, 0, lane);
        if (!low) attn[1] = matrix_block<3, false>(m, tile, 1, lane);
    };
    load_k(0), load_rows(0), load_inverse(0);
    if (!STATES) load_attn(0);
    for (int chunk = 0; chunk < a.chunks; ++chunk) {
        const int t0 = chunk * C, n = min(C, a.T - t0), next = min(chunk + 1, a.chunks - 1);
        const int64_t place = first + chunk;
        uint16_t* kc = kt + (TWO_K<T, DK> ? (chunk & 1) * N * C * KP : 0);
        if (!TWO_K<T, DK> && chunk > 0) __syncthreads();
        K.template to_lds<KP>(kc);
        if (rows_here) {
#pragma unroll
            for (int i = 0; i < KT; ++i) put4<3, VB, SP>(st, column, row_of(i), S[i]);
        }
        if (STATES) {
            float* to = a.states + place * a.dk * a.dv + vc;
            each_row([&](int i, int r, int64_t at) { to[at] = S[i][r]; });
        }
        __syncthreads();
        load_k(next);
        // R = beta (V - gamma K S), and gamma Q S
        f32x4 O = {0, 0, 0, 0};
        {
            f32x4 P[3] = {}, QS[3] = {};
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                const Operand<3> s = rows_of<3, VB, SP>(st, vt, 32 * kk, lane);
                spread<2>(rows_of<N, C, KP>(kc, 16 * tile, 32 * kk, lane), s, P);
                if (!STATES) spread<2>(s, Q[kk].operand(), QS);
            }
            const f32x4 x = V.values(), p = gather(P);
            f32x4 R;
#pragma unroll
            for (int r = 0; r < 4; ++r) R[r] = beta[r] * fmaf(-gamma[r], p[r], x[r]);
            put4<3, VB, CP>(rt, column, tokens, R);
            if (!STATES) O = gather(QS) * (a.scale * gamma_o);
        }
        const f32x4 leave = delta;
        const float end = whole;
        __syncthreads();
        load_rows(next);
        // U = T R
        {
            f32x4 sums[3] = {};
            spread<2>(inverse[0], rows_of<3, VB, CP>(rt, vt, 0, lane), sums);
            if (!low) spread<2>(inverse[1], rows_of<3, VB, CP>(rt, vt, 32, lane), sums);
            const f32x4 U = gather(sums);
            if (STATES) {
                if (vc < a.dv)
#pragma unroll
                    for (int r = 0; r < 4; ++r) a.puts[(place * C + tokens + r) * a.dv + vc] = U[r];
            } else {
                put4<3, VB, CP>(ut, column, tokens, U);
            }
            put4<3, VB, CP>(dt, column, tokens, U * leave);
        }
        __syncthreads();
        load_inverse(next);
        // S = gamma S + K^T (delta U), O += A U
        if (rows_here) {
            f32x4 sums[KT][3] = {};
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const Operand<3> u = rows_of<3, VB, CP>(dt, vt, 32 * kk, lane);
#pragma unroll
                for (int i = 0; i < KT; ++i) spread<2>(cols_of<N, C, KP>(kc, 32 * kk, 16 * (tile * KT + i), lane), u, sums[i]);
            }
#pragma unroll
            for (int i = 0; i < KT; ++i) S[i] = S[i] * end + gather(sums[i]);
        }
        if (!STATES) {
            f32x4 sums[3] = {};
            spread<2>(rows_of<3, VB, CP>(ut, vt, 0, lane), attn[0], sums);
            if (!low) spread<2>(rows_of<3, VB, CP>(ut, vt, 32, lane), attn[1], sums);
            if (token < n) write4<BY>(out + static_cast<int64_t>(t0 + token) * a.o.st, vo, a.dv, O + gather(sums));
            load_attn(next);
        }
    }
    if (a.state_out) each_row([&](int i, int r, int64_t at) { a.state_out[state_at + at] = S[i][r]; });
}
template <typename T, int DK, int VB, bool STATES>
constexpr size_t walk_lds() {
    return sizeof(uint16_t) * ((TWO_K<T, DK> ? 2 : 1) * PARTS<T> * C * (DK + 16) + 3 * VB * (DK + 8) + (STATES ? 6 : 9) * VB * CP);
}

// ---- token by token ----
// A workgroup for CB columns of a head's state, four of them and every RG-th row to a thread. Both products of a token with the decayed state, S^T k and S^T q, are formed in one walk
// over the rows and added up in one exchange: o = scale (e^g S^T q + (q.k) u).
constexpr int STEP_NT = 256;
template <typename T, int CB, int RPT>
__global__ __launch_bounds__(STEP_NT) void steps(Rule a) {
    constexpr int QUADS = CB / 4, RG = STEP_NT / QUADS, WG = 64 / QUADS, WAVES = STEP_NT / 64;
    __shared__ f32x4 sums[2][2][WAVES][QUADS];
    __shared__ float dots[2][WAVES];
    const int tid = threadIdx.x, wave = tid >> 6, quad = tid % QUADS, rg = tid / QUADS;
    const int nblk = (a.dv + CB - 1) / CB, unit = quotient(blockIdx.x, nblk), blk = blockIdx.x - unit * nblk;
    const int b = quotient(unit, a.Hv), h = unit - b * a.Hv, hk = quotient(h, a.Hv / a.Hk), c = CB * blk + 4 * quad;
    const T *q = head<const T>(a.q, b, hk), *k = head<const T>(a.k, b, hk), *v = head<const T>(a.v, b, h);
    T* out = head<T>(a.o, b, h);
    const int64_t state_at = static_cast<int64_t>(unit) * a.dk * a.dv;
    f32x4 S[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int r = rg + i * RG;
        S[i] = a.state_in && r < a.dk ? load4(a.state_in + state_at + static_cast<int64_t>(r) * a.dv, c, a.dv) : f32x4{0, 0, 0, 0};
    }
    for (int t = 0; t < a.T; ++t) {
        float kr[RPT], qr[RPT];
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int r = rg + i * RG;
            kr[i] = r < a.dk ? elem(k, t * a.k.st + r) : 0.0f, qr[i] = r < a.dk ? elem(q, t * a.q.st + r) : 0.0f;
        }
        const int64_t at = (static_cast<int64_t>(b) * a.T + t) * a.Hv + h;
        const float decay = decay_of(held(a.g[at])), beta = a.beta[at];
        const f32x4 x = load4(v + t * a.v.st, c, a.dv);
        f32x4 sk = {0, 0, 0, 0}, sq = sk;
        float qk = 0.0f;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            S[i] *= decay;
#pragma unroll
            for (int e = 0; e < 4; ++e) sk[e] = fmaf(S[i][e], kr[i], sk[e]), sq[e] = fmaf(S[i][e], qr[i], sq[e]);
            qk = fmaf(qr[i], kr[i], qk);
        }
#pragma unroll
        for (int o = QUADS; o < 64; o <<= 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sk[e] += __shfl_xor(sk[e], o), sq[e] += __shfl_xor(sq[e], o);
            qk += __shfl_xor(qk, o);
        }
        const int turn = t & 1;  // the sums of the token before may still be read
        if ((tid & 63) < QUADS) sums[turn][0][wave][quad] = sk, sums[turn][1][wave][quad] = sq;
        if ((tid & 63) == 0) dots[turn][wave] = qk;
        __syncthreads();
        sk = sums[turn][0][0][quad], sq = sums[turn][1][0][quad], qk = dots[turn][0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) sk += sums[turn][0][w][quad], sq += sums[turn][1][w][quad], qk += dots[turn][w];
        f32x4 u;
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = beta * (x[e] - sk[e]);
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[i][e] = fmaf(kr[i], u[e], S[i][e]);
        if (rg == 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sq[e] = a.scale * fmaf(qk, u[e], sq[e]);
            store4(out + t * a.o.st, c, a.dv, sq);
        }
    }
    if (!a.state_out) return;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int r = rg + i * RG;
        if (r < a.dk) store4(a.state_out + state_at + static_cast<int64_t>(r) * a.dv, c, a.dv, S[i]);
    }
}

// ---- launches ----

// Up to here a sequence is walked through token by token. A chunk takes what 7 tokens take (8 heads of 128 of one sequence in bf16: 15.7 us for 8 tokens by tokens, 13.5 by chunks) to 17 and more
// (256 sequences of 16 heads in fp32): 8 tokens of 32 sequences of 16 heads by tokens and by chunks in bf16 56 and 58 us at 128, 20 and 30 at 64, 12 and 21 at 32; in fp32 37 and 79, 18 and 38,
// 11 and 22; 16 tokens in bf16 100 and 58, 34 and 31, 21 and 21, in fp32 62 and 81, 32 and 38, 19 and 22; of 256 sequences at 128 345 and 446, in fp32 217 and 620.
constexpr int FEW_TOKENS = 8;
template <typename T, int DK, int VB, bool STATES, Rows BY>
int launch_walk(const Rule& a, hipStream_t st) {
    constexpr size_t lds = walk_lds<T, DK, VB, STATES>();
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    PK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(walk<T, DK, VB, STATES, BY>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
    walk<T, DK, VB, STATES, BY><<<unit_grid(static_cast<int64_t>(a.B) * a.Hv, blocks(a.dv, VB)), 16 * VB, lds, st>>>(a);
    return launched();
}
template <typename T, bool STATES>
int launch_walk(const Rule& a, hipStream_t st) {
    return by_size(a.dk, [&](auto dk) {
        constexpr int DK = decltype(dk)::value;
        if (wide(a)) return by_rows(rows_by(a, DK, 32), [&](auto by) { return launch_walk<T, DK, 32, STATES, decltype(by)::value>(a, st); });
        return by_rows(rows_by(a, DK, 16), [&](auto by) { return launch_walk<T, DK, 16, STATES, decltype(by)::value>(a, st); });
    });
}
template <typename T>
int launch_matrices(const Rule& a, bool backward, hipStream_t st) {
    return by_size(a.dk, [&](auto dk) {
        constexpr int DK = decltype(dk)::value;
        const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.B) * a.Hv * a.chunks));
        return by_rows(rows_by(a, DK, 1), [&](auto by) {
            constexpr Rows BY = decltype(by)::value;
            backward ? chunk_matrices<T, DK, true, BY><<<grid, 256, 0, st>>>(a) : chunk_matrices<T, DK, false, BY><<<grid, 256, 0, st>>>(a);
            return launched();
        });
    });
}
template <typename T>
void launch_steps(const Rule& a, hipStream_t st) {
    constexpr int CB = 32;
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(a.B) * a.Hv * ((a.dv + CB - 1) / CB)));
    if (a.dk <= 32) return steps<T, CB, 1><<<grid, STEP_NT, 0, st>>>(a);
    if (a.dk <= 64) return steps<T, CB, 2><<<grid, STEP_NT, 0, st>>>(a);
    steps<T, CB, 4><<<grid, STEP_NT, 0, st>>>(a);
}

struct Room {
    size_t inverse, attn, scalars, all;
};
Room room_of(const pk_delta_shape* s) {
    const size_t places = static_cast<size_t>(s->B) * s->Hv * chunks(s->T);
    Room r;
    r.inverse = r.attn = pad(places * 3 * MATRIX), r.scalars = pad(places * 3 * C * sizeof(float));
    r.all = r.inverse + r.attn + r.scalars;
    return r;
}

}  // namespace

int launch_chunks(const Rule& a, int dtype, bool backward, hipStream_t st) {
    return dtype == PK_BF16 ? launch_matrices<uint16_t>(a, backward, st) : launch_matrices<float>(a, backward, st);
}
int launch_states(const Rule& a, int dtype, hipStream_t st) { return dtype == PK_BF16 ? launch_walk<uint16_t, true>(a, st) : launch_walk<float, true>(a, st); }

int check(const char* who, const pk_delta_shape* s) {
    const std::string w(who);
    if (!s) return fail(PK_ERR_ARGUMENT, w + ": null pointer");
    if (s->B < 0 || s->T < 0 || s->Hk < 1 || s->Hv < 1 || s->Hv % s->Hk) return fail(PK_ERR_SHAPE, w + ": shape mismatch (heads of v are shared out evenly to those of k)");
    if (s->dk < 1 || s->dk > 128 || s->dv < 1 || s->dv > 256) return fail(PK_ERR_SHAPE, w + ": shape mismatch (dk 1 to 128, dv 1 to 256)");
    // a launch has fewer than 2^32 threads: 512 for each chunk, and for each of a head's 8 blocks of columns
    if (static_cast<int64_t>(s->B) * s->Hv > (1 << 19) || s->T > (1 << 26) || static_cast<int64_t>(s->B) * s->Hv * (chunks(s->T) + 1) > (1 << 22))
        return fail(PK_ERR_SHAPE, w + ": shape mismatch (at most 2^19 heads of sequences and 2^22 chunks of 64 tokens)");
    if (!known_dtype(s->dtype)) return fail(PK_ERR_ARGUMENT, w + ": dtype must be PK_F32 or PK_BF16");
    if (!std::isfinite(s->scale)) return fail(PK_ERR_ARGUMENT, w + ": scale must be finite");
    return PK_OK;
}
bool view_of(const pk_tensor4* t, View& v) {
    if (!t || !t->ptr) return false;
    v = View{t->ptr, t->stride_b, t->stride_t, t->stride_h};
    return true;
}
Span span_of(const void* dense, size_t bytes) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(dense);
    return Span{p, dense ? p + bytes : p, false, false};
}
Span span_of(const View& v, const pk_delta_shape* s, int heads, int width) {
    if (!v.ptr || !s->B || !s->T) return Span{0, 0, true, true};
    int64_t low = 0, high = width;
    for (const int64_t reach : {(s->B - 1) * v.sb, (s->T - 1) * v.st, (heads - 1) * v.sh}) (reach < 0 ? low : high) += reach;
    const uintptr_t p = reinterpret_cast<uintptr_t>(v.ptr);
    const int64_t es = elem_size(s->dtype);
    return Span{p + static_cast<uintptr_t>(low * es), p + static_cast<uintptr_t>(high * es), true, high - low > static_cast<int64_t>(s->B) * s->T * heads * width};
}
bool apart(std::initializer_list<Span> written, std::initializer_list<Span> read) {
    const auto clash = [](const Span& x, const Span& y) {
        if (x.from == x.to || y.from == y.to) return false;
        return x.heads && y.heads && (x.gaps || y.gaps) ? x.from == y.from : x.from < y.to && y.from < x.to;
    };
    for (const Span* w = written.begin(); w != written.end(); ++w) {
        for (const Span& r : read)
            if (clash(*w, r)) return false;
        for (const Span* o = written.begin(); o != w; ++o)
            if (clash(*w, *o)) return false;
    }
    return true;
}
bool shares(const View& v, const pk_delta_shape* s, int heads) { return v.ptr && ((s->B > 1 && !v.sb) || (s->T > 1 && !v.st) || (heads > 1 && !v.sh)); }

}  // namespace delta
}  // namespace pk

using namespace pk;
using namespace pk::delta;

extern "C" {

size_t pk_delta_rule_fwd_workspace_bytes(const pk_delta_shape* s) {
    if (delta::check("pk_delta_rule_fwd", s) != PK_OK || s->T <= FEW_TOKENS) return 0;
    return room_of(s).all;
}

int pk_delta_rule_fwd(const pk_delta_shape* s, const pk_tensor4* q, const pk_tensor4* k, const pk_tensor4* v, const float* g, const float* beta, const float* state_in,
                      const pk_tensor4* o, float* state_out, void* workspace, size_t workspace_bytes, void* stream) {
    return c_entry([&] {
        const std::string who = "pk_delta_rule_fwd";
        if (int rc = delta::check(who.c_str(), s)) return rc;
        Rule a{};
        const bool tokens = static_cast<int64_t>(s->B) * s->T > 0;
        if (s->B == 0) return static_cast<int>(PK_OK);
        if (tokens && (!view_of(q, a.q) || !view_of(k, a.k) || !view_of(v, a.v) || !view_of(o, a.o) || !g || !beta)) return fail(PK_ERR_ARGUMENT, who + ": null pointer");
        const size_t need = pk_delta_rule_fwd_workspace_bytes(s);
        if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
            return fail(PK_ERR_WORKSPACE, who + ": workspace too small (pk_delta_rule_fwd_workspace_bytes)");
        if (shares(a.o, s, s->Hv)) return fail(PK_ERR_ARGUMENT, who + ": elements of o share memory");
        const size_t gates = sizeof(float) * s->B * s->T * s->Hv, state = sizeof(float) * s->B * s->Hv * s->dk * s->dv;
        if (!apart({span_of(a.o, s, s->Hv, s->dv), span_of(state_out, state), span_of(workspace, need)},
                   {span_of(a.q, s, s->Hk, s->dk), span_of(a.k, s, s->Hk, s->dk), span_of(a.v, s, s->Hv, s->dv), span_of(g, gates), span_of(beta, gates),
                    span_of(state_in == state_out ? nullptr : state_in, state)}))
            return fail(PK_ERR_ARGUMENT, who + ": results lie clear of one another, of the workspace and of what is read (state_out may be state_in)");
        touch({a.q.ptr, a.k.ptr, a.v.ptr, g, beta, state_in, a.o.ptr, state_out, workspace}, stream);
        hipStream_t st = static_cast<hipStream_t>(stream);
        a.g = g, a.beta = beta, a.state_in = state_in, a.state_out = state_out;
        a.B = s->B, a.T = s->T, a.Hk = s->Hk, a.Hv = s->Hv, a.dk = s->dk, a.dv = s->dv, a.chunks = chunks(s->T), a.scale = s->scale;
        if (s->T <= FEW_TOKENS) {
            if (s->T == 0 && (!state_out || state_out == state_in)) return static_cast<int>(PK_OK);
            s->dtype == PK_BF16 ? launch_steps<uint16_t>(a, st) : launch_steps<float>(a, st);
            return launched();
        }
        const Room r = room_of(s);
        char* ws = static_cast<char*>(workspace);
        a.inverse = reinterpret_cast<uint16_t*>(ws), a.attn = reinterpret_cast<uint16_t*>(ws + r.inverse), a.scalars = reinterpret_cast<float*>(ws + r.inverse + r.attn);
        if (int rc = launch_chunks(a, s->dtype, false, st)) return rc;
        return s->dtype == PK_BF16 ? launch_walk<uint16_t, false>(a, st) : launch_walk<float, false>(a, st);
    });
}

}  // extern "C"
