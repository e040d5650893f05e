// Gated delta rule, backward. With the names of delta_rule.h, dS' the gradient of the state that a chunk leaves:
//
//   dU = A^T dO + delta K dS'     dR = T^T dU     dV = beta dR     dS = gamma_63 dS' + (scale gamma Q)^T dO - (beta gamma K)^T dR
//   with X = dO U^T, Z = dR U^T (64 x 64), E_ij = scale D_ij X_ij (j <= i), F_ij = -beta_i D_ij Z_ij (j < i), Y = dO S^T, Yr = dR S^T, Yu = U dS'^T (64 x dk):
//   dQ = scale gamma Y + E K     dK = delta Yu - beta gamma Yr + E^T Q + (F + F^T) K
//   dbeta_i = dR_i.V_i - gamma_i k_i.Yr_i - sum_j D_ij Z_ij k_i.k_j
//   dG_i = scale gamma_i q_i.Y_i - beta_i gamma_i k_i.Yr_i - delta_i k_i.Yu_i + sum_j H_ij - sum_j H_ji,  H = E (q.k) + F (k.k) below the diagonal; at the chunk's end what S'
//   gives through gamma and delta as well, sum_i delta_i k_i.Yu_i + gamma_63 <S, dS'>;  dg_t = the sum of dG from t on
// In that sum every H_ij of two tokens on one side of t is there once with either sign, and so are the terms of delta: added up in 64 bits from the same values they go out exactly, and
// what is left is as exact as its own terms: a token behind a decay of e^-40 has its dg to 1e-16 of the others' and not to 1e-7.
//
// Four launches: the chunks' matrices; the states that the chunks begin with, formed again by the forward's walk (only the inputs are kept between the passes); the walk back, which like the
// forward's takes 16 or 32 columns of a state by themselves; then, a workgroup for a chunk and a head of k, all that needs every column of a state. 4 x 4096 tokens, 16 heads of 128 in
// bf16: 89, 203, 323 and 411 us. The walks are bound by their own chain, 3.2 and 5.0 us a chunk; the last launch by the states of all chunks (0.8 GB, 0.16 ms of a copy's rate), since a CU
// has one workgroup's loads under way at a time: its wavefronts have tokens, so both states go through LDS, in three parts beside K and Q, and fill it.
#include "delta_rule.h"

namespace pk {
namespace delta {
namespace {

__device__ inline float decay_of(double x) { return __builtin_amdgcn_exp2f(static_cast<float>(x * 1.4426950408889634074)); }
constexpr float LEAST = -1000.0f;  // a log-decay below it is held to it, and has no derivative

// ---- the walk back ----
// As the forward's: four wavefronts for each 16 columns, loads a chunk ahead.
template <int DK>
constexpr bool TWO_K = DK < 128;  // a second tile of K in LDS would leave room for one workgroup on a CU in place of two
template <typename T, int DK, int VB>
constexpr size_t back_lds() {
    return sizeof(uint16_t) * ((TWO_K<DK> ? 3 : 2) * PARTS<T> * C * (DK + 16) + 3 * VB * (DK + 8) + (9 + PARTS<T>) * VB * CP);
}
template <typename T, int DK, int VB, Rows BY>
__global__ __launch_bounds__(16 * VB) void walk_back(Rule a) {
    constexpr int N = PARTS<T>, KP = DK + 16, SP = DK + 8, KS = DK / 32, KT = (DK + 63) / 64;
    extern __shared__ uint16_t lds[];
    uint16_t *kt = lds, *qt = kt + (TWO_K<DK> ? 2 : 1) * N * C * KP, *st = qt + N * C * KP, *ut = st + 3 * VB * SP, *wt = ut + 3 * VB * CP, *dt = wt + 3 * VB * CP, *rt = dt + 3 * VB * CP;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c16 = lane & 15;
    int unit, blk;
    if (!unit_of(blockIdx.x, a.B * a.Hv, (a.dv + VB - 1) / VB, unit, blk)) return;
    const int b = unit / a.Hv, h = unit - b * a.Hv, hk = h / (a.Hv / a.Hk);
    const int tile = wave >> (VB / 32), vt = VB == 32 ? 16 * (wave & 1) : 0;
    const int column = vt + c16, vc = VB * blk + column, tokens = 16 * tile + 4 * g;
    const bool high = tile >= 2;  // rows of the transposed matrices with nothing in their first 32 columns
    const bool rows_here = DK > 32 || tile < DK / 16, in = vc < a.dv;
    const T *q = head<const T>(a.q, b, hk), *k = head<const T>(a.k, b, hk), *dout = head<const T>(a.dout, b, h);
    T* dv = head<T>(a.dv_, b, h) + vc;
    const int64_t state_at = static_cast<int64_t>(unit) * a.dk * a.dv + vc, first = static_cast<int64_t>(unit) * a.chunks;
    const auto row_of = [&](int i) { return 16 * (tile * KT + i) + 4 * g; };
    const auto each_row = [&](auto&& f) {
        if (!rows_here || !in) return;
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (row_of(i) + r < a.dk) f(i, r, static_cast<int64_t>(row_of(i) + r) * a.dv);
    };
    f32x4 S[KT] = {};  // of the gradient of the state
    if (a.dstate_out) each_row([&](int i, int r, int64_t at) { S[i][r] = a.dstate_out[state_at + at]; });
    Tile<BY, T, DK, 16 * VB> K, Q;
    Tokens<BY, T> D;
    Operand<3> attn_t[2], inverse_t[2];
    f32x4 gamma, delta, beta;
    float whole;
    const auto load_k = [&](int chunk) { K.load(k + static_cast<int64_t>(chunk) * C * a.k.st, a.k.st, min(C, a.T - chunk * C), a.dk); };
    const auto load_q = [&](int chunk) { Q.load(q + static_cast<int64_t>(chunk) * C * a.q.st, a.q.st, min(C, a.T - chunk * C), a.dk); };
    const auto load_rows = [&](int chunk) {
        const float* d = a.scalars + (first + chunk) * 3 * C;
        gamma = *reinterpret_cast<const f32x4*>(d + tokens), delta = *reinterpret_cast<const f32x4*>(d + C + tokens), beta = *reinterpret_cast<const f32x4*>(d + 2 * C + tokens);
        whole = d[C - 1];
        D.load(dout + static_cast<int64_t>(chunk) * C * a.dout.st, a.dout.st, tokens, min(C, a.T - chunk * C), vc, a.dv);
    };
    const auto load_matrix = [&](const uint16_t* all, int chunk, Operand<3>(&o)[2]) {
        const uint16_t* m = all + (first + chunk) * 3 * (BLOCKS * BLOCK);
        if (!high) o[0] = matrix_block<3, true>(m, tile, 0, lane);
        o[1] = matrix_block<3, true>(m, tile, 1, lane);
    };
    if (a.chunks > 0) load_k(a.chunks - 1), load_rows(a.chunks - 1), load_matrix(a.attn_t, a.chunks - 1, attn_t), load_q(a.chunks - 1), load_matrix(a.inverse_t, a.chunks - 1, inverse_t);
    for (int chunk = a.chunks - 1; chunk >= 0; --chunk) {
        const int t0 = chunk * C, n = min(C, a.T - t0), next = max(chunk - 1, 0);
        const int64_t place = first + chunk;
        uint16_t* kc = kt + (TWO_K<DK> ? (chunk & 1) * N * C * KP : 0);
        if (!TWO_K<DK> && chunk < a.chunks - 1) __syncthreads();
        K.template to_lds<KP>(kc);
        if (rows_here) {
#pragma unroll
            for (int i = 0; i < KT; ++i) put4<3, VB, SP>(st, column, row_of(i), S[i]);
        }
        f32x4 x = D.values();
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = tokens + r < n ? x[r] : 0.0f;
        put4<N, VB, CP>(rt, column, tokens, x);
        {
            float* to = a.dstates + place * a.dk * a.dv + vc;
            each_row([&](int i, int r, int64_t at) { to[at] = S[i][r]; });
        }
        __syncthreads();
        load_k(next);
        // dU = A^T dO + delta K dS'; the scaled dO and Q for the end
        {
            f32x4 X[3] = {}, Y[3] = {};
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) spread<2>(rows_of<N, C, KP>(kc, 16 * tile, 32 * kk, lane), rows_of<3, VB, SP>(st, vt, 32 * kk, lane), X);
            if (!high) spread<2>(attn_t[0], rows_of<N, VB, CP>(rt, vt, 0, lane), Y);
            spread<2>(attn_t[1], rows_of<N, VB, CP>(rt, vt, 32, lane), Y);
            put4<3, VB, CP>(ut, column, tokens, gather(Y) + gather(X) * delta);
            put4<3, VB, CP>(dt, column, tokens, x * gamma * a.scale);
            Q.template to_lds<KP>(qt);
        }
        const f32x4 scale_w = -beta * gamma, step = beta;
        const float end = whole;
        __syncthreads();
        load_rows(next), load_matrix(a.attn_t, next, attn_t), load_q(next);
        // dR = T^T dU
        {
            f32x4 sums[3] = {};
            if (!high) spread<2>(inverse_t[0], rows_of<3, VB, CP>(ut, vt, 0, lane), sums);
            spread<2>(inverse_t[1], rows_of<3, VB, CP>(ut, vt, 32, lane), sums);
            const f32x4 R = gather(sums);
            put4<3, VB, CP>(wt, column, tokens, R * scale_w);
            if (in) {
                float* to = a.dputs + (place * C + tokens) * a.dv + vc;
                T* to_v = dv + static_cast<int64_t>(t0 + tokens) * a.dv_.st;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    to[r * a.dv] = R[r];
                    if (tokens + r < n) put(to_v, r * a.dv_.st, R[r] * step[r]);
                }
            }
        }
        __syncthreads();
        load_matrix(a.inverse_t, next, inverse_t);
        // dS = gamma dS' + (scale gamma Q)^T dO - (beta gamma K)^T dR
        if (rows_here) {
            f32x4 sums[KT][3] = {};
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const Operand<3> w = rows_of<3, VB, CP>(wt, vt, 32 * kk, lane), d = rows_of<3, VB, CP>(dt, vt, 32 * kk, lane);
#pragma unroll
                for (int i = 0; i < KT; ++i) {
                    spread<2>(cols_of<N, C, KP>(kc, 32 * kk, 16 * (tile * KT + i), lane), w, sums[i]);
                    spread<2>(cols_of<N, C, KP>(qt, 32 * kk, 16 * (tile * KT + i), lane), d, sums[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < KT; ++i) S[i] = S[i] * end + gather(sums[i]);
        }
    }
    if (a.dstate_in) each_row([&](int i, int r, int64_t at) { a.dstate_in[state_at + at] = S[i][r]; });
}

// ---- what needs all columns of a state ----
// A workgroup for a chunk of a head of k, its heads of v one after the other. Of its eight wavefronts w and w + 4 have tokens 16w .. 16w+15, a lane one of them; each has half of the
// 64 x dk products' rows, the first one E, the second one F.
constexpr int VQ = GB + 8, AP = C + 8, HP = C + 4, GRAD_NT = 512;  // pitches of rows that are read along k; of H
// K and Q stay in LDS beside what goes by, but for three parts of 128 columns each, which come one after the other when that is done.
template <typename T, int DK>
constexpr bool BESIDE = PARTS<T> == 1 || DK < 128;
template <typename T, int DK>
constexpr int tile_size() {
    return PARTS<T> * C * (DK + 16);
}
template <typename T, int DK>
constexpr size_t grads_lds() {
    constexpr int by = (6 * DK + 3 * C) * VQ, then = 4 * C * HP + 6 * C * AP;
    return sizeof(uint16_t) * (BESIDE<T, DK> ? 2 * tile_size<T, DK>() + std::max(by, then) : std::max(by, tile_size<T, DK>() + then));
}
template <Rows BY, typename T, int DK, int P>
__device__ inline void tile_in(const T* base, int64_t st, int n, int dk, uint16_t* m) {
    Tile<BY, T, DK, GRAD_NT> t;
    t.load(base, st, n, dk);
    t.template to_lds<P>(m);
}
__device__ inline float over_groups(float x) {  // the four lanes of a token
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}
template <typename T, int DK, Rows BY>
__global__ __launch_bounds__(GRAD_NT, 2) void chunk_grads(Rule a, float* sums) {
    constexpr int N = PARTS<T>, MOST = N == 1 ? 0 : 2, KP = DK + 16, KS = DK / 32, KT = DK / 32, SN = (DK * (GB / 4) + GRAD_NT - 1) / GRAD_NT;
    constexpr bool BOTH = BESIDE<T, DK>, AHEAD = BOTH || BY != ANY;  // with everything held the loads ahead of rows of any size would not fit into the registers
    extern __shared__ uint16_t lds[];
    __shared__ double total[C];
    __shared__ double across[8][C];
    __shared__ float ends[2][C], tails[2][C], dbs[2][C], dots[8];
    uint16_t *kt = lds, *qt = BOTH ? kt + tile_size<T, DK>() : kt, *s0 = BOTH ? qt + tile_size<T, DK>() : lds;
    uint16_t *s1 = s0 + 3 * DK * VQ, *ut = s1 + 3 * DK * VQ;                                                          // while the columns of the state go by
    uint16_t *hs = BOTH ? s0 : s0 + tile_size<T, DK>(), *et = hs + 4 * C * HP, *ft = et + 3 * C * AP;  // then
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), tile = wave & 3, half = wave >> 2, g = lane >> 4, c16 = lane & 15, i = 16 * tile + c16;
    float* ht = reinterpret_cast<float*>(hs) + half * C * HP;
    const int64_t group = blockIdx.x / static_cast<unsigned>(a.chunks);
    const int chunk = blockIdx.x % static_cast<unsigned>(a.chunks), b = static_cast<int>(group / a.Hk), hk = static_cast<int>(group % a.Hk), rep = a.Hv / a.Hk;
    const int t0 = chunk * C, n = min(C, a.T - t0), mine_at = min(i, n - 1);  // a token behind the last one reads its row and counts for nothing
    const bool here = i < n;
    const T *q = head<const T>(a.q, b, hk) + static_cast<int64_t>(t0) * a.q.st, *k = head<const T>(a.k, b, hk) + static_cast<int64_t>(t0) * a.k.st;
    float* rows = sums + static_cast<int64_t>(blockIdx.x) * 2 * C * DK;  // what the heads of v before have given to dQ's and dK's rows, where there are several
    if (BOTH) tile_in<BY, T, DK, KP>(k, a.k.st, n, a.dk, kt), tile_in<BY, T, DK, KP>(q, a.q.st, n, a.dk, qt);
    const auto d_of = [&](int d) { return 16 * (half * KT + d); };
    for (int head_v = 0; head_v < rep; ++head_v) {
        const int h = hk * rep + head_v;
        const int64_t unit = static_cast<int64_t>(b) * a.Hv + h, place = unit * a.chunks + chunk;
        const T *v = head<const T>(a.v, b, h) + static_cast<int64_t>(t0) * a.v.st, *dout = head<const T>(a.dout, b, h) + static_cast<int64_t>(t0) * a.dout.st;
        const float *states = a.states + place * a.dk * a.dv, *dstates = a.dstates + place * a.dk * a.dv, *puts = a.puts + place * C * a.dv, *dputs = a.dputs + place * C * a.dv;
        // what a block of columns needs from memory, asked for a block ahead
        f32x4 x[SN], y[SN], u, r0, r1;
        Eight<BY, T> dov, vv;
        const int row = tid / (GB / 4), col = tid % (GB / 4) * 4;
        const auto load = [&](int v0) {
#pragma unroll
            for (int e = 0; e < SN; ++e)
                if (DK >= 64 || row < DK) x[e] = dense4<BY>(states, row + 64 * e, v0 + col, a.dk, a.dv), y[e] = dense4<BY>(dstates, row + 64 * e, v0 + col, a.dk, a.dv);
            u = dense4<BY>(puts, row, v0 + col, C, a.dv);
            r0 = dense4<BY>(dputs, i, v0 + 8 * g, C, a.dv), r1 = dense4<BY>(dputs, i, v0 + 8 * g + 4, C, a.dv);
            dov.load(dout, a.dout.st, mine_at, v0 + 8 * g, a.dv);
            if (half == 0) vv.load(v, a.v.st, mine_at, v0 + 8 * g, a.dv);
        };
        load(0);
        if (wave == 0) {  // the sum of the log-decays
            const float f = lane < n ? a.g[(static_cast<int64_t>(b) * a.T + t0 + lane) * a.Hv + h] : 0.0f;
            double s = f < LEAST ? LEAST : f;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double up = __shfl_up(s, o);
                if (lane >= o) s += up;
            }
            total[lane] = s;
        }
        f32x4 X[4] = {}, Y[KT] = {}, Yr[KT] = {}, Yu[KT] = {};  // X: of dO, or of dR
        float inner = 0.0f, rv = 0.0f;  // of <S, dS'>; of dR_i.V_i
#pragma unroll 1
        for (int v0 = 0; v0 < a.dv; v0 += GB) {
#pragma unroll
            for (int e = 0; e < SN; ++e)
                if (DK >= 64 || row < DK) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) inner = fmaf(x[e][j], y[e][j], inner);
                    put4<3, DK, VQ>(s0, row + 64 * e, col, x[e]), put4<3, DK, VQ>(s1, row + 64 * e, col, y[e]);
                }
            put4<3, C, VQ>(ut, row, col, u);
            if (half == 0) {
                f32x4 x0, x1;
                values_of(vv, x0, x1);
#pragma unroll
                for (int j = 0; j < 4; ++j) rv = fmaf(r0[j], x0[j], fmaf(r1[j], x1[j], rv));
            }
            const Operand<3> dr = split8<3>(r0, r1);
            const Operand<N> od = dov.operand();
            __syncthreads();
            if (AHEAD && v0 + GB < a.dv) load(v0 + GB);
            const Operand<3> ui = rows_of<3, C, VQ>(ut, 16 * tile, 0, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j <= tile) {
                    const Operand<3> uj = rows_of<3, C, VQ>(ut, 16 * j, 0, lane);
                    if (half == 0)
                        product<2>(uj, od, X[j]);
                    else
                        product<2>(uj, dr, X[j]);
                }
#pragma unroll
            for (int d = 0; d < KT; ++d) {
                __builtin_amdgcn_sched_barrier(0);  // the operands of one d at a time: those of all would not fit into the registers
                const Operand<3> s = rows_of<3, DK, VQ>(s0, d_of(d), 0, lane), t = rows_of<3, DK, VQ>(s1, d_of(d), 0, lane);
                product<2>(s, od, Y[d]), product<2>(s, dr, Yr[d]), product<2>(t, ui, Yu[d]);
            }
            if (!AHEAD && v0 + GB < a.dv) load(v0 + GB);
            __syncthreads();
        }
        // Addresses from here on are formed of numbers that the compiler cannot know: formed before the columns go by, they would be held, or spilled, through all of that.
        int lane_then = lane, i_then = i, mine_then = mine_at;
        asm volatile("" : "+v"(lane_then), "+v"(i_then), "+v"(mine_then));
        const float* scalars = a.scalars + place * 3 * C;
        const float2 decay = make_float2(scalars[i_then], scalars[C + i_then]);
        const float beta = scalars[2 * C + i_then];
        // E and F, and what they give to dbeta and to the decays
        float db = 0.0f;
        {
            const int g = lane_then >> 4, c16 = lane_then & 15, i = i_then;
            // rows of K and Q as operands: from LDS, or from memory
            const auto row_k = [&](int j, int s) {
                if constexpr (BOTH) return rows_of<N, C, KP>(kt, 16 * j, 32 * s, lane_then);
                Eight<BY, T> e;
                e.load(k, a.k.st, min(16 * j + c16, n - 1), 32 * s + 8 * g, a.dk);
                return e.operand();
            };
            const auto row_own = [&](int s) {
                if constexpr (BOTH) return rows_of<N, C, KP>(half == 0 ? qt : kt, 16 * tile, 32 * s, lane_then);
                Eight<BY, T> e;
                if (half == 0)
                    e.load(q, a.q.st, mine_then, 32 * s + 8 * g, a.dk);
                else
                    e.load(k, a.k.st, mine_then, 32 * s + 8 * g, a.dk);
                return e.operand();
            };
            const float factor = half == 0 ? a.scale : -beta;
            f32x4 xk[4] = {};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                __builtin_amdgcn_sched_barrier(0);
                const Operand<N> own = row_own(s);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j <= tile) product<MOST>(row_k(j, s), own, xk[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4 H = {0, 0, 0, 0};
                if (j <= tile) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int at = 16 * j + 4 * g + r;
                        const float D = here && (half == 0 ? at <= i : at < i) ? decay_of(total[i] - total[at]) : 0.0f, z = D == 0.0f ? 0.0f : D * X[j][r];
                        X[j][r] = factor * z;
                        H[r] = at < i ? X[j][r] * xk[j][r] : 0.0f;
                        db = fmaf(z, xk[j][r], db);
                    }
                }
                put4<3, C, AP>(half == 0 ? et : ft, i, 16 * j + 4 * g, X[j]);
                *reinterpret_cast<f32x4*>(ht + i * HP + 16 * j + 4 * g) = H;
            }
        }
        const int g4 = lane_then >> 4 << 2;
        float qy = 0.0f, kr = 0.0f, ku = 0.0f;
#pragma unroll
        for (int d = 0; d < KT; ++d) {
            f32x4 xq, xk;
            if constexpr (N == 1) {
                xq = load4(qt + i_then * KP, d_of(d) + g4, DK), xk = load4(kt + i_then * KP, d_of(d) + g4, DK);
            } else {
                xq = load4(q + mine_then * a.q.st, d_of(d) + g4, a.dk), xk = load4(k + mine_then * a.k.st, d_of(d) + g4, a.dk);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) qy = fmaf(xq[r], Y[d][r], qy), kr = fmaf(xk[r], Yr[d][r], kr), ku = fmaf(xk[r], Yu[d][r], ku);
        }
        const float in = here ? a.scale * decay.x : 0.0f, back = -beta * decay.x;
        const float tail = over_groups(ku) * decay.y, end = over_groups(fmaf(in, qy, back * kr));
        db = over_groups(fmaf(-decay.x, kr, half == 0 ? rv : -db));
        inner = group_sum<64>(inner);
        if (g == 0) ends[half][i] = end, tails[half][i] = tail, dbs[half][i] = db;
        if (lane == 0) dots[wave] = inner;
        __syncthreads();
        {
            double s = 0.0;
#pragma unroll
            for (int j = 0; j < 16; ++j) s += static_cast<double>(ht[lane * HP + 16 * tile + j]) - static_cast<double>(ht[(16 * tile + j) * HP + lane]);
            across[wave][lane] = s;
        }
        __syncthreads();
        if (!BOTH) {
            tile_in<BY, T, DK, KP>(k, a.k.st, n, a.dk, kt);
            __syncthreads();
        }
        if (wave == 0) {
            double all = 0.0, t = static_cast<double>(tails[0][lane]) + tails[1][lane], s = static_cast<double>(ends[0][lane]) + ends[1][lane] - t;
#pragma unroll
            for (int w = 0; w < 8; ++w) all += dots[w], s += across[w][lane];
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) t += __shfl_xor(t, o);
            if (lane == 63) s += t + scalars[C - 1] * all;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double down = __shfl_down(s, o);
                if (lane + o < 64) s += down;
            }
            const int64_t at = (static_cast<int64_t>(b) * a.T + t0 + lane_then) * a.Hv + h;
            if (lane < n) a.dg[at] = a.g[at] < LEAST ? 0.0f : static_cast<float>(s), a.dbeta[at] = dbs[0][lane] + dbs[1][lane];
        }
        // dQ = scale gamma Y + E K, dK = delta Yu - beta gamma Yr + F K + F^T K + E^T Q
#pragma unroll
        for (int d = 0; d < KT; ++d) {
            Y[d] *= in;
            Yu[d] = Yu[d] * decay.y + Yr[d] * back;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const Operand<3> e = rows_of<3, C, AP>(et, 16 * tile, 32 * s, lane_then), f = rows_of<3, C, AP>(ft, 16 * tile, 32 * s, lane_then),
                              ft_ = cols_of<3, C, AP>(ft, 32 * s, 16 * tile, lane_then);
#pragma unroll
            for (int d = 0; d < KT; ++d) {
                const Operand<N> x = cols_of<N, C, KP>(kt, 32 * s, d_of(d), lane_then);
                product<2>(x, e, Y[d]), product<2>(x, f, Yu[d]), product<2>(x, ft_, Yu[d]);
            }
        }
        if (!BOTH) {
            __syncthreads();
            tile_in<BY, T, DK, KP>(q, a.q.st, n, a.dk, qt);
            __syncthreads();
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const Operand<3> et_ = cols_of<3, C, AP>(et, 32 * s, 16 * tile, lane_then);
#pragma unroll
            for (int d = 0; d < KT; ++d) product<2>(cols_of<N, C, KP>(qt, 32 * s, d_of(d), lane_then), et_, Yu[d]);
        }
        const bool last = head_v == rep - 1;
        float* mine = rows + i_then * DK;
        T *dq = head<T>(a.dq, b, hk) + (static_cast<int64_t>(t0) + mine_then) * a.dq.st, *dk = head<T>(a.dk_, b, hk) + (static_cast<int64_t>(t0) + mine_then) * a.dk_.st;
#pragma unroll
        for (int d = 0; d < KT; ++d) {
            const int c = d_of(d) + g4;
            if (head_v > 0) Y[d] += *reinterpret_cast<const f32x4*>(mine + c), Yu[d] += *reinterpret_cast<const f32x4*>(mine + C * DK + c);
            if (!last) *reinterpret_cast<f32x4*>(mine + c) = Y[d], *reinterpret_cast<f32x4*>(mine + C * DK + c) = Yu[d];
            if (last && here) write4<BY>(dq, c, a.dk, Y[d]), write4<BY>(dk, c, a.dk, Yu[d]);
        }
        __syncthreads();  // the next head's columns come where these matrices are
    }
}

// ---- launches ----
template <typename T, int DK, int VB, Rows BY>
int launch_back(const Rule& a, hipStream_t st) {
    constexpr size_t lds = back_lds<T, DK, VB>();
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    PK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(walk_back<T, DK, VB, BY>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
    walk_back<T, DK, VB, BY><<<unit_grid(static_cast<int64_t>(a.B) * a.Hv, blocks(a.dv, VB)), 16 * VB, lds, st>>>(a);
    return launched();
}
template <typename T, int DK, Rows BY>
int launch_grads(const Rule& a, float* sums, hipStream_t st) {
    constexpr size_t lds = grads_lds<T, DK>();
    static_assert(lds <= 156 * 1024, "LDS of a CU");
    PK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(chunk_grads<T, DK, BY>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
    chunk_grads<T, DK, BY><<<dim3(static_cast<unsigned>(static_cast<int64_t>(a.B) * a.Hk * a.chunks)), GRAD_NT, lds, st>>>(a, sums);
    return launched();
}
template <typename T>
int launch_backward(const Rule& a, float* sums, int dtype, hipStream_t st) {
    if (a.chunks > 0) {
        if (int rc = launch_chunks(a, dtype, true, st)) return rc;
        if (int rc = launch_states(a, dtype, st)) return rc;
    }
    const int rc = by_size(a.dk, [&](auto dk) {
        constexpr int DK = decltype(dk)::value;
        if constexpr (back_lds<T, DK, 32>() <= 160 * 1024)
            if (wide(a)) return by_rows(rows_by(a, DK, 32), [&](auto by) { return launch_back<T, DK, 32, decltype(by)::value>(a, st); });
        return by_rows(rows_by(a, DK, 16), [&](auto by) { return launch_back<T, DK, 16, decltype(by)::value>(a, st); });
    });
    if (rc || a.chunks == 0) return rc;
    return by_size(a.dk, [&](auto dk) {
        constexpr int DK = decltype(dk)::value;
        return by_rows(rows_by(a, DK, GB), [&](auto by) { return launch_grads<T, DK, decltype(by)::value>(a, sums, st); });
    });
}

struct Room {
    size_t matrix, scalars, states, puts, sums, all;
};
Room room_of(const pk_delta_shape* s) {
    const size_t places = static_cast<size_t>(s->B) * s->Hv * chunks(s->T), groups = static_cast<size_t>(s->B) * s->Hk * chunks(s->T);
    const size_t rows = s->dk <= 32 ? 32 : s->dk <= 64 ? 64 : 128;
    Room r;
    r.matrix = pad(places * 3 * MATRIX), r.scalars = pad(places * 3 * C * sizeof(float)), r.states = pad(places * s->dk * s->dv * sizeof(float)), r.puts = pad(places * C * s->dv * sizeof(float));
    r.sums = s->Hv > s->Hk ? pad(groups * 2 * C * rows * sizeof(float)) : 0;
    r.all = 3 * r.matrix + r.scalars + 2 * r.states + 2 * r.puts + r.sums;
    return r;
}

}  // namespace
}  // namespace delta
}  // namespace pk

using namespace pk;
using namespace pk::delta;

extern "C" {

size_t pk_delta_rule_bwd_workspace_bytes(const pk_delta_shape* s) { return delta::check("pk_delta_rule_bwd", s) == PK_OK ? room_of(s).all : 0; }

int pk_delta_rule_bwd(const pk_delta_shape* s, const pk_tensor4* d_o, const float* dstate_out, const pk_tensor4* q, const pk_tensor4* k, const pk_tensor4* v, const float* g,
                      const float* beta, const float* state_in, const pk_tensor4* dq, const pk_tensor4* dk, const pk_tensor4* dv, float* dg, float* dbeta, float* dstate_in,
                      void* workspace, size_t workspace_bytes, void* stream) {
    return c_entry([&] {
        const std::string who = "pk_delta_rule_bwd";
        if (int rc = delta::check(who.c_str(), s)) return rc;
        Rule a{};
        if (s->B == 0) return static_cast<int>(PK_OK);
        if (s->T > 0 && (!view_of(d_o, a.dout) || !view_of(q, a.q) || !view_of(k, a.k) || !view_of(v, a.v) || !view_of(dq, a.dq) || !view_of(dk, a.dk_) || !view_of(dv, a.dv_) || !g ||
                         !beta || !dg || !dbeta))
            return fail(PK_ERR_ARGUMENT, who + ": null pointer");
        const Room r = room_of(s);
        if (r.all && (!workspace || workspace_bytes < r.all || !aligned(workspace, 16)))
            return fail(PK_ERR_WORKSPACE, who + ": workspace too small (pk_delta_rule_bwd_workspace_bytes)");
        if (shares(a.dq, s, s->Hk) || shares(a.dk_, s, s->Hk) || shares(a.dv_, s, s->Hv)) return fail(PK_ERR_ARGUMENT, who + ": elements of a gradient share memory");
        const size_t gates = sizeof(float) * s->B * s->T * s->Hv, state = sizeof(float) * s->B * s->Hv * s->dk * s->dv;
        if (!apart({span_of(a.dq, s, s->Hk, s->dk), span_of(a.dk_, s, s->Hk, s->dk), span_of(a.dv_, s, s->Hv, s->dv), span_of(dg, gates), span_of(dbeta, gates), span_of(dstate_in, state),
                    span_of(workspace, r.all)},
                   {span_of(a.dout, s, s->Hv, s->dv), span_of(dstate_out, state), span_of(a.q, s, s->Hk, s->dk), span_of(a.k, s, s->Hk, s->dk), span_of(a.v, s, s->Hv, s->dv),
                    span_of(g, gates), span_of(beta, gates), span_of(state_in, state)}))
            return fail(PK_ERR_ARGUMENT, who + ": results lie clear of one another, of the workspace and of what is read");
        touch({a.dout.ptr, dstate_out, a.q.ptr, a.k.ptr, a.v.ptr, g, beta, state_in, a.dq.ptr, a.dk_.ptr, a.dv_.ptr, dg, dbeta, dstate_in, workspace}, stream);
        a.g = g, a.beta = beta, a.state_in = state_in, a.dg = dg, a.dbeta = dbeta, a.dstate_out = dstate_out, a.dstate_in = dstate_in;
        a.B = s->B, a.T = s->T, a.Hk = s->Hk, a.Hv = s->Hv, a.dk = s->dk, a.dv = s->dv, a.chunks = chunks(s->T), a.scale = s->scale;
        char* at = static_cast<char*>(workspace);
        const auto take = [&](size_t bytes) {
            char* p = at;
            at += bytes;
            return p;
        };
        a.inverse = reinterpret_cast<uint16_t*>(take(r.matrix)), a.inverse_t = reinterpret_cast<uint16_t*>(take(r.matrix)), a.attn_t = reinterpret_cast<uint16_t*>(take(r.matrix));
        a.attn = a.attn_t;  // not written in the backward
        a.scalars = reinterpret_cast<float*>(take(r.scalars));
        a.states = reinterpret_cast<float*>(take(r.states)), a.dstates = reinterpret_cast<float*>(take(r.states));
        a.puts = reinterpret_cast<float*>(take(r.puts)), a.dputs = reinterpret_cast<float*>(take(r.puts));
        float* sums = reinterpret_cast<float*>(take(r.sums));
        hipStream_t st = static_cast<hipStream_t>(stream);
        return s->dtype == PK_BF16 ? launch_backward<uint16_t>(a, sums, s->dtype, st) : launch_backward<float>(a, sums, s->dtype, st);
    });
}

}  // extern "C"
