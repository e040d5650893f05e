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
// forward's takes 32 columns of a state by themselves; then, a workgroup for a chunk and a head of k, all that needs every column of a state. What bounds it: the states of all
// chunks, written and read once each way, and the matrix cores in the last launch.
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
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c16 = lane & 15;
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
// A workgroup for a chunk of a head of k, its heads of v one after the other; wavefront w has tokens 16w .. 16w+15, a lane one of them.
constexpr int VQ = GB + 8, AP = C + 8, HP = C + 4;  // pitches of rows that are read along k; of H
template <typename T, int DK>
constexpr int tiles() {
    return std::max((PARTS<T> == 1 ? 2 : 3) * C * (DK + 16), 2 * C * HP);
}
template <typename T, int DK>
constexpr size_t grads_lds() {
    constexpr int PE = PARTS<T> == 1 ? 2 : 3;
    return sizeof(uint16_t) * std::max((6 * DK + 3 * C) * VQ, tiles<T, DK>() + 2 * PE * C * AP);
}
__device__ inline float over_groups(float x) {  // the four lanes of a token
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}
template <typename T, int DK>
__global__ __launch_bounds__(256) void chunk_grads(Rule a, float* sums) {
    constexpr int N = PARTS<T>, MOST = N == 1 ? 0 : 2, PE = N == 1 ? 2 : 3, KP = DK + 16, KS = DK / 32, KT = DK / 16;
    constexpr bool BOTH = N == 1;
    extern __shared__ uint16_t lds[];
    __shared__ double total[C];
    __shared__ double across[4][C];
    __shared__ float ends[C], tails[C], dots[4];
    uint16_t *s0 = lds, *s1 = s0 + 3 * DK * VQ, *ut = s1 + 3 * DK * VQ;                            // while the columns of the state go by
    uint16_t *kt = lds, *qt = BOTH ? kt + C * KP : kt, *et = kt + tiles<T, DK>(), *ft = et + PE * C * AP;  // then
    float* ht = reinterpret_cast<float*>(lds);  // before K and Q come there
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c16 = lane & 15, i = 16 * wave + c16;
    const int64_t group = blockIdx.x / static_cast<unsigned>(a.chunks);
    const int chunk = blockIdx.x % static_cast<unsigned>(a.chunks), b = static_cast<int>(group / a.Hk), hk = static_cast<int>(group % a.Hk), rep = a.Hv / a.Hk;
    const int t0 = chunk * C, n = min(C, a.T - t0);
    const bool here = i < n;
    const int64_t row = t0 + (here ? i : 0);
    const T *q = head<const T>(a.q, b, hk), *k = head<const T>(a.k, b, hk), *qi = q + row * a.q.st, *ki = k + row * a.k.st;
    float* mine = rep > 1 ? sums + static_cast<int64_t>(blockIdx.x) * 2 * C * DK + i * DK : nullptr;  // what the heads of v before have given to dQ's and dK's rows
    for (int head_v = 0; head_v < rep; ++head_v) {
        const int h = hk * rep + head_v;
        const int64_t unit = static_cast<int64_t>(b) * a.Hv + h, place = unit * a.chunks + chunk, scalar_at = (static_cast<int64_t>(b) * a.T + t0 + i) * a.Hv + h;
        const T *v = head<const T>(a.v, b, h) + row * a.v.st, *dout = head<const T>(a.dout, b, h) + row * a.dout.st;
        const float *states = a.states + place * a.dk * a.dv, *dstates = a.dstates + place * a.dk * a.dv, *puts = a.puts + place * C * a.dv, *dputs = a.dputs + (place * C + i) * a.dv;
        if (wave == 0) {  // the sum of the log-decays
            const float x = lane < n ? a.g[(static_cast<int64_t>(b) * a.T + t0 + lane) * a.Hv + h] : 0.0f;
            double s = x < LEAST ? LEAST : x;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double up = __shfl_up(s, o);
                if (lane >= o) s += up;
            }
            total[lane] = s;
        }
        f32x4 X[4] = {}, Z[4] = {}, Y[KT] = {}, Yr[KT] = {}, Yu[KT] = {};
        float inner = 0.0f, rv = 0.0f;  // of <S, dS'>; of dR_i.V_i
        for (int v0 = 0; v0 < a.dv; v0 += GB) {
            for (int e = tid; e < DK * (GB / 4); e += 256) {
                const int r = e / (GB / 4), c = e % (GB / 4) * 4;
                const f32x4 x = load4(states + (r < a.dk ? r : 0) * a.dv, v0 + c, r < a.dk ? a.dv : 0), y = load4(dstates + (r < a.dk ? r : 0) * a.dv, v0 + c, r < a.dk ? a.dv : 0);
#pragma unroll
                for (int j = 0; j < 4; ++j) inner = fmaf(x[j], y[j], inner);
                put4<3, DK, VQ>(s0, r, c, x), put4<3, DK, VQ>(s1, r, c, y);
            }
            for (int e = tid; e < C * (GB / 4); e += 256) {
                const int r = e / (GB / 4), c = e % (GB / 4) * 4;
                put4<3, C, VQ>(ut, r, c, load4(puts + r * a.dv, v0 + c, a.dv));
            }
            const int c = v0 + 8 * g;
            const f32x4 r0 = load4(dputs, c, a.dv), r1 = load4(dputs, c + 4, a.dv), x0 = load4(v, c, here ? a.dv : 0), x1 = load4(v, c + 4, here ? a.dv : 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) rv = fmaf(r0[j], x0[j], fmaf(r1[j], x1[j], rv));
            const Operand<3> dr = split8<3>(r0, r1);
            const Operand<N> od = load8(dout, c, here ? a.dv : 0);
            __syncthreads();
            const Operand<3> u = rows_of<3, C, VQ>(ut, 16 * wave, 0, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j <= wave) {
                    const Operand<3> uj = rows_of<3, C, VQ>(ut, 16 * j, 0, lane);
                    product<2>(uj, od, X[j]), product<2>(uj, dr, Z[j]);
                }
#pragma unroll
            for (int d = 0; d < KT; ++d) {
                const Operand<3> s = rows_of<3, DK, VQ>(s0, 16 * d, 0, lane);
                product<2>(s, od, Y[d]), product<2>(s, dr, Yr[d]);
                product<2>(rows_of<3, DK, VQ>(s1, 16 * d, 0, lane), u, Yu[d]);
            }
            __syncthreads();
        }
        const float* scalars = a.scalars + place * 3 * C;
        const float2 decay = make_float2(scalars[i], scalars[C + i]);
        const float beta = scalars[2 * C + i];
        // E and F, and what they give to dbeta and to the decays
        float db = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x4 qk = {0, 0, 0, 0}, kk = qk, H = qk;
            if (j <= wave) {
                const int other = 16 * j + c16;
                const T* kj = k + static_cast<int64_t>(t0 + (other < n ? other : 0)) * a.k.st;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const Operand<N> x = load8(kj, 32 * s + 8 * g, other < n ? a.dk : 0);
                    product<MOST>(x, load8(qi, 32 * s + 8 * g, here ? a.dk : 0), qk), product<MOST>(x, load8(ki, 32 * s + 8 * g, here ? a.dk : 0), kk);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = 16 * j + 4 * g + r;
                    const float D = at <= i ? decay_of(total[i] - total[at]) : 0.0f, z = at < i ? D * Z[j][r] : 0.0f;
                    X[j][r] *= a.scale * D, Z[j][r] = -beta * z;
                    if (at > i) X[j][r] = 0.0f;
                    H[r] = at < i ? fmaf(X[j][r], qk[r], Z[j][r] * kk[r]) : 0.0f;
                    db = fmaf(z, kk[r], db);
                }
            }
            put4<PE, C, AP>(et, i, 16 * j + 4 * g, X[j]), put4<PE, C, AP>(ft, i, 16 * j + 4 * g, Z[j]);
            *reinterpret_cast<f32x4*>(ht + i * HP + 16 * j + 4 * g) = H;
        }
        float qy = 0.0f, kr = 0.0f, ku = 0.0f;
#pragma unroll
        for (int d = 0; d < KT; ++d) {
            const f32x4 x = load4(qi, 16 * d + 4 * g, here ? a.dk : 0), y = load4(ki, 16 * d + 4 * g, here ? a.dk : 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) qy = fmaf(x[r], Y[d][r], qy), kr = fmaf(y[r], Yr[d][r], kr), ku = fmaf(y[r], Yu[d][r], ku);
        }
        const float in = a.scale * decay.x, back = -beta * decay.x;
        const float tail = over_groups(ku) * decay.y, end = over_groups(fmaf(in, qy, back * kr));
        db = over_groups(rv - fmaf(decay.x, kr, db));
        inner = group_sum<64>(inner);
        if (g == 0) {
            ends[i] = end, tails[i] = tail;
            if (here) a.dbeta[scalar_at] = db;
        }
        if (lane == 0) dots[wave] = inner;
        __syncthreads();
        {
            double s = 0.0;
#pragma unroll
            for (int j = 0; j < 16; ++j) s += static_cast<double>(ht[lane * HP + 16 * wave + j]) - static_cast<double>(ht[(16 * wave + j) * HP + lane]);
            across[wave][lane] = s;
        }
        __syncthreads();
        tile_to_lds<T, DK, KP, 256>(k + static_cast<int64_t>(t0) * a.k.st, a.k.st, n, a.dk, kt);
        if (BOTH) tile_to_lds<T, DK, KP, 256>(q + static_cast<int64_t>(t0) * a.q.st, a.q.st, n, a.dk, qt);
        __syncthreads();
        if (wave == 0) {
            const double all = static_cast<double>(dots[0]) + dots[1] + dots[2] + dots[3];
            double t = tails[lane], s = static_cast<double>(ends[lane]) - t + (across[0][lane] + across[1][lane]) + (across[2][lane] + across[3][lane]);
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) t += __shfl_xor(t, o);
            if (lane == 63) s += t + scalars[C - 1] * all;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double down = __shfl_down(s, o);
                if (lane + o < 64) s += down;
            }
            const int64_t at = (static_cast<int64_t>(b) * a.T + t0 + lane) * a.Hv + h;
            if (lane < n) a.dg[at] = a.g[at] < LEAST ? 0.0f : static_cast<float>(s);
        }
        // dQ = scale gamma Y + E K, dK = delta Yu - beta gamma Yr + F K + F^T K + E^T Q
#pragma unroll
        for (int d = 0; d < KT; ++d) {
            Y[d] *= in;
            Yu[d] = Yu[d] * decay.y + Yr[d] * back;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const Operand<PE> e = rows_of<PE, C, AP>(et, 16 * wave, 32 * s, lane), f = rows_of<PE, C, AP>(ft, 16 * wave, 32 * s, lane),
                              ft_ = cols_of<PE, C, AP>(ft, 32 * s, 16 * wave, lane);
#pragma unroll
            for (int d = 0; d < KT; ++d) {
                const Operand<N> x = cols_of<N, C, KP>(kt, 32 * s, 16 * d, lane);
                product<PE - 1>(x, e, Y[d]), product<PE - 1>(x, f, Yu[d]), product<PE - 1>(x, ft_, Yu[d]);
            }
        }
        if (!BOTH) {
            __syncthreads();
            tile_to_lds<T, DK, KP, 256>(q + static_cast<int64_t>(t0) * a.q.st, a.q.st, n, a.dk, qt);
            __syncthreads();
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const Operand<PE> et_ = cols_of<PE, C, AP>(et, 32 * s, 16 * wave, lane);
#pragma unroll
            for (int d = 0; d < KT; ++d) product<PE - 1>(cols_of<N, C, KP>(qt, 32 * s, 16 * d, lane), et_, Yu[d]);
        }
        const bool last = head_v == rep - 1;
        T *dq = head<T>(a.dq, b, hk) + row * a.dq.st, *dk = head<T>(a.dk_, b, hk) + row * a.dk_.st;
#pragma unroll
        for (int d = 0; d < KT; ++d) {
            const int c = 16 * d + 4 * g;
            if (head_v > 0) Y[d] += *reinterpret_cast<const f32x4*>(mine + c), Yu[d] += *reinterpret_cast<const f32x4*>(mine + C * DK + c);
            if (!last) *reinterpret_cast<f32x4*>(mine + c) = Y[d], *reinterpret_cast<f32x4*>(mine + C * DK + c) = Yu[d];
            if (last && here) store4(dq, c, a.dk, Y[d]), store4(dk, c, a.dk, Yu[d]);
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
template <typename T, int DK>
int launch_grads(const Rule& a, float* sums, hipStream_t st) {
    constexpr size_t lds = grads_lds<T, DK>();
    static_assert(lds <= 156 * 1024, "LDS of a CU");
    PK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(chunk_grads<T, DK>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
    chunk_grads<T, DK><<<dim3(static_cast<unsigned>(static_cast<int64_t>(a.B) * a.Hk * a.chunks)), 256, lds, st>>>(a, sums);
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
        return by_rows(rows_by(a, DK, 16), [&](auto by) { return launch_back<T, DK, 16, decltype(by)::value>(a, st); });
    });
    if (rc || a.chunks == 0) return rc;
    return by_size(a.dk, [&](auto dk) { return launch_grads<T, decltype(dk)::value>(a, sums, st); });
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
