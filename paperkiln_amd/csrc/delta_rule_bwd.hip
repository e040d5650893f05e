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
__device__ inline int token_tile(int wave, int i) { return (wave >> 1) ? 1 + i : 3 * i; }

template <typename T, int DK>
constexpr size_t back_lds() {
    return sizeof(uint16_t) * ((PARTS<T> == 1 ? 2 : 3) * C * (DK + 16) + 3 * DK * VP + 9 * C * VP + PARTS<T> * C * VP);
}
template <typename T, int DK>
__global__ __launch_bounds__(256) void walk_back(Rule a) {
    constexpr int N = PARTS<T>, KP = DK + 16, KS = DK / 32, KT = DK / 32;
    constexpr bool BOTH = N == 1;  // K and Q side by side in LDS; three parts of each take turns
    extern __shared__ uint16_t lds[];
    uint16_t *kt = lds, *qt = BOTH ? kt + C * KP : kt, *st = kt + (BOTH ? 2 : 3) * C * KP, *ut = st + 3 * DK * VP, *wt = ut + 3 * C * VP, *dt = wt + 3 * C * VP, *rt = dt + 3 * C * VP;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c16 = lane & 15;
    int unit, blk;
    if (!unit_of(blockIdx.x, a.B * a.Hv, (a.dv + VB - 1) / VB, unit, blk)) return;
    const int b = unit / a.Hv, h = unit - b * a.Hv, hk = h / (a.Hv / a.Hk);
    const int vt = 16 * (wave & 1), vc = VB * blk + vt + 4 * g;
    const T *q = head<const T>(a.q, b, hk), *k = head<const T>(a.k, b, hk), *dout = head<const T>(a.dout, b, h);
    T* dv = head<T>(a.dv_, b, h);
    const int64_t state_at = static_cast<int64_t>(unit) * a.dk * a.dv;
    f32x4 S[KT];  // of the gradient of the state
#pragma unroll
    for (int i = 0; i < KT; ++i) {
        const int r = 16 * ((wave >> 1) * KT + i) + c16;
        S[i] = a.dstate_out && r < a.dk ? load4(a.dstate_out + state_at + static_cast<int64_t>(r) * a.dv, vc, a.dv) : f32x4{0, 0, 0, 0};
    }
    for (int chunk = a.chunks - 1; chunk >= 0; --chunk) {
        const int t0 = chunk * C, n = min(C, a.T - t0);
        const int64_t place = static_cast<int64_t>(unit) * a.chunks + chunk;
        const float2* decay = a.decay + place * C;
        tile_to_lds<T, DK, KP, 256>(k + static_cast<int64_t>(t0) * a.k.st, a.k.st, n, a.dk, kt);
        if (BOTH) tile_to_lds<T, DK, KP, 256>(q + static_cast<int64_t>(t0) * a.q.st, a.q.st, n, a.dk, qt);
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            const int r = 16 * ((wave >> 1) * KT + i) + c16;
            put4<3, DK, VP>(st, r, vt + 4 * g, S[i]);
            if (r < a.dk) store4(a.dstates + (place * a.dk + r) * a.dv, vc, a.dv, S[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = 16 * token_tile(wave, i) + c16;
            const f32x4 x = load4(dout + static_cast<int64_t>(t0 + (t < n ? t : 0)) * a.dout.st, vc, t < n ? a.dv : 0);
            put4<N, C, VP>(rt, t, vt + 4 * g, x);
            put4<3, C, VP>(dt, t, vt + 4 * g, x * (a.scale * decay[t].x));
        }
        __syncthreads();
        // dU = A^T dO + delta K dS'
        {
            f32x4 X[2] = {}, Y[2] = {};
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                const Operand<3> s = cols_of<3, DK, VP>(st, 32 * kk, vt, lane);
#pragma unroll
                for (int i = 0; i < 2; ++i) product<2>(s, rows_of<N, C, KP>(kt, 16 * token_tile(wave, i), 32 * kk, lane), X[i]);
            }
            const uint16_t* attn_t = a.attn_t + place * 3 * (C * C);
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const Operand<N> d = cols_of<N, C, VP>(rt, 32 * kk, vt, lane);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (kk == 1 || token_tile(wave, i) < 2) product<2>(d, rows_of<3, C, C>(attn_t, 16 * token_tile(wave, i), 32 * kk, lane), Y[i]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int t = 16 * token_tile(wave, i) + c16;
                put4<3, C, VP>(ut, t, vt + 4 * g, Y[i] + X[i] * decay[t].y);
            }
        }
        __syncthreads();
        // dR = T^T dU
        {
            const uint16_t* inverse_t = a.inverse_t + place * 3 * (C * C);
            f32x4 R[2] = {};
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const Operand<3> u = cols_of<3, C, VP>(ut, 32 * kk, vt, lane);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (kk == 1 || token_tile(wave, i) < 2) product<2>(u, rows_of<3, C, C>(inverse_t, 16 * token_tile(wave, i), 32 * kk, lane), R[i]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int t = 16 * token_tile(wave, i) + c16;
                const float beta = t < n ? a.beta[(static_cast<int64_t>(b) * a.T + t0 + t) * a.Hv + h] : 0.0f;
                store4(a.dputs + (place * C + t) * a.dv, vc, a.dv, R[i]);
                if (t < n) store4(dv + static_cast<int64_t>(t0 + t) * a.dv_.st, vc, a.dv, R[i] * beta);
                put4<3, C, VP>(wt, t, vt + 4 * g, R[i] * (-beta * decay[t].x));
            }
        }
        __syncthreads();
        const float whole = decay[C - 1].x;
#pragma unroll
        for (int i = 0; i < KT; ++i) S[i] *= whole;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const Operand<3> w = cols_of<3, C, VP>(wt, 32 * kk, vt, lane);
#pragma unroll
            for (int i = 0; i < KT; ++i) product<2>(w, cols_of<N, C, KP>(kt, 32 * kk, 16 * ((wave >> 1) * KT + i), lane), S[i]);
        }
        if (!BOTH) {
            __syncthreads();
            tile_to_lds<T, DK, KP, 256>(q + static_cast<int64_t>(t0) * a.q.st, a.q.st, n, a.dk, qt);
            __syncthreads();
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const Operand<3> d = cols_of<3, C, VP>(dt, 32 * kk, vt, lane);
#pragma unroll
            for (int i = 0; i < KT; ++i) product<2>(d, cols_of<N, C, KP>(qt, 32 * kk, 16 * ((wave >> 1) * KT + i), lane), S[i]);
        }
        __syncthreads();
    }
    if (!a.dstate_in) return;
#pragma unroll
    for (int i = 0; i < KT; ++i) {
        const int r = 16 * ((wave >> 1) * KT + i) + c16;
        if (r < a.dk) store4(a.dstate_in + state_at + static_cast<int64_t>(r) * a.dv, vc, a.dv, S[i]);
    }
}

// ---- what needs all columns of a state ----
// A workgroup for a chunk of a head of k, its heads of v one after the other; wavefront w has tokens 16w .. 16w+15, a lane one of them.
constexpr int VQ = VB + 8, AP = C + 8, HP = C + 4;  // pitches of rows that are read along k; of H
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
        for (int v0 = 0; v0 < a.dv; v0 += VB) {
            for (int e = tid; e < DK * (VB / 4); e += 256) {
                const int r = e / (VB / 4), c = e % (VB / 4) * 4;
                const f32x4 x = load4(states + (r < a.dk ? r : 0) * a.dv, v0 + c, r < a.dk ? a.dv : 0), y = load4(dstates + (r < a.dk ? r : 0) * a.dv, v0 + c, r < a.dk ? a.dv : 0);
#pragma unroll
                for (int j = 0; j < 4; ++j) inner = fmaf(x[j], y[j], inner);
                put4<3, DK, VQ>(s0, r, c, x), put4<3, DK, VQ>(s1, r, c, y);
            }
            for (int e = tid; e < C * (VB / 4); e += 256) {
                const int r = e / (VB / 4), c = e % (VB / 4) * 4;
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
        const float2 decay = a.decay[place * C + i];
        const float beta = here ? a.beta[scalar_at] : 0.0f;
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
            if (lane == 63) s += t + a.decay[place * C + 63].x * all;
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
template <typename T, int DK>
int launch_back(const Rule& a, hipStream_t st) {
    constexpr size_t lds = back_lds<T, DK>();
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    PK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(walk_back<T, DK>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
    walk_back<T, DK><<<unit_grid(static_cast<int64_t>(a.B) * a.Hv, blocks(a.dv)), 256, lds, st>>>(a);
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
    const auto by_rows = [&](auto&& f) { return a.dk <= 32 ? f(std::integral_constant<int, 32>{}) : a.dk <= 64 ? f(std::integral_constant<int, 64>{}) : f(std::integral_constant<int, 128>{}); };
    if (a.chunks > 0) {
        if (int rc = launch_chunks(a, dtype, true, st)) return rc;
        if (int rc = launch_states(a, dtype, st)) return rc;
    }
    if (int rc = by_rows([&](auto dk) { return launch_back<T, decltype(dk)::value>(a, st); })) return rc;
    return a.chunks == 0 ? PK_OK : by_rows([&](auto dk) { return launch_grads<T, decltype(dk)::value>(a, sums, st); });
}

struct Room {
    size_t matrix, decay, states, puts, sums, all;
};
Room room_of(const pk_delta_shape* s) {
    const size_t places = static_cast<size_t>(s->B) * s->Hv * chunks(s->T), groups = static_cast<size_t>(s->B) * s->Hk * chunks(s->T);
    const size_t rows = s->dk <= 32 ? 32 : s->dk <= 64 ? 64 : 128;
    Room r;
    r.matrix = pad(places * 3 * MATRIX), r.decay = pad(places * C * sizeof(float2)), r.states = pad(places * s->dk * s->dv * sizeof(float)), r.puts = pad(places * C * s->dv * sizeof(float));
    r.sums = s->Hv > s->Hk ? pad(groups * 2 * C * rows * sizeof(float)) : 0;
    r.all = 3 * r.matrix + r.decay + 2 * r.states + 2 * r.puts + r.sums;
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
        a.decay = reinterpret_cast<float2*>(take(r.decay));
        a.states = reinterpret_cast<float*>(take(r.states)), a.dstates = reinterpret_cast<float*>(take(r.states));
        a.puts = reinterpret_cast<float*>(take(r.puts)), a.dputs = reinterpret_cast<float*>(take(r.puts));
        float* sums = reinterpret_cast<float*>(take(r.sums));
        hipStream_t st = static_cast<hipStream_t>(stream);
        return s->dtype == PK_BF16 ? launch_backward<uint16_t>(a, sums, s->dtype, st) : launch_backward<float>(a, sums, s->dtype, st);
    });
}

}  // extern "C"
