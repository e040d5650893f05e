// Layer norm with the residual addition in front of it, and its gradient with the sums over all rows that its weights need.
//
//   h = x + residual (rounded to its type)     mean = sum h / C     rstd = 1 / sqrt(sum (h - mean)^2 / C + eps)     y = (h - mean) rstd w + b
//   du = dy w, u = (h - mean) rstd:   dx = rstd (du - sum du / C - u sum(du u) / C) + dh,   dw = sum over rows of dy u,   db = of dy
//
// What bounds it: memory, every tensor read or written once. A row stays in registers between its sums and its result, so the variance is the sum of squares of
// differences and not a difference of sums. In the backward a lane keeps its columns while its wavefront walks down the rows, and adds dw and db up in registers;
// workgroups leave their sums as rows of a small matrix, which a second launch adds in a fixed order.
#include "rows.h"

#include <algorithm>

namespace pk {
namespace {

typedef f32x4 f32x4_any __attribute__((aligned(4)));

struct Norm {
    const void *x, *residual;
    int64_t ldx, ldr, rows;
    const float *w, *b;  // b may be null
    void *y, *h;         // dense; h where there is a residual
    float *mean, *rstd;
    int cols;
    float eps;
};
struct NormGrad {
    const void *dy, *h, *dh;  // dh may be null
    int64_t lddy, ldh, lddh, rows;
    const float *w, *mean, *rstd;
    void* dx;      // dense
    float* parts;  // [workgroups][2][cols]
    int cols;
};

template <typename T>
__device__ inline Piece<T> load_any(const T* p) {
    return Piece<T>{*reinterpret_cast<const u32x4_any*>(p)};
}
// as many weights as a piece has elements
template <int N>
__device__ inline void load_weights(const float* p, float (&w)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4_any*>(p + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[i + e] = v[e];
    }
}
__device__ inline float rounded(float x, float) { return x; }
__device__ inline float rounded(float x, uint16_t) { return __uint_as_float(pack_bf16(x, 0.0f) << 16); }

// x added up over the WAVES wavefronts of a row; with one of them nothing is shared. Called in turn with different places of LDS, so one barrier is enough.
template <int WAVES>
__device__ inline float row_total(float x, float* sh) {
    x = group_sum<64>(x);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) sh[(threadIdx.x >> 6) % WAVES] = x;
        __syncthreads();
        x = sh[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) x += sh[w];
    }
    return x;
}

// A row to WAVES wavefronts, PER pieces to a lane; rows of one wavefront four to a workgroup.
template <typename T, int WAVES, int PER, bool RESIDUAL>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void norm_held(Norm a) {
    constexpr int N = Piece<T>::N, ROW = WAVES * 64;
    __shared__ float sh[2][WAVES];
    const int tid = threadIdx.x, at = WAVES == 1 ? tid & 63 : tid;
    const int64_t r = WAVES == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + (tid >> 6) : blockIdx.x;
    if (r >= a.rows) return;
    const int pieces = a.cols / N, tail = a.cols - pieces * N, end = pieces * N + at;
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    const T* res = static_cast<const T*>(a.residual) + (RESIDUAL ? r * a.ldr : 0);
    float v[PER][N], edge = 0.0f, s = 0.0f;
    Piece<T> px[PER], pr[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int p = at + k * ROW;
        px[k] = p < pieces ? load_any(x + p * N) : Piece<T>{{0, 0, 0, 0}};
        if (RESIDUAL) pr[k] = p < pieces ? load_any(res + p * N) : Piece<T>{{0, 0, 0, 0}};
    }
    if (at < tail) edge = RESIDUAL ? rounded(elem(x, end) + elem(res, end), T()) : elem(x, end);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        int i = 0;
        px[k].each([&](float e) { v[k][i++] = e; });
        if constexpr (RESIDUAL) {
            i = 0;
            pr[k].each([&](float e) { v[k][i++] += e; });
            const Piece<T> h = px[k].map([&](int j, float) { return v[k][j]; });
            i = 0;
            h.each([&](float e) { v[k][i++] = e; });
            const int p = at + k * ROW;
            if (p < pieces) store_piece<false>(static_cast<T*>(a.h) + r * a.cols + p * N, h);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) s += v[k][j];
    }
    if (RESIDUAL && at < tail) put(static_cast<T*>(a.h) + r * a.cols, end, edge);
    const float mean = row_total<WAVES>(s + edge, sh[0]) / a.cols;
    s = at < tail ? (edge - mean) * (edge - mean) : 0.0f;
#pragma unroll
    for (int k = 0; k < PER; ++k)
        if (at + k * ROW < pieces) {
#pragma unroll
            for (int j = 0; j < N; ++j) s = fmaf(v[k][j] - mean, v[k][j] - mean, s);
        }
    const float rstd = 1.0f / sqrtf(row_total<WAVES>(s, sh[1]) / a.cols + a.eps);
    if (at == 0) a.mean[r] = mean, a.rstd[r] = rstd;
    T* y = static_cast<T*>(a.y) + r * a.cols;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int p = at + k * ROW;
        if (p >= pieces) continue;
        float w[N], b[N] = {};
        load_weights(a.w + p * N, w);
        if (a.b) load_weights(a.b + p * N, b);
        store_piece<false>(y + p * N, px[k].map([&](int j, float) { return fmaf((v[k][j] - mean) * rstd, w[j], b[j]); }));
    }
    if (at < tail) put(y, end, fmaf((edge - mean) * rstd, a.w[end], a.b ? a.b[end] : 0.0f));
}

// Rows that no workgroup holds: read three times, each element by the same thread.
constexpr int LONG_NT = 1024;
template <typename T, bool RESIDUAL>
__global__ __launch_bounds__(LONG_NT) void norm_long(Norm a) {
    constexpr int WAVES = LONG_NT / 64;
    __shared__ float sh[2][WAVES];
    const int64_t r = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    const T* res = static_cast<const T*>(a.residual) + (RESIDUAL ? r * a.ldr : 0);
    T* h = RESIDUAL ? static_cast<T*>(a.h) + r * a.cols : nullptr;
    const auto value = [&](int j) { return RESIDUAL ? rounded(elem(x, j) + elem(res, j), T()) : elem(x, j); };
    float s = 0.0f;
    for (int j = threadIdx.x; j < a.cols; j += LONG_NT) {
        const float e = value(j);
        if (RESIDUAL) put(h, j, e);
        s += e;
    }
    const float mean = row_total<WAVES>(s, sh[0]) / a.cols;
    s = 0.0f;
    for (int j = threadIdx.x; j < a.cols; j += LONG_NT) {
        const float e = value(j) - mean;
        s = fmaf(e, e, s);
    }
    const float rstd = 1.0f / sqrtf(row_total<WAVES>(s, sh[1]) / a.cols + a.eps);
    if (threadIdx.x == 0) a.mean[r] = mean, a.rstd[r] = rstd;
    T* y = static_cast<T*>(a.y) + r * a.cols;
    for (int j = threadIdx.x; j < a.cols; j += LONG_NT) put(y, j, fmaf((value(j) - mean) * rstd, a.w[j], a.b ? a.b[j] : 0.0f));
}

// ---- backward ----

template <typename T, int PER, bool ADD>
struct GradRow {  // what a lane holds of a row
    Piece<T> dy[PER], h[PER], dh[ADD ? PER : 1];
    float edge_dy, edge_h, edge_dh, mean, rstd;
};
template <int ROW, bool AHEAD, typename T, int PER, bool ADD>
__device__ inline void load_row(const NormGrad& a, int64_t r, int at, int pieces, int tail, GradRow<T, PER, ADD>& o) {
    constexpr int N = Piece<T>::N;
    const bool row = r < a.rows;
    const int64_t from = row ? r : 0;
    const T *dy = static_cast<const T*>(a.dy) + from * a.lddy, *h = static_cast<const T*>(a.h) + from * a.ldh, *dh = static_cast<const T*>(a.dh) + (ADD ? from * a.lddh : 0);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int p = at + k * ROW;
        const bool in = row && p < pieces;
        o.dy[k] = in ? load_any(dy + p * N) : Piece<T>{{0, 0, 0, 0}};
        o.h[k] = in ? load_any(h + p * N) : Piece<T>{{0, 0, 0, 0}};
        if constexpr (ADD && AHEAD) o.dh[k] = in ? load_any(dh + p * N) : Piece<T>{{0, 0, 0, 0}};
    }
    const bool in = row && at < tail;
    const int end = pieces * N + at;
    o.edge_dy = in ? elem(dy, end) : 0.0f, o.edge_h = in ? elem(h, end) : 0.0f, o.edge_dh = ADD && in ? elem(dh, end) : 0.0f;
    o.mean = row ? a.mean[r] : 0.0f, o.rstd = row ? a.rstd[r] : 0.0f;
}

// Rows that a walk adds up one behind the other in registers; what they come to is added to what the rows before have left. So however tall an input is, roundings that all go one way
// stay below 2^-16 of a sum. 262144 rows of 4096 columns in bf16: 1215 us, 1189 with one chain, 1413 with a workgroup for every 256 rows.
constexpr int MOST_CHAIN = 256;
// A workgroup walks down the rows, WALKS of them side by side, each WAVES wavefronts' own. AHEAD: the next rows' loads are on their way while one is worked on.
template <typename T, int WAVES, int PER, int WALKS, bool ADD, bool AHEAD>
__global__ __launch_bounds__(WAVES * 64 * WALKS) void norm_grad(NormGrad a) {
    constexpr int N = Piece<T>::N, ROW = WAVES * 64;
    __shared__ float sh[2][2][WALKS][WAVES];
    extern __shared__ float sums[];  // several walks: [WALKS][2][cols]
    const int tid = threadIdx.x, walk = tid / ROW, at = tid % ROW;
    const int pieces = a.cols / N, tail = a.cols - pieces * N, end = pieces * N + at;
    float w[PER][N], aw[PER][N], ab[PER][N], ew = 0.0f, eb = 0.0f;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
#pragma unroll
        for (int j = 0; j < N; ++j) w[k][j] = aw[k][j] = ab[k][j] = 0.0f;
        if (at + k * ROW < pieces) load_weights(a.w + (at + k * ROW) * N, w[k]);
    }
    const float edge_w = at < tail ? a.w[end] : 0.0f, per_col = 1.0f / a.cols;
    float* part = a.parts + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
    float* mine = WALKS > 1 ? sums + walk * 2 * a.cols : part;
    bool more = false;  // there are sums of rows before
    const auto leave = [&] {
        const auto add = [&](float* to, float x) { *to = more ? *to + x : x; };
        int at_then = at;  // the addresses are formed here, not held through the rows
        asm volatile("" : "+v"(at_then));
        const int end = pieces * N + at_then;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int p = at_then + k * ROW;
            if (p >= pieces) continue;
#pragma unroll
            for (int j = 0; j < N; ++j) add(mine + p * N + j, aw[k][j]), add(mine + a.cols + p * N + j, ab[k][j]);
        }
        if (at_then < tail) add(mine + end, ew), add(mine + a.cols + end, eb);
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * WALKS;
    GradRow<T, PER, ADD> next;
    int64_t r0 = static_cast<int64_t>(blockIdx.x) * WALKS;
    if (AHEAD) load_row<ROW, AHEAD>(a, r0 + walk, at, pieces, tail, next);
    for (int turn = 0, rows = 0; r0 < a.rows; r0 += step, turn ^= 1) {  // all walks take as many steps: a row behind the last one is zeros
        if (rows++ == MOST_CHAIN) {
            leave();
            more = true, rows = 1, ew = eb = 0.0f;
#pragma unroll
            for (int k = 0; k < PER; ++k)
#pragma unroll
                for (int j = 0; j < N; ++j) aw[k][j] = ab[k][j] = 0.0f;
        }
        const int64_t r = r0 + walk;
        if (!AHEAD) load_row<ROW, AHEAD>(a, r, at, pieces, tail, next);
        const GradRow<T, PER, ADD> c = next;
        if (AHEAD && r0 + step < a.rows) load_row<ROW, AHEAD>(a, r + step, at, pieces, tail, next);
        const float u = (c.edge_h - c.mean) * c.rstd;
        float s1 = c.edge_dy * edge_w, s2 = s1 * u;
        ew = fmaf(c.edge_dy, u, ew), eb += c.edge_dy;  // nothing where there is no edge: dy is zero there
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            float d[N];
            int i = 0;
            c.dy[k].each([&](float e) { d[i++] = e; });
            i = 0;
            c.h[k].each([&](float e) {
                const float v = (e - c.mean) * c.rstd, du = d[i] * w[k][i];
                aw[k][i] = fmaf(d[i], v, aw[k][i]), ab[k][i] += d[i];
                s1 += du, s2 = fmaf(du, v, s2);
                ++i;
            });
        }
        const float m1 = row_total<WAVES>(s1, sh[turn][0][walk]) * per_col, m2 = row_total<WAVES>(s2, sh[turn][1][walk]) * per_col;
        if (r >= a.rows) continue;
        T* dx = static_cast<T*>(a.dx) + r * a.cols;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int p = at + k * ROW;
            if (p >= pieces) continue;
            float v[N], add[N] = {};
            int i = 0;
            c.h[k].each([&](float e) { v[i++] = (e - c.mean) * c.rstd; });
            if constexpr (ADD) {
                i = 0;
                const Piece<T> dh = AHEAD ? c.dh[k] : load_any(static_cast<const T*>(a.dh) + r * a.lddh + p * N);
                dh.each([&](float e) { add[i++] = e; });
            }
            store_piece<false>(dx + p * N, c.dy[k].map([&](int j, float e) { return fmaf(c.rstd, fmaf(e, w[k][j], -m1) - v[j] * m2, add[j]); }));
        }
        if (at < tail) put(dx, end, fmaf(c.rstd, fmaf(c.edge_dy, edge_w, -m1) - u * m2, c.edge_dh));
    }
    leave();
    if constexpr (WALKS > 1) {
        __syncthreads();
        for (int j = tid; j < 2 * a.cols; j += ROW * WALKS) {
            float s = sums[j];
#pragma unroll
            for (int k = 1; k < WALKS; ++k) s += sums[k * 2 * a.cols + j];
            part[j] = s;
        }
    }
}

// Rows that no workgroup holds: dx from two readings, and the columns' sums from a third, an element at a time: 2000 rows of 20000 columns in bf16 110 us, 2.2 TB/s of the 240 MB that have to
// go by, in fp32 195 us, 2.5 TB/s.
template <typename T, bool ADD>
__global__ __launch_bounds__(LONG_NT) void norm_grad_long(NormGrad a) {
    constexpr int WAVES = LONG_NT / 64;
    __shared__ float sh[2][WAVES];
    const int64_t r = blockIdx.x;
    const T *dy = static_cast<const T*>(a.dy) + r * a.lddy, *h = static_cast<const T*>(a.h) + r * a.ldh, *dh = static_cast<const T*>(a.dh) + (ADD ? r * a.lddh : 0);
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s1 = 0.0f, s2 = 0.0f;
    for (int j = threadIdx.x; j < a.cols; j += LONG_NT) {
        const float du = elem(dy, j) * a.w[j];
        s1 += du, s2 = fmaf(du, (elem(h, j) - mean) * rstd, s2);
    }
    const float m1 = row_total<WAVES>(s1, sh[0]) / a.cols, m2 = row_total<WAVES>(s2, sh[1]) / a.cols;
    T* dx = static_cast<T*>(a.dx) + r * a.cols;
    for (int j = threadIdx.x; j < a.cols; j += LONG_NT)
        put(dx, j, fmaf(rstd, fmaf(elem(dy, j), a.w[j], -m1) - (elem(h, j) - mean) * rstd * m2, ADD ? elem(dh, j) : 0.0f));
}
template <typename T>
__global__ __launch_bounds__(256) void norm_columns(NormGrad a) {
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j >= a.cols) return;
    float w = 0.0f, b = 0.0f;
    for (int64_t r = blockIdx.y; r < a.rows;) {  // 64 rows at a time: a term goes through 64 additions and a few, however many rows there are
        float pw = 0.0f, pb = 0.0f;
        for (int i = 0; i < 64 && r < a.rows; ++i, r += gridDim.y) {
            const float d = elem(static_cast<const T*>(a.dy), r * a.lddy + j);
            pw = fmaf(d, (elem(static_cast<const T*>(a.h), r * a.ldh + j) - a.mean[r]) * a.rstd[r], pw), pb += d;
        }
        w += pw, b += pb;
    }
    float* part = a.parts + static_cast<int64_t>(blockIdx.y) * 2 * a.cols;
    part[j] = w, part[a.cols + j] = b;
}

// 64 columns of the workgroups' sums to a workgroup, sixteen threads to a column.
__global__ __launch_bounds__(1024) void norm_sums(const float* parts, int count, int cols, float* dw, float* db) {
    __shared__ float sh[16][64];
    const int lane = threadIdx.x & 63, g = threadIdx.x >> 6, j = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (j < 2 * cols) {
#pragma unroll 8
        for (int p = g; p < count; p += 16) s += parts[static_cast<int64_t>(p) * 2 * cols + j];
    }
    sh[g][lane] = s;
    __syncthreads();
    if (g != 0 || j >= 2 * cols) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) s += sh[i][lane];
    (j < cols ? dw[j] : db[j - cols]) = s;
}

// ---- launches ----

constexpr int HELD_COLS = 16384;  // what the backward keeps of a row, and its sums, in registers
// How many wavefronts the backward gives a row, and how many rows a workgroup has side by side.
int grad_walks(int64_t cols) { return cols <= 1024 ? 4 : cols <= 2048 ? 2 : 1; }
// Workgroups of the backward, each with sums of its own: one on a CU, two of narrow rows, whose loads are few. More of them leave more sums than they save waiting: 16384 rows of 4096 columns
// in bf16, with dh, take 100 us with 256 workgroups, 110 with 512 and 117 with 768 (128: 149); 65536 rows of 512 columns without 59, 43 and 43.
int64_t grad_parts(int64_t rows, int64_t cols) {
    if (cols > HELD_COLS) return std::min<int64_t>(rows, 64);
    const int64_t walks = grad_walks(cols);
    return std::min<int64_t>((rows + walks - 1) / walks, cols <= 1024 ? 512 : 256);
}
// Up to 2048 columns a wavefront holds a row, then four, then sixteen of them: the fewest that have the registers, but for few rows. 8192 rows of 2048 in bf16 take 21.3 us with one wavefront
// and 21.8 with four; 4096 of 4096 columns 21.8 and 22.1, 16 of them 6.0 and 3.9.
template <typename T, bool RESIDUAL>
void launch_norm(const Norm& a, hipStream_t st) {
    constexpr int F = 8 / Piece<T>::N;  // fp32 takes twice the pieces
    const dim3 four(static_cast<unsigned>((a.rows + 3) / 4)), one(static_cast<unsigned>(a.rows));
    if (a.cols <= 512) return norm_held<T, 1, F, RESIDUAL><<<four, 256, 0, st>>>(a);
    if (a.cols <= 1024) return norm_held<T, 1, 2 * F, RESIDUAL><<<four, 256, 0, st>>>(a);
    if (a.cols <= 2048) return norm_held<T, 1, 4 * F, RESIDUAL><<<four, 256, 0, st>>>(a);
    if (a.cols <= 8192) return norm_held<T, 4, 4 * F, RESIDUAL><<<one, 256, 0, st>>>(a);
    if (a.cols <= 32768) return norm_held<T, 16, 4 * F, RESIDUAL><<<one, 1024, 0, st>>>(a);
    norm_long<T, RESIDUAL><<<one, LONG_NT, 0, st>>>(a);
}
// Half of the columns that the forward gives a wavefront, since it has their sums too: 8192 rows of 2048 take 31.2 us with two wavefronts and 34.4 with four.
template <typename T, bool ADD>
void launch_norm_grad(const NormGrad& a, int64_t parts, hipStream_t st) {
    constexpr int F = 8 / Piece<T>::N;
    const dim3 grid(static_cast<unsigned>(parts));
    const size_t lds = sizeof(float) * 2 * a.cols * grad_walks(a.cols);
    if (a.cols <= 512) return norm_grad<T, 1, F, 4, ADD, true><<<grid, 256, lds, st>>>(a);
    if (a.cols <= 1024) return norm_grad<T, 1, 2 * F, 4, ADD, true><<<grid, 256, lds, st>>>(a);
    if (a.cols <= 2048) return norm_grad<T, 2, 2 * F, 2, ADD, true><<<grid, 256, lds, st>>>(a);
    if (a.cols <= 4096) return norm_grad<T, 4, 2 * F, 1, ADD, true><<<grid, 256, 0, st>>>(a);
    if (a.cols <= 8192) return norm_grad<T, 8, 2 * F, 1, ADD, true><<<grid, 512, 0, st>>>(a);
    if (a.cols <= HELD_COLS) return norm_grad<T, 16, 2 * F, 1, ADD, false><<<grid, 1024, 0, st>>>(a);
    norm_grad_long<T, ADD><<<dim3(static_cast<unsigned>(a.rows)), LONG_NT, 0, st>>>(a);
    norm_columns<T><<<dim3(static_cast<unsigned>((a.cols + 255) / 256), static_cast<unsigned>(parts)), 256, 0, st>>>(a);
}

constexpr int64_t MOST_ROWS = 1 << 22;  // a launch has fewer than 2^32 threads, 1024 for a row at most

int check(const char* who, const pk_norm_shape* s) {
    const std::string w(who);
    if (!s) return fail(PK_ERR_ARGUMENT, w + ": null pointer");
    if (s->rows < 0 || s->rows >= MOST_ROWS || s->cols < 1 || s->cols > (1 << 24)) return fail(PK_ERR_SHAPE, w + ": shape mismatch (rows or columns out of range)");
    if (!known_dtype(s->dtype)) return fail(PK_ERR_ARGUMENT, w + ": dtype must be PK_F32 or PK_BF16");
    return PK_OK;
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" {

int pk_layernorm_fwd(const pk_norm_shape* s, const void* x, int64_t ldx, const void* residual, int64_t ldr, const float* w, const float* b, float eps, void* y,
                     void* h, float* mean, float* rstd, void* stream) {
    return c_entry([&] {
        const std::string who = "pk_layernorm_fwd";
        if (int rc = check(who.c_str(), s)) return rc;
        if (ldx < 0 || ldr < 0) return fail(PK_ERR_SHAPE, who + ": shape mismatch (a row stride is negative)");
        if (!(eps >= 0.0f) || std::isinf(eps)) return fail(PK_ERR_ARGUMENT, who + ": eps must be a number that is not negative");
        if (!residual != !h) return fail(PK_ERR_ARGUMENT, who + ": h is written where there is a residual, and only there");
        if (s->rows == 0) return static_cast<int>(PK_OK);
        if (!x || !w || !y || !mean || !rstd) return fail(PK_ERR_ARGUMENT, who + ": null pointer");
        const int64_t es = elem_size(s->dtype), R = s->rows, C = s->cols;
        if (!clear_of_all({Span(y, C, R, C, es), Span(h, C, R, C, es), Span(mean, 1, R, 1, 4), Span(rstd, 1, R, 1, 4)},
                          {Span(x, ldx, R, C, es), Span(residual, ldr, R, C, es), Span(w, 0, 1, C, 4), Span(b, 0, 1, C, 4)}))
            return fail(PK_ERR_ARGUMENT, who + ": a result overlaps another tensor of the call");
        touch({x, residual, w, b, y, h, mean, rstd}, stream);
        const Norm a{x, residual, ldx, ldr, R, w, b, y, h, mean, rstd, static_cast<int>(C), eps};
        hipStream_t st = static_cast<hipStream_t>(stream);
        if (s->dtype == PK_BF16)
            residual ? launch_norm<uint16_t, true>(a, st) : launch_norm<uint16_t, false>(a, st);
        else
            residual ? launch_norm<float, true>(a, st) : launch_norm<float, false>(a, st);
        return launched();
    });
}

size_t pk_layernorm_bwd_workspace_bytes(const pk_norm_shape* s) {
    if (!s || s->rows < 0 || s->rows >= MOST_ROWS || s->cols < 1 || s->cols > (1 << 24)) return 0;
    return sizeof(float) * 2 * static_cast<size_t>(s->cols) * static_cast<size_t>(grad_parts(s->rows, s->cols));
}

int pk_layernorm_bwd(const pk_norm_shape* s, const void* dy, int64_t lddy, const void* h, int64_t ldh, const void* dh, int64_t lddh, const float* w, const float* mean,
                     const float* rstd, void* dx, float* dw, float* db, void* workspace, size_t workspace_bytes, void* stream) {
    return c_entry([&] {
        const std::string who = "pk_layernorm_bwd";
        if (int rc = check(who.c_str(), s)) return rc;
        if (lddy < 0 || ldh < 0 || lddh < 0) return fail(PK_ERR_SHAPE, who + ": shape mismatch (a row stride is negative)");
        const int64_t es = elem_size(s->dtype), R = s->rows, C = s->cols;
        if (!dw || !db || (R > 0 && (!dy || !h || !w || !mean || !rstd || !dx))) return fail(PK_ERR_ARGUMENT, who + ": null pointer");
        const size_t need = pk_layernorm_bwd_workspace_bytes(s);
        if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 4)))
            return fail(PK_ERR_WORKSPACE, who + ": workspace too small (pk_layernorm_bwd_workspace_bytes)");
        if (!clear_of_all({Span(dx, C, R, C, es), Span(dw, 0, 1, C, 4), Span(db, 0, 1, C, 4), Span(need ? workspace : nullptr, 0, 1, static_cast<int64_t>(need), 1)},
                          {Span(dy, lddy, R, C, es), Span(h, ldh, R, C, es), Span(dh, lddh, R, C, es), Span(w, 0, 1, C, 4), Span(mean, 1, R, 1, 4), Span(rstd, 1, R, 1, 4)}))
            return fail(PK_ERR_ARGUMENT, who + ": a result overlaps another tensor of the call");
        touch({dy, h, dh, w, mean, rstd, dx, dw, db, workspace}, stream);
        const int64_t parts = grad_parts(R, C);
        const NormGrad a{dy, h, dh, lddy, ldh, lddh, R, w, mean, rstd, dx, static_cast<float*>(workspace), static_cast<int>(C)};
        hipStream_t st = static_cast<hipStream_t>(stream);
        if (R > 0) {
            if (s->dtype == PK_BF16)
                dh ? launch_norm_grad<uint16_t, true>(a, parts, st) : launch_norm_grad<uint16_t, false>(a, parts, st);
            else
                dh ? launch_norm_grad<float, true>(a, parts, st) : launch_norm_grad<float, false>(a, parts, st);
            if (int rc = launched()) return rc;
        }
        norm_sums<<<dim3(static_cast<unsigned>((2 * C + 63) / 64)), 1024, 0, st>>>(a.parts, static_cast<int>(parts), static_cast<int>(C), dw, db);
        return launched();
    });
}

}  // extern "C"
