// Queries and keys on their way into attention: every head's row normalised by its root mean square, multiplied by a weight of the head size and
// turned pair by pair by its token's position, in one pass over both tensors, and the gradients of that.
//
//   r = 1 / sqrt(mean_j x_j^2 + eps)      u_j = x_j r w_j      (y_a, y_b) = (u_a cos t - u_b sin t, u_a sin t + u_b cos t),  t = pos theta^(-2i/R)
//   du = y's gradient turned back         dw_j = sum over rows of du_j x_j r       dx_j = r (w_j du_j - x_j r^2 mean_i(w_i du_i x_i))
//
// What bounds it: memory. The forward reads and writes each element once, the backward reads two and writes one; r is formed again there instead of
// being kept, because the row is in registers anyway. The angle is formed in 64 bits, in turns, and its whole turns are dropped there: at position
// 10^6 an angle in 32 bits is 0.06 rad off.
#include "post.h"

namespace pk {
namespace {

constexpr int MAX_DK = 256, MAX_PAIRS = MAX_DK / 2, NT = 256, WAVES = NT / 64;

struct Rows {  // one [B, T, H, dk] tensor
    const void* p;
    int64_t sb, st, sh;
};
struct RowsOut {
    void* p;
    int64_t sb, st, sh;
};
struct Qk {
    Rows x[2], dy[2];     // queries, keys
    RowsOut y[2];         // forward: y; backward: dx
    const float* w[2];
    const int* pos;
    int64_t pos_sb;
    float* part;          // backward: a workgroup's sums of dw, queries' then keys'
    int B, T, Hq, Hkv, dk, rotary, halves;
    float eps;
    double turns[MAX_PAIRS];  // turns a position moves each pair by: theta^(-2i/R) / 2 pi
};

// cos and sin of a position's angle
template <bool FINE>
__device__ inline void cos_sin(int pos, double turns, float& c, float& s) {
    const double t = pos * turns;
    const float f = static_cast<float>(t - rint(t));  // -1/2 .. 1/2 of a turn
    sincospif(2.0f * f, &s, &c);
}

// The two columns of pair p: of the first `rotary` ones neighbours, or one from each half; behind them neighbours, which are not turned.
__device__ inline void columns(int p, int rotary, bool halves, int& a, int& b) {
    const bool turned = halves && p < rotary / 2;
    a = turned ? p : 2 * p;
    b = turned ? p + rotary / 2 : 2 * p + 1;
}

// Any even head size, any strides: a wavefront takes a row, a lane its pairs lane and lane + 64.
template <typename T>
__global__ __launch_bounds__(NT) void qk_fwd_any(Qk a) {
    const int lane = threadIdx.x & 63, heads = a.Hq + a.Hkv, pairs = a.dk / 2;
    const int64_t items = static_cast<int64_t>(a.B) * a.T * heads, stride = static_cast<int64_t>(gridDim.x) * WAVES;
    for (int64_t item = blockIdx.x * static_cast<int64_t>(WAVES) + (threadIdx.x >> 6); item < items; item += stride) {
        const int64_t token = item / heads;
        const int head = static_cast<int>(item - token * heads), which = head >= a.Hq, h = which ? head - a.Hq : head;
        const int64_t b = token / a.T, t = token - b * a.T;
        const T* x = static_cast<const T*>(a.x[which].p) + b * a.x[which].sb + t * a.x[which].st + h * a.x[which].sh;
        T* y = static_cast<T*>(a.y[which].p) + b * a.y[which].sb + t * a.y[which].st + h * a.y[which].sh;
        const int pos = a.pos[b * a.pos_sb + t];
        float xa[2], xb[2], ss = 0.0f;
        int ca[2], cb[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int p = lane + 64 * k;
            xa[k] = xb[k] = 0.0f;
            columns(p, a.rotary, a.halves, ca[k], cb[k]);
            if (p < pairs) xa[k] = elem(x, ca[k]), xb[k] = elem(x, cb[k]);
            ss += xa[k] * xa[k] + xb[k] * xb[k];
        }
        const float r = 1.0f / sqrtf(group_sum<64>(ss) / static_cast<float>(a.dk) + a.eps);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int p = lane + 64 * k;
            if (p >= pairs) continue;
            const float ua = xa[k] * r * a.w[which][ca[k]], ub = xb[k] * r * a.w[which][cb[k]];
            if (p < a.rotary / 2) {
                float c, s;
                cos_sin<true>(pos, a.turns[p], c, s);
                put(y, ca[k], ua * c - ub * s);
                put(y, cb[k], ua * s + ub * c);
            } else {
                put(y, ca[k], ua);
                put(y, cb[k], ub);
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(NT) void qk_bwd_any(Qk a) {
    __shared__ float sh[WAVES][2 * MAX_DK];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, heads = a.Hq + a.Hkv, pairs = a.dk / 2;
    const int64_t items = static_cast<int64_t>(a.B) * a.T * heads, stride = static_cast<int64_t>(gridDim.x) * WAVES;
    float dwa[2][2] = {}, dwb[2][2] = {};  // [queries, keys][pair]
    int ca[2], cb[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) columns(lane + 64 * k, a.rotary, a.halves, ca[k], cb[k]);
    for (int64_t item = blockIdx.x * static_cast<int64_t>(WAVES) + wave; item < items; item += stride) {
        const int64_t token = item / heads;
        const int head = static_cast<int>(item - token * heads), which = head >= a.Hq, h = which ? head - a.Hq : head;
        const int64_t b = token / a.T, t = token - b * a.T;
        const T* x = static_cast<const T*>(a.x[which].p) + b * a.x[which].sb + t * a.x[which].st + h * a.x[which].sh;
        const T* dy = static_cast<const T*>(a.dy[which].p) + b * a.dy[which].sb + t * a.dy[which].st + h * a.dy[which].sh;
        T* dx = static_cast<T*>(a.y[which].p) + b * a.y[which].sb + t * a.y[which].st + h * a.y[which].sh;
        const int pos = a.pos[b * a.pos_sb + t];
        float xa[2] = {}, xb[2] = {}, ga[2] = {}, gb[2] = {}, wa[2] = {}, wb[2] = {}, ss = 0.0f, sg = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int p = lane + 64 * k;
            if (p >= pairs) continue;
            xa[k] = elem(x, ca[k]), xb[k] = elem(x, cb[k]);
            wa[k] = a.w[which][ca[k]], wb[k] = a.w[which][cb[k]];
            const float da = elem(dy, ca[k]), db = elem(dy, cb[k]);
            ga[k] = da, gb[k] = db;
            if (p < a.rotary / 2) {
                float c, s;
                cos_sin<true>(pos, a.turns[p], c, s);
                ga[k] = da * c + db * s;
                gb[k] = db * c - da * s;
            }
            ss += xa[k] * xa[k] + xb[k] * xb[k];
            sg += wa[k] * ga[k] * xa[k] + wb[k] * gb[k] * xb[k];
        }
        const float n = static_cast<float>(a.dk);
        const float r = 1.0f / sqrtf(group_sum<64>(ss) / n + a.eps), m = r * r * (group_sum<64>(sg) / n);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (which) {
                dwa[1][k] += ga[k] * xa[k] * r, dwb[1][k] += gb[k] * xb[k] * r;
            } else {
                dwa[0][k] += ga[k] * xa[k] * r, dwb[0][k] += gb[k] * xb[k] * r;
            }
            if (lane + 64 * k >= pairs) continue;
            put(dx, ca[k], r * (wa[k] * ga[k] - xa[k] * m));
            put(dx, cb[k], r * (wb[k] * gb[k] - xb[k] * m));
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (lane + 64 * k >= pairs) continue;
        for (int which = 0; which < 2; ++which) {
            sh[wave][which * a.dk + ca[k]] = dwa[which][k];
            sh[wave][which * a.dk + cb[k]] = dwb[which][k];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.dk; i += NT) {
        float s = 0.0f;
        for (int w = 0; w < WAVES; ++w) s += sh[w][i];
        a.part[blockIdx.x * static_cast<int64_t>(2 * a.dk) + i] = s;
    }
}

// The workgroups' sums of dw added up in a fixed order: 16 columns to a workgroup, 16 of its threads to a column.
__global__ __launch_bounds__(NT) void qk_dw_sum(const float* part, int parts, int dk, float* dwq, float* dwk) {
    __shared__ float sh[16][17];
    const int c = threadIdx.x & 15, slice = threadIdx.x >> 4, col = static_cast<int>(blockIdx.x) * 16 + c;
    float s = 0.0f;
    if (col < 2 * dk)
        for (int i = slice; i < parts; i += 16) s += part[i * static_cast<int64_t>(2 * dk) + col];
    sh[slice][c] = s;
    __syncthreads();
    if (slice != 0 || col >= 2 * dk) return;
    s = 0.0f;
    for (int i = 0; i < 16; ++i) s += sh[i][c];
    (col < dk ? dwq[col] : dwk[col - dk]) = s;
}

int check(const pk_qk_shape* s, const char* who) {
    const std::string w(who);
    if (!s) return fail(PK_ERR_ARGUMENT, w + ": null shape");
    if (s->B < 0 || s->T < 0 || s->Hq <= 0 || s->Hkv <= 0) return fail(PK_ERR_SHAPE, w + ": shape mismatch (negative or empty dimension)");
    if (s->dk <= 0 || s->dk > MAX_DK || s->dk % 2) return fail(PK_ERR_SHAPE, w + ": head_dim must be even and at most 256");
    if (s->rotary < 0 || s->rotary > s->dk || s->rotary % 2) return fail(PK_ERR_SHAPE, w + ": rotary columns must be even and at most head_dim");
    if (!known_dtype(s->dtype)) return fail(PK_ERR_ARGUMENT, w + ": dtype must be PK_F32 or PK_BF16");
    if (!(s->theta > 0.0) || !std::isfinite(s->theta)) return fail(PK_ERR_ARGUMENT, w + ": theta must be positive");
    if (!(s->eps >= 0.0f) || !std::isfinite(s->eps)) return fail(PK_ERR_ARGUMENT, w + ": eps must not be negative");
    return PK_OK;
}
bool bad(const pk_tensor4* t) { return !t || !t->ptr; }

void fill(Qk& a, const pk_qk_shape* s) {
    a.B = s->B, a.T = s->T, a.Hq = s->Hq, a.Hkv = s->Hkv, a.dk = s->dk, a.rotary = s->rotary ? s->rotary : s->dk, a.halves = s->halves != 0;
    a.eps = s->eps, a.pos_sb = s->pos_stride_b, a.part = nullptr;
    for (int i = 0; i < MAX_PAIRS; ++i) a.turns[i] = i < a.rotary / 2 ? std::pow(s->theta, -2.0 * i / a.rotary) / 6.283185307179586476925 : 0.0;
}
Rows rows_of(const pk_tensor4* t) { return Rows{t->ptr, t->stride_b, t->stride_t, t->stride_h}; }
RowsOut out_of(const pk_tensor4* t) { return RowsOut{t->ptr, t->stride_b, t->stride_t, t->stride_h}; }

int64_t items_of(const pk_qk_shape* s) { return static_cast<int64_t>(s->B) * s->T * (s->Hq + s->Hkv); }
// workgroups of the backward, each of which leaves sums of dw: enough to fill the chip several times over
int bwd_groups(const pk_qk_shape* s) {
    const int64_t want = (items_of(s) + WAVES - 1) / WAVES;
    return static_cast<int>(want < 1 ? 1 : want > 1024 ? 1024 : want);
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" {

int pk_qk_norm_rope_fwd(const pk_qk_shape* s, const pk_tensor4* q, const pk_tensor4* k, const float* wq, const float* wk, const int* pos,
                        const pk_tensor4* yq, const pk_tensor4* yk, void* stream) {
    return c_entry([&] {
        if (int rc = check(s, "pk_qk_norm_rope_fwd")) return rc;
        if (static_cast<int64_t>(s->B) * s->T == 0) return static_cast<int>(PK_OK);
        if (bad(q) || bad(k) || bad(yq) || bad(yk) || !wq || !wk || !pos) return fail(PK_ERR_ARGUMENT, "pk_qk_norm_rope_fwd: null tensor");
        Qk a;
        fill(a, s);
        a.x[0] = rows_of(q), a.x[1] = rows_of(k), a.y[0] = out_of(yq), a.y[1] = out_of(yk), a.dy[0] = a.dy[1] = Rows{nullptr, 0, 0, 0};
        a.w[0] = wq, a.w[1] = wk, a.pos = pos;
        const void* used[] = {q->ptr, k->ptr, yq->ptr, yk->ptr, wq, wk, pos};
        for (const void* p : used) dev_touch(p, stream);
        const int64_t want = (items_of(s) + WAVES - 1) / WAVES;
        const dim3 grid(static_cast<unsigned>(want < 65536 ? want : 65536));
        hipStream_t st = static_cast<hipStream_t>(stream);
        if (s->dtype == PK_BF16)
            qk_fwd_any<uint16_t><<<grid, NT, 0, st>>>(a);
        else
            qk_fwd_any<float><<<grid, NT, 0, st>>>(a);
        return launched();
    });
}

size_t pk_qk_norm_rope_bwd_workspace_bytes(const pk_qk_shape* s) {
    if (check(s, "pk_qk_norm_rope_bwd_workspace_bytes")) return 0;
    return sizeof(float) * static_cast<size_t>(bwd_groups(s)) * 2 * s->dk;
}

int pk_qk_norm_rope_bwd(const pk_qk_shape* s, const pk_tensor4* dyq, const pk_tensor4* dyk, const pk_tensor4* q, const pk_tensor4* k, const float* wq,
                        const float* wk, const int* pos, const pk_tensor4* dq, const pk_tensor4* dk, float* dwq, float* dwk, void* workspace,
                        size_t workspace_bytes, void* stream) {
    return c_entry([&] {
        if (int rc = check(s, "pk_qk_norm_rope_bwd")) return rc;
        if (!wq || !wk || !dwq || !dwk) return fail(PK_ERR_ARGUMENT, "pk_qk_norm_rope_bwd: null tensor");
        const bool none = static_cast<int64_t>(s->B) * s->T == 0;
        if (!none && (bad(dyq) || bad(dyk) || bad(q) || bad(k) || bad(dq) || bad(dk) || !pos)) return fail(PK_ERR_ARGUMENT, "pk_qk_norm_rope_bwd: null tensor");
        if (!workspace || workspace_bytes < pk_qk_norm_rope_bwd_workspace_bytes(s) || !aligned(workspace, 4))
            return fail(PK_ERR_WORKSPACE, "pk_qk_norm_rope_bwd: workspace too small (pk_qk_norm_rope_bwd_workspace_bytes)");
        hipStream_t st = static_cast<hipStream_t>(stream);
        Qk a;
        fill(a, s);
        a.part = static_cast<float*>(workspace);
        a.w[0] = wq, a.w[1] = wk, a.pos = pos;
        const int groups = bwd_groups(s);
        for (const void* p : {static_cast<const void*>(wq), static_cast<const void*>(wk), static_cast<const void*>(dwq), static_cast<const void*>(dwk),
                              static_cast<const void*>(pos), static_cast<const void*>(workspace)})
            dev_touch(p, stream);
        if (!none) {
            a.x[0] = rows_of(q), a.x[1] = rows_of(k), a.dy[0] = rows_of(dyq), a.dy[1] = rows_of(dyk), a.y[0] = out_of(dq), a.y[1] = out_of(dk);
            const void* used[] = {q->ptr, k->ptr, dyq->ptr, dyk->ptr, dq->ptr, dk->ptr};
            for (const void* p : used) dev_touch(p, stream);
            if (s->dtype == PK_BF16)
                qk_bwd_any<uint16_t><<<dim3(groups), NT, 0, st>>>(a);
            else
                qk_bwd_any<float><<<dim3(groups), NT, 0, st>>>(a);
            if (int rc = launched()) return rc;
        }
        qk_dw_sum<<<dim3((2 * s->dk + 15) / 16), NT, 0, st>>>(a.part, none ? 0 : groups, s->dk, dwq, dwk);
        return launched();
    });
}

}  // extern "C"
