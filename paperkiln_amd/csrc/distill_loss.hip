// Distillation from a teacher's top logits: loss, and gradient by the student's logits, in one pass over them.
//
//   p_k = exp(t_k / tau - log of the sum over the row's slots, or the teacher's own)     q = softmax(z / tau)     P = sum_k p_k
//   KL = sum_k p_k (log p_k - log q_{i_k})     loss = tau^2 sum_r w_r KL_r     dz_j = upstream w tau (P q_j - sum of p_k over the slots with i_k = j)
//
// What bounds it: memory, the student's logits read and their gradient written; the teacher has a few words for a row. A workgroup holds a row in registers, so that
// the gradient leaves in the pass that reads it. The words of the teacher are read beside the row and written over behind it: every word's element once more, by the
// thread of its slot. Log-probabilities are formed and added up in 64 bits, since the loss is a difference of near numbers.
#include "rows.h"

#include <algorithm>

namespace pk {
namespace {

constexpr int MOST_TOP = 1024;
struct Distill {
    const void* logits;
    void* dlogits;  // null: the loss alone
    int64_t ld, dld, rows;
    const int* indices;  // [rows][top], a negative one is an empty slot
    const float *teacher, *teacher_lse, *weights;  // teacher_lse may be null
    float* kl;
    double* row_loss;
    int vocab, top;
    float scale;  // 1 / tau
    double per_tau, s2, per_s2;
    float s2_hi, s2_lo;
    double tau;
    float upstream;
};

// The teacher's side of a row, `top` values each in LDS: a slot's word, the student's logit there, the teacher's logit and later its probability.
struct Slots {
    int* at;
    float *z, *p;
};
__device__ inline Slots slots_in(float* lds, int top) { return Slots{reinterpret_cast<int*>(lds), lds + top, lds + 2 * top}; }

template <typename T>
__device__ inline void read_slots(const Distill& a, int64_t r, const T* x, const Slots& s, int n) {
    for (int k = threadIdx.x; k < a.top; k += n) {
        const int i = a.indices[r * a.top + k];
        s.at[k] = i;
        s.z[k] = i < 0 ? 0.0f : i < a.vocab ? elem(x, i) : NAN;  // a word that is none has no probability
        s.p[k] = a.teacher[r * a.top + k];
    }
}
struct Row {
    float top, per_sum, coef, sum_p;  // coef: upstream w tau; 0 where there is nothing to learn from the row
    __device__ float power(float x, float s2) const { return __builtin_amdgcn_exp2f((x - top) * s2); }
};
__device__ inline double wave_max(double x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = fmax(x, __shfl_xor(x, o));
    return x;
}
// A wavefront: the slots' probabilities in place of the teacher's logits, the row's loss, and what its gradient is made of. Every lane has the same.
__device__ inline Row finish(const Distill& a, int64_t r, const Slots& s, const RowSum& sum) {
    const int lane = threadIdx.x & 63;
    const double per = a.per_tau;
    double lse;
    int words = 0;
    for (int k = lane; k < a.top; k += 64) words += s.at[k] >= 0;
    if (!__ballot(words != 0)) {
        if (lane == 0) a.kl[r] = 0.0f, a.row_loss[r] = 0.0;
        return Row{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if (a.teacher_lse) {
        lse = a.teacher_lse[r];
    } else {
        double high = -INFINITY, all = 0.0;
        for (int k = lane; k < a.top; k += 64)
            if (s.at[k] >= 0) high = fmax(high, s.p[k] * per);
        high = wave_max(high);
        for (int k = lane; k < a.top; k += 64)
            if (s.at[k] >= 0) all += exp(s.p[k] * per - high);
        lse = high + log(lanes_sum(all));  // no slot with a probability: no number
    }
    double kl = 0.0, mass = 0.0;
    for (int k = lane; k < a.top; k += 64) {
        double p = 0.0;
        if (s.at[k] >= 0) {
            const double logp = s.p[k] * per - lse, logq = ((static_cast<double>(s.z[k]) - static_cast<double>(sum.top)) * a.s2 - sum.log2) * LN2;
            p = exp(logp);
            if (p != 0.0) kl += p * (logp - logq);  // a word that the teacher rules out adds nothing, also where the student does
        }
        s.p[k] = static_cast<float>(p);
        mass += p;
    }
    kl = lanes_sum(kl), mass = lanes_sum(mass);
    const double w = a.weights[r], tau = a.tau;
    if (lane == 0) {
        a.kl[r] = static_cast<float>(kl);
        a.row_loss[r] = w * tau * tau * kl;
    }
    return Row{sum.top, static_cast<float>(exp2(-sum.log2)), static_cast<float>(w * tau * a.upstream), static_cast<float>(mass)};
}
// The teacher's words written over, by the threads of a workgroup. A word that several slots name gets all of theirs, from each of them the same value.
template <typename T>
__device__ inline void write_slots(const Distill& a, T* dx, const Slots& s, const Row& o, float s2, int n) {
    for (int k = threadIdx.x; k < a.top; k += n) {
        const int i = s.at[k];
        if (i < 0 || i >= a.vocab) continue;
        float p = 0.0f;
        for (int j = 0; j < a.top; ++j) p += s.at[j] == i ? s.p[j] : 0.0f;
        put(dx, i, o.coef * fmaf(o.sum_p * o.per_sum, o.power(s.z[k], s2), -p));
    }
}

// ROW_NT threads hold a row, PER pieces each.
template <typename T, int ROW_NT, int PER, bool PAST, bool GRAD>
__global__ __launch_bounds__(ROW_NT) void distill_held(Distill a) {
    constexpr int WAVES = ROW_NT / 64, N = Piece<T>::N;
    __shared__ float sh_m[WAVES];
    __shared__ double sh_s[WAVES];
    __shared__ Row sh_o;
    extern __shared__ float lds[];
    const Slots slots = slots_in(lds, a.top);
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, V = a.vocab;
    const T* x = static_cast<const T*>(a.logits) + r * a.ld;
    T* dx = GRAD ? static_cast<T*>(a.dlogits) + r * a.dld : nullptr;
    const Cut<T> cut(x, V);
    if (a.weights[r] == 0.0f) {
        if (tid == 0) a.kl[r] = 0.0f, a.row_loss[r] = 0.0;
        if (GRAD) zero_row<T, ROW_NT, PAST>(dx, cut, tid);
        return;
    }
    Piece<T> held[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int p = tid + k * ROW_NT;
        held[k] = p < cut.pieces ? load_piece<PAST>(x + cut.head + p * N) : Piece<T>::nothing();
    }
    const float edge = tid < cut.edges ? elem(x, cut.edge(tid)) : -INFINITY;
    read_slots(a, r, x, slots, ROW_NT);
    float m = edge;
#pragma unroll
    for (int k = 0; k < PER; ++k) held[k].each([&](float v) { m = fmaxf(m, v); });
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float ref = m == -INFINITY ? 0.0f : m;
    float first = power_of(a, edge, ref);
    keep_packed(held);
#pragma unroll
    for (int k = 0; k < PER; ++k) held[k].each([&](float v) { first += power_of(a, v, ref); });
    double s = group_sum<64>(first);
    if (s != 0.0 && s < 1.25) {  // one word has most of it: what the others have is kept in 64 bits
        s = power_of(a, edge, ref);
        keep_packed(held);
#pragma unroll
        for (int k = 0; k < PER; ++k) held[k].each([&](float v) { s += power_of(a, v, ref); });
        s = lanes_sum(s);
    }
    if ((tid & 63) == 0) sh_m[tid >> 6] = s == 0.0 ? -INFINITY : ref, sh_s[tid >> 6] = s;
    __syncthreads();
    if (tid < 64) {
        const Row o = finish(a, r, slots, sum_of_row(a, sh_m, sh_s));
        if (tid == 0) sh_o = o;
    }
    if constexpr (GRAD) {
        __syncthreads();
        const Row o = sh_o;
        if (o.coef == 0.0f) return zero_row<T, ROW_NT, PAST>(dx, cut, tid);
        const float s2 = a.scale * LOG2E, c = o.coef * o.sum_p * o.per_sum;
        keep_packed(held);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int p = tid + k * ROW_NT;
            if (p < cut.pieces) store_piece<PAST>(dx + cut.head + p * N, held[k].map([&](int, float v) { return c * o.power(v, s2); }));
        }
        if (tid < cut.edges) put(dx, cut.edge(tid), c * o.power(edge, s2));
        __syncthreads();  // the row is there before its words are written over
        write_slots(a, dx, slots, o, s2, ROW_NT);
    }
}

// Rows that no workgroup holds: read in strides with a running maximum and sum, and again for the gradient.
constexpr int LONG_NT = 1024;
template <typename T, bool PAST, bool GRAD>
__global__ __launch_bounds__(LONG_NT) void distill_long(Distill a) {
    constexpr int WAVES = LONG_NT / 64, N = Piece<T>::N;
    __shared__ float sh_m[WAVES];
    __shared__ double sh_s[WAVES];
    __shared__ Row sh_o;
    extern __shared__ float lds[];
    const Slots slots = slots_in(lds, a.top);
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(a.logits) + r * a.ld;
    T* dx = GRAD ? static_cast<T*>(a.dlogits) + r * a.dld : nullptr;
    const Cut<T> cut(x, a.vocab);
    if (a.weights[r] == 0.0f) {
        if (tid == 0) a.kl[r] = 0.0f, a.row_loss[r] = 0.0;
        if (GRAD) zero_row<T, LONG_NT, PAST>(dx, cut, tid);
        return;
    }
    const float edge = tid < cut.edges ? elem(x, cut.edge(tid)) : -INFINITY;
    read_slots(a, r, x, slots, LONG_NT);
    running<T, LONG_NT>(a, x, cut, 0, cut.pieces, edge, sh_m, sh_s);
    if (tid < 64) {
        const Row o = finish(a, r, slots, sum_of_row(a, sh_m, sh_s));
        if (tid == 0) sh_o = o;
    }
    if constexpr (GRAD) {
        __syncthreads();
        const Row o = sh_o;
        if (o.coef == 0.0f) return zero_row<T, LONG_NT, PAST>(dx, cut, tid);
        const float s2 = a.scale * LOG2E, c = o.coef * o.sum_p * o.per_sum;
        for (int p = tid; p < cut.pieces; p += LONG_NT) {
            const int j0 = cut.head + p * N;
            store_piece<PAST>(dx + j0, load_piece<PAST>(x + j0).map([&](int, float v) { return c * o.power(v, s2); }));
        }
        if (tid < cut.edges) put(dx, cut.edge(tid), c * o.power(edge, s2));
        __syncthreads();
        write_slots(a, dx, slots, o, s2, LONG_NT);
    }
}

// The rows' losses in a fixed order.
__global__ __launch_bounds__(1024) void distill_sum(const double* x, int64_t n, float* out) {
    const double s = sum_of<1024>(x, n);
    if (threadIdx.x == 0) *out = static_cast<float>(s);
}

// ---- launches ----

// From here on logits and gradient do not stay in the 256 MB of the last-level cache together (as for the losses on log-probabilities).
constexpr int64_t PAST_BYTES = int64_t{96} << 20;
template <typename T, bool PAST, bool GRAD>
void launch_held(const Distill& a, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(a.rows));
    const int pieces = a.vocab / Piece<T>::N;
    const size_t lds = 12 * static_cast<size_t>(a.top);
    if (pieces <= 64) return distill_held<T, 64, 1, PAST, GRAD><<<grid, 64, lds, st>>>(a);
    if (pieces <= 128) return distill_held<T, 64, 2, PAST, GRAD><<<grid, 64, lds, st>>>(a);
    if (pieces <= 256) return distill_held<T, 64, 4, PAST, GRAD><<<grid, 64, lds, st>>>(a);
    if (pieces <= 512) return distill_held<T, 128, 4, PAST, GRAD><<<grid, 128, lds, st>>>(a);
    if (pieces <= 1024) return distill_held<T, 256, 4, PAST, GRAD><<<grid, 256, lds, st>>>(a);
    if (pieces <= 2048) return distill_held<T, 512, 4, PAST, GRAD><<<grid, 512, lds, st>>>(a);
    if (pieces <= 4096) return distill_held<T, 512, 8, PAST, GRAD><<<grid, 512, lds, st>>>(a);
    if (pieces <= 8192) return distill_held<T, 1024, 8, PAST, GRAD><<<grid, 1024, lds, st>>>(a);
    distill_long<T, PAST, GRAD><<<grid, LONG_NT, lds, st>>>(a);
}
template <typename T>
void launch_distill(const Distill& a, hipStream_t st) {
    if (!a.dlogits) return launch_held<T, false, false>(a, st);
    a.rows * a.vocab * static_cast<int64_t>(sizeof(T)) >= PAST_BYTES ? launch_held<T, true, true>(a, st) : launch_held<T, false, true>(a, st);
}
constexpr int64_t MOST_ROWS = (1 << 22) - 2;  // a launch has fewer than 2^32 threads, 1024 for a row at most

bool clear_of(const void* p, int64_t bytes, const void* q, int64_t more) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
    return !q || x + static_cast<uintptr_t>(bytes) <= y || y + static_cast<uintptr_t>(more) <= x;
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" int pk_distill_loss(const pk_distill_config* c, const void* logits, int64_t ld, const int* indices, const float* teacher, const float* teacher_lse,
                               const float* weights, int64_t rows, int64_t vocab, int64_t top, void* dlogits, int64_t dld, float* kl, double* row_loss, float* loss,
                               int dtype, void* stream) {
    return c_entry([&] {
        const std::string who = "pk_distill_loss";
        if (!c || !loss) return fail(PK_ERR_ARGUMENT, who + ": null pointer");
        if (rows < 0 || rows > MOST_ROWS || vocab < 1 || vocab > (1 << 30)) return fail(PK_ERR_SHAPE, who + ": shape mismatch (rows or vocabulary out of range)");
        if (top < 1 || top > MOST_TOP) return fail(PK_ERR_SHAPE, who + ": shape mismatch (1 to 1024 words of the teacher for a row)");
        if (!known_dtype(dtype)) return fail(PK_ERR_ARGUMENT, who + ": dtype must be PK_F32 or PK_BF16");
        if (!(c->temperature >= 0x1p-20 && c->temperature <= 0x1p20)) return fail(PK_ERR_ARGUMENT, who + ": temperature must lie between 2^-20 and 2^20");
        if (!std::isfinite(c->upstream)) return fail(PK_ERR_ARGUMENT, who + ": upstream must be finite");
        if (ld < 0 || (dlogits && rows > 1 && dld < vocab)) return fail(PK_ERR_SHAPE, who + ": rows of logits overlap");
        if (rows > 0 && (!logits || !indices || !teacher || !weights || !kl || !row_loss)) return fail(PK_ERR_ARGUMENT, who + ": null pointer");
        const int64_t es = elem_size(dtype), read = rows ? ((rows - 1) * ld + vocab) * es : 0, written = rows ? ((rows - 1) * dld + vocab) * es : 0;
        if (dlogits && rows > 0) {
            if (!(dlogits == logits && (ld == dld || rows == 1)) && !clear_of(dlogits, written, logits, read))
                return fail(PK_ERR_ARGUMENT, who + ": dlogits may lie where the logits do, row for row, or clear of them");
            if (!clear_of(dlogits, written, indices, 4 * rows * top) || !clear_of(dlogits, written, teacher, 4 * rows * top) ||
                !clear_of(dlogits, written, teacher_lse, 4 * rows) || !clear_of(dlogits, written, weights, 4 * rows))
                return fail(PK_ERR_ARGUMENT, who + ": dlogits overlap the teacher's tensors or the weights");
        }
        touch({logits, indices, teacher, teacher_lse, weights, dlogits, kl, row_loss, loss}, stream);
        hipStream_t st = static_cast<hipStream_t>(stream);
        Distill a{};
        a.logits = logits, a.dlogits = dlogits, a.ld = ld, a.dld = dld, a.rows = rows, a.indices = indices, a.teacher = teacher, a.teacher_lse = teacher_lse;
        a.weights = weights, a.kl = kl, a.row_loss = row_loss, a.vocab = static_cast<int>(vocab), a.top = static_cast<int>(top);
        a.tau = c->temperature, a.upstream = c->upstream;
        a.per_tau = 1.0 / c->temperature;
        set_scale(a, a.per_tau);
        if (rows > 0) {
            dtype == PK_BF16 ? launch_distill<uint16_t>(a, st) : launch_distill<float>(a, st);
            if (int rc = launched()) return rc;
        }
        distill_sum<<<1, 1024, 0, st>>>(row_loss, rows, loss);
        return launched();
    });
}
