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

// The teacher's side of a row in LDS: a slot's word, the student's logit there, the teacher's logit and its probability. Four arrays of whole 16 bytes; what completes them is empty.
struct Slots {
    int* at;
    float *z, *t, *p;
    int count;
};
__host__ __device__ constexpr int pitch_of(int top) { return (top + 3) & ~3; }
__device__ inline Slots slots_in(float* lds, int top) {
    const int n = pitch_of(top);
    return Slots{reinterpret_cast<int*>(lds), lds + n, lds + 2 * n, lds + 3 * n, n};
}
// A thread's first slot, asked for before the row is: the teacher's part is done while the row is on its way.
struct Slot {
    int at;
    float t;
};
__device__ inline Slot slot(const Distill& a, int64_t r, int k) { return k < a.top ? Slot{a.indices[r * a.top + k], a.teacher[r * a.top + k]} : Slot{-1, 0.0f}; }
// The words and logits of the teacher, and the student's logits but for the first slots', which are the result.
template <typename T>
__device__ inline float put_slots(const Distill& a, int64_t r, const T* x, const Slots& s, Slot first, int n) {
    const auto logit = [&](int i) { return i < 0 ? 0.0f : i < a.vocab ? elem(x, i) : NAN; };  // a word that is none has no probability
    const int k0 = threadIdx.x;
    if (k0 < s.count) s.at[k0] = first.at, s.t[k0] = first.t;
    for (int k = k0 + n; k < s.count; k += n) {
        const Slot o = slot(a, r, k);
        s.at[k] = o.at, s.t[k] = o.t, s.z[k] = logit(o.at);
    }
    return logit(first.at);
}
// What a row's gradient needs of its teacher.
struct Teacher {
    double lse;
    float mass;  // the sum of the slots' probabilities
    int words;   // 0: there is nothing to learn from the row
};
__device__ inline double wave_max(double x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = fmax(x, __shfl_xor(x, o));
    return x;
}
// A wavefront: the slots' probabilities. Every lane has the result.
__device__ inline Teacher teacher_of(const Distill& a, int64_t r, const Slots& s) {
    const int lane = threadIdx.x & 63;
    const double per = a.per_tau;
    int words = 0;
    for (int k = lane; k < s.count; k += 64) words += s.at[k] >= 0;
    if (!__ballot(words != 0)) return Teacher{0.0, 0.0f, 0};
    double lse;
    if (a.teacher_lse) {
        lse = a.teacher_lse[r];
    } else {
        double high = -INFINITY, all = 0.0;
        for (int k = lane; k < s.count; k += 64)
            if (s.at[k] >= 0) high = fmax(high, s.t[k] * per);
        high = wave_max(high);
        for (int k = lane; k < s.count; k += 64)
            if (s.at[k] >= 0) all += exp(s.t[k] * per - high);
        lse = high + log(lanes_sum(all));  // no slot with a probability: no number
    }
    double mass = 0.0;
    for (int k = lane; k < s.count; k += 64) {
        const double p = s.at[k] >= 0 ? exp(s.t[k] * per - lse) : 0.0;
        s.p[k] = static_cast<float>(p);
        mass += s.at[k] >= a.vocab && p != 0.0 ? NAN : p;  // a word that is none: the row has no gradient either
    }
    return Teacher{lse, static_cast<float>(lanes_sum(mass)), 1};
}
// A wavefront, when the row is known: its loss. The probabilities are formed again in 64 bits, since the loss is a difference.
__device__ inline void finish(const Distill& a, int64_t r, const Slots& s, const Teacher& t, const RowTotal& total) {
    const int lane = threadIdx.x & 63;
    double kl = 0.0;
    if (t.words) {
        const RowSum sum = row_sum(total.top, total.sum);
        for (int k = lane; k < s.count; k += 64)
            if (s.at[k] >= 0) {
                const double logp = s.t[k] * a.per_tau - t.lse, logq = ((static_cast<double>(s.z[k]) - static_cast<double>(sum.top)) * a.s2 - sum.log2) * LN2;
                const double p = exp(logp);
                if (p != 0.0) kl += p * (logp - logq);  // a word that the teacher rules out adds nothing, also where the student does
            }
        kl = lanes_sum(kl);
    }
    if (lane == 0) {
        a.kl[r] = static_cast<float>(kl);
        a.row_loss[r] = t.words ? a.weights[r] * a.tau * a.tau * kl : 0.0;
    }
}
struct Row {
    float top, coef, even;  // coef: upstream w tau, 0 where there is nothing to learn from the row; even: what every word's probability is multiplied by
};
__device__ inline Row row_of(const Distill& a, double w, float mass, int words, const RowTotal& t) {
    if (!words) return Row{0.0f, 0.0f, 0.0f};
    const float coef = static_cast<float>(w * a.tau * a.upstream), per_sum = t.sum == 0.0 ? NAN : static_cast<float>(1.0 / t.sum);
    return Row{t.top, coef, mass * per_sum};
}
// The teacher's words written over, by the threads of a workgroup. A word that several slots name gets all of theirs, from each of them the same value.
template <typename T>
__device__ inline void write_slots(const Distill& a, T* dx, const Slots& s, const Row& o, int n) {
    for (int k = threadIdx.x; k < a.top; k += n) {
        const int i = s.at[k];
        if (i < 0 || i >= a.vocab) continue;
        float p = 0.0f;
        for (int j = 0; j < s.count; j += 4) {
            const int4 at = *reinterpret_cast<const int4*>(s.at + j);
            const float4 more = *reinterpret_cast<const float4*>(s.p + j);
            p += at.x == i ? more.x : 0.0f, p += at.y == i ? more.y : 0.0f, p += at.z == i ? more.z : 0.0f, p += at.w == i ? more.w : 0.0f;
        }
        put(dx, i, o.coef * fmaf(o.even, power_of(a, s.z[k], o.top), -p));
    }
}

// ROW_NT threads hold a row, PER pieces each.
template <typename T, int ROW_NT, int PER, bool PAST, bool GRAD>
__global__ __launch_bounds__(ROW_NT) void distill_held(Distill a) {
    constexpr int WAVES = ROW_NT / 64, N = Piece<T>::N;
    __shared__ float sh_m[WAVES];
    __shared__ double sh_s[WAVES];
    __shared__ float sh_mass;
    __shared__ int sh_words;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const Slots slots = slots_in(lds, a.top);
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, V = a.vocab;
    const T* x = static_cast<const T*>(a.logits) + r * a.ld;
    T* dx = GRAD ? static_cast<T*>(a.dlogits) + r * a.dld : nullptr;
    const Cut<T> cut(x, V);
    const Slot mine = slot(a, r, tid);
    const float w = a.weights[r];
    if (w == 0.0f) {
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
    const float z = put_slots(a, r, x, slots, mine, ROW_NT);
    Teacher teacher;
    if constexpr (GRAD) {
        __syncthreads();
        if (tid < 64) {
            teacher = teacher_of(a, r, slots);
            if (tid == 0) sh_mass = teacher.mass, sh_words = teacher.words;
        }
        keep_packed(held);
    }
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
    if (tid < slots.count) slots.z[tid] = z;
    __syncthreads();
    if constexpr (GRAD) {
        const RowTotal total = total_of_row(a, sh_m, sh_s);
        const Row o = row_of(a, w, sh_mass, sh_words, total);
        if (o.coef == 0.0f) {
            zero_row<T, ROW_NT, PAST>(dx, cut, tid);
        } else {
            const float c = o.coef * o.even;
            keep_packed(held);
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const int p = tid + k * ROW_NT;
                if (p < cut.pieces) store_piece<PAST>(dx + cut.head + p * N, held[k].map([&](int, float v) { return c * power_of(a, v, o.top); }));
            }
            if (tid < cut.edges) put(dx, cut.edge(tid), c * power_of(a, edge, o.top));
            __syncthreads();  // the row is there before its words are written over
            write_slots(a, dx, slots, o, ROW_NT);
        }
        if (tid < 64) finish(a, r, slots, teacher, total);
    } else if (tid < 64) {  // beside the row the teacher's part would take registers past the 64 with which 1024 threads are on a CU twice
        teacher = teacher_of(a, r, slots);
        finish(a, r, slots, teacher, total_of_row(a, sh_m, sh_s));
    }
}

// Rows that no workgroup holds: read in strides with a running maximum and sum, and again for the gradient.
constexpr int LONG_NT = 1024;
template <typename T, bool PAST, bool GRAD>
__global__ __launch_bounds__(LONG_NT) void distill_long(Distill a) {
    constexpr int WAVES = LONG_NT / 64, N = Piece<T>::N;
    __shared__ float sh_m[WAVES];
    __shared__ double sh_s[WAVES];
    __shared__ float sh_mass;
    __shared__ int sh_words;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const Slots slots = slots_in(lds, a.top);
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(a.logits) + r * a.ld;
    T* dx = GRAD ? static_cast<T*>(a.dlogits) + r * a.dld : nullptr;
    const Cut<T> cut(x, a.vocab);
    const Slot mine = slot(a, r, tid);
    const float w = a.weights[r];
    if (w == 0.0f) {
        if (tid == 0) a.kl[r] = 0.0f, a.row_loss[r] = 0.0;
        if (GRAD) zero_row<T, LONG_NT, PAST>(dx, cut, tid);
        return;
    }
    const float edge = tid < cut.edges ? elem(x, cut.edge(tid)) : -INFINITY;
    const float z = put_slots(a, r, x, slots, mine, LONG_NT);
    if (tid < slots.count) slots.z[tid] = z;
    running<T, LONG_NT>(a, x, cut, 0, cut.pieces, edge, sh_m, sh_s);  // its end waits for all
    Teacher teacher;
    if (tid < 64) {
        teacher = teacher_of(a, r, slots);
        if (tid == 0) sh_mass = teacher.mass, sh_words = teacher.words;
    }
    __syncthreads();
    const RowTotal total = total_of_row(a, sh_m, sh_s);
    if constexpr (GRAD) {
        const Row o = row_of(a, w, sh_mass, sh_words, total);
        if (o.coef == 0.0f) {
            zero_row<T, LONG_NT, PAST>(dx, cut, tid);
        } else {
            const float c = o.coef * o.even;
            for (int p = tid; p < cut.pieces; p += LONG_NT) {
                const int j0 = cut.head + p * N;
                store_piece<PAST>(dx + j0, load_piece<PAST>(x + j0).map([&](int, float v) { return c * power_of(a, v, o.top); }));
            }
            if (tid < cut.edges) put(dx, cut.edge(tid), c * power_of(a, edge, o.top));
            __syncthreads();
            write_slots(a, dx, slots, o, LONG_NT);
        }
    }
    if (tid < 64) finish(a, r, slots, teacher, total);
}

// The rows' losses in a fixed order.
__global__ __launch_bounds__(1024) void distill_sum(const double* x, int64_t n, float* out) {
    const double s = sum_of<1024>(x, n);
    if (threadIdx.x == 0) *out = static_cast<float>(s);
}

// ---- launches ----

// From here on logits and gradient do not stay in the 256 MB of the last-level cache together, and go past it: 8192 rows of 32000 in bf16 200 us, 213 through it; 8192 of 2000 (31 MB) 28.7
// and 26.8; between 60 and 96 MB it is level.
constexpr int64_t PAST_BYTES = int64_t{96} << 20;
// A row to as few threads as hold it in eight pieces each, in four where a wavefront or a few of them do: what is done once for a row is done by fewer. 8192 rows of 32000 in bf16: 200 us with
// 512 threads of eight pieces, 307 with 1024 of four; 8192 of 2000: 26.7 with a wavefront, 33.7 with four; 4096 of 8000: 38.2 with 256 of four, 39.9 with 128 of eight.
template <typename T, bool PAST, bool GRAD>
void launch_held(const Distill& a, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(a.rows));
    const int pieces = a.vocab / Piece<T>::N;
    const size_t lds = 16 * static_cast<size_t>(pitch_of(a.top));
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
        if (!aligned(row_loss, 8)) return fail(PK_ERR_ARGUMENT, who + ": row_loss must be aligned to 8 bytes");
        if (rows > 0) {
            const int64_t es = elem_size(dtype);
            const Span read(logits, ld, rows, vocab, es), written(dlogits, dld, rows, vocab, es);
            if (written.meets(read) && !(dlogits == logits && (ld == dld || rows == 1)))
                return fail(PK_ERR_ARGUMENT, who + ": dlogits may lie where the logits do, row for row, or clear of them");
            const Span out_kl(kl, 1, rows, 1, 4), out_rows(row_loss, 1, rows, 1, 8), out_loss(loss, 0, 1, 1, 4);
            if (read.meets(out_kl) || read.meets(out_rows) || read.meets(out_loss) ||
                !clear_of_all({written, out_kl, out_rows, out_loss},
                              {Span(indices, top, rows, top, 4), Span(teacher, top, rows, top, 4), Span(teacher_lse, 1, rows, 1, 4), Span(weights, 1, rows, 1, 4)}))
                return fail(PK_ERR_ARGUMENT, who + ": a result overlaps another tensor of the call");
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
