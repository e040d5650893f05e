// Log-probabilities of chosen tokens from a model's logits, their gradient, and the two losses that are built on them.
//
//   z = scale * logits     lse = log sum_j exp z_j     logp = z_t - lse     d logp / d logits_j = scale ([j = t] - exp(z_j - lse))
//   policy:      rho = exp(logp - old);  L = -min(rho A, clamp(rho, 1 - lo, 1 + hi) A) + kl (exp(d) - d - 1), d = ref - logp;  loss = sum_r w_r L_r
//                dL/dlogp = -(rho A where rho A <= clamp(rho) A, else 0) + kl (1 - exp d)
//   preference:  s = sum over a sequence's rows of logp - ref;  u = beta (s_chosen - s_rejected);  loss = mean over pairs of
//                -(1 - e) log sigma(u) - e log sigma(-u);  dL/du = e sigma(u) - (1 - e) sigma(-u)
//
// What bounds it: memory, the logits read and their gradient written. A policy row's coefficient depends on its own row only, so its gradient leaves
// in the pass that reads it (but for a few long rows, which several workgroups read). A preference row's depends on both sequences of its pair, so the logits are read twice.
// Exponentials are taken in base 2 against the largest logit; sums are in 32 bits inside a wavefront, where no word has most of it, and in 64 across them, and a token's
// log-probability, a difference of near numbers, is formed in 64, and stays there, or in two numbers of 32, until it has been added to its loss.
#include "post.h"

#include <algorithm>

namespace pk {
namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr double LN2 = 0.693147180559945309417;

struct Loss {
    const void* logits;
    void* dlogits;
    int64_t ld, dld, rows;
    const int* targets;
    int vocab;
    float scale;
    double s2;                // scale * log2(e), and as a sum of two 32-bit numbers, both of them positive
    float s2_hi, s2_lo;
    double per_s2;            // 1 / s2
    float *logp, *lse;        // written; lse may be null
    float* low;               // LOGP: what the log-probability is beyond its 32 bits, or null
    float2* sums;             // written unless null; GRAD: the rows' sums, or null and lse_in instead
    float* clear;             // LOGP: a word per row to set to zero, or null
    const float *lse_in, *coef;  // GRAD
    const double* losses;     // GRAD: the pairs' or rows' losses, whose sum over `divisor` the workgroup behind the last row's writes to `loss`
    int64_t terms;
    double divisor;
    float* loss;
    float2* parts;            // LOGP: room for the parts of rows that are dealt out, or null
    const float *old_logp, *ref_logp, *adv, *weights;  // POLICY; ref_logp may be null
    double* row_loss;
    float* coef_out;  // POLICY, a row that is dealt out: what its gradient is multiplied by
    int64_t coef_step;  // words from one row's to the next one's, in coef and coef_out
    float clip_low, clip_high, kl, upstream;
};
enum Mode { LOGP, GRAD, POLICY };

// 2^(s2 (x - m)). The difference is taken before the product, so a row of the type's lowest value has its probabilities too. The exponent from both parts of s2: rounded to 32
// bits it would turn every row's log-probability by up to 6e-8 times its logits, always the same way, and a preference loss adds up hundreds of them (margins
// 4e-7 off, 1e-7 so). A logit of -inf stays one: the low part is not zero nor negative.
__device__ inline float power_of(const Loss& a, float x, float m) {
    const float d = x - m;
    return __builtin_amdgcn_exp2f(fmaf(d, a.s2_hi, d * a.s2_lo));
}
void set_scale(Loss& a, float scale) {
    a.scale = scale;
    a.s2 = static_cast<double>(scale) * 1.4426950408889634074;
    a.per_s2 = 1.0 / a.s2;
    a.s2_hi = static_cast<float>(a.s2);
    if (static_cast<double>(a.s2_hi) >= a.s2) a.s2_hi = std::nextafter(a.s2_hi, 0.0f);
    a.s2_lo = static_cast<float>(a.s2 - static_cast<double>(a.s2_hi));
}

// A policy row's loss and the derivative of it by the row's log-probability, both before the row's weight.
__device__ inline void policy_row(const Loss& a, int64_t r, double logp, double& loss, double& slope) {
    const double adv = a.adv[r], ratio = exp(logp - static_cast<double>(a.old_logp[r]));
    const double held = fmin(fmax(ratio, 1.0 - static_cast<double>(a.clip_low)), 1.0 + static_cast<double>(a.clip_high));
    const double free_ = ratio * adv, stop = held * adv;
    const bool open = !(free_ > stop);  // a ratio that is no number stays one
    loss = -(open ? free_ : stop);
    slope = open ? -free_ : 0.0;
    if (a.ref_logp) {
        const double d = static_cast<double>(a.ref_logp[r]) - logp, e = exp(d);
        loss += a.kl * (e - d - 1.0);
        slope += a.kl * (1.0 - e);
    }
}

// n values added up in 64 bits in a fixed order by a workgroup, eight loads of a thread on their way together; the sum in its first thread.
template <int NT>
__device__ inline double sum_of(const double* x, int64_t n) {
    __shared__ double sh[NT / 64];
    double s = 0.0;
    for (int64_t i0 = threadIdx.x; i0 < n; i0 += 8 * NT) {
        double v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = i0 + k * NT < n ? x[i0 + k * NT] : 0.0;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += v[k];
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    s = sh[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) s += sh[w];
    return s;
}
template <int NT>
__device__ inline void losses_sum(const Loss& a) {
    const double s = sum_of<NT>(a.losses, a.terms);
    if (threadIdx.x == 0) *a.loss = static_cast<float>(s / a.divisor);
}

// x added up over the wavefront's lanes, the sum in every one, by group_sum's moves.
__device__ inline double lanes_sum(double x) {
    const auto words = [](uint32_t lo, uint32_t hi) { return __longlong_as_double(static_cast<int64_t>(lo) | static_cast<int64_t>(hi) << 32); };
    const auto lo = [](double v) { return static_cast<uint32_t>(__double_as_longlong(v)); };
    const auto hi = [](double v) { return static_cast<uint32_t>(__double_as_longlong(v) >> 32); };
    const auto l32 = __builtin_amdgcn_permlane32_swap(lo(x), lo(x), false, false), h32 = __builtin_amdgcn_permlane32_swap(hi(x), hi(x), false, false);
    x = words(l32[0], h32[0]) + words(l32[1], h32[1]);
    const auto l16 = __builtin_amdgcn_permlane16_swap(lo(x), lo(x), false, false), h16 = __builtin_amdgcn_permlane16_swap(hi(x), hi(x), false, false);
    x = words(l16[0], h16[0]) + words(l16[1], h16[1]);
    const auto moved = [&](auto ctrl) {
        constexpr int C = decltype(ctrl)::value;
        return words(__builtin_amdgcn_update_dpp(0, lo(x), C, 0xf, 0xf, true), __builtin_amdgcn_update_dpp(0, hi(x), C, 0xf, 0xf, true));
    };
    x += moved(std::integral_constant<int, 0x128>{});
    x += moved(std::integral_constant<int, 0x141>{});
    x += moved(std::integral_constant<int, 0x4E>{});
    return x + moved(std::integral_constant<int, 0xB1>{});
}

// log2 of the sum of 2^(s2 x) over a row: s2 top + log2. Its two parts stay apart, since their sum, in 32 bits, knows the second one no more where logits are large; each by itself
// may go through 32 bits from one launch to another: top is a logit, log2 that of the vocabulary's size at most.
struct RowSum {
    float top;
    double log2;
};
__device__ inline RowSum row_sum(float top, double sum) { return RowSum{top, sum == 0.0 ? static_cast<double>(NAN) : log2(sum)}; }  // a row without a word has no probabilities
// From what each wavefront has: the logit that it took its exponentials against and their sum; one without a word has none to scale.
template <int WAVES>
__device__ inline RowSum sum_of_row(const Loss& a, const float (&m)[WAVES], const double (&s)[WAVES]) {
    float top = m[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, m[w]);
    double sum = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += s[w] == 0.0 ? 0.0 : s[w] * power_of(a, m[w], top);
    return row_sum(top, sum);
}

// What a row's gradient is made of once its sum is known: -coef 2^(s2 (x - top) - log2), and the target's element.
struct RowOut {
    float top, log2, coef, target;
    __device__ float probability(float x, float s2) const { return __builtin_amdgcn_exp2f(fmaf(x - top, s2, -log2)); }
    __device__ float other(float x, float s2) const { return -coef * probability(x, s2); }
};
template <Mode MODE>
__device__ inline RowOut finish(const Loss& a, int64_t r, float xt, const RowSum& sum, bool writes = true) {
    const double logp = ((static_cast<double>(xt) - static_cast<double>(sum.top)) * a.s2 - sum.log2) * LN2;
    RowOut o{sum.top, static_cast<float>(sum.log2), 0.0f, 0.0f};
    double w = 0.0, loss = 0.0;
    if (MODE == POLICY) {
        double slope;
        policy_row(a, r, logp, loss, slope);
        w = a.weights[r];
        o.coef = static_cast<float>(w * slope * a.upstream * a.scale);
        if (writes && a.coef_out) a.coef_out[r * a.coef_step] = static_cast<float>(w * slope * a.upstream);
        o.target = o.coef * static_cast<float>(-expm1(logp));
    }
    if (writes) {
        if (MODE == POLICY) a.row_loss[r] = w * loss;
        const float high = static_cast<float>(logp);
        a.logp[r] = high;
        if (a.lse) a.lse[r] = static_cast<float>((static_cast<double>(sum.top) * a.s2 + sum.log2) * LN2);
        if (a.sums) a.sums[r] = make_float2(o.top, o.log2);
        if (MODE == LOGP && a.low) a.low[r] = isfinite(high) ? static_cast<float>(logp - high) : 0.0f;
    }
    return o;
}
// GRAD: from a row's sum. The target's element, -coef expm1(log-probability), is as exact as that.
__device__ inline RowOut summed_row(const Loss& a, float coef, float xt, const RowSum& sum, bool word) {
    if (!word) coef = NAN;  // a token that is no word has no gradient
    const double logp = ((static_cast<double>(xt) - static_cast<double>(sum.top)) * a.s2 - sum.log2) * LN2;
    return RowOut{sum.top, static_cast<float>(sum.log2), coef, coef * -expm1f(static_cast<float>(logp))};
}
__device__ inline RowOut known_row(const Loss& a, int64_t r, float coef, bool word) {
    if (!word) coef = NAN;
    const float2 sum = a.sums[r];
    return RowOut{sum.x, sum.y, coef, coef * -expm1f(a.logp[r])};
}
// From the log of the sum in 32 bits, as a logit and what is beside it; without the target.
__device__ inline RowOut given_row(const Loss& a, float lse, float coef, bool word) {
    const double log2 = lse * (1.0 / LN2);
    const float top = static_cast<float>(log2 * a.per_s2);
    const auto scalar = [](float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); };  // a row's, so the workgroup's
    return RowOut{scalar(top), static_cast<float>(log2 - top * a.s2), scalar(word ? coef : NAN), 0.0f};
}
// What that log's rounding, 2^-24 of it, may turn an element by: 2^-17 of it in 32 bits, 2^-14 before a rounding to bf16. The others turn by as much as the sum, so past a log of 128 or
// 1024 the row is read once more for it (2048 rows of 32000 words bf16 54 us, up to there 45). The target, which has 1 - p of the coefficient, turns by as much of the whole
// coefficient: where 1 - p is small (under 0.08 or 0.01 at a log of 10) its element is what the others come to as they are written.
template <typename T>
constexpr float ALLOWED = sizeof(T) == 4 ? 0x1p-17f : 0x1p-14f;
template <typename T>
__device__ inline bool far(float lse) {
    return fabsf(lse) * 0x1p-24f > ALLOWED<T>;
}
template <typename T>
__device__ inline bool faint(float lse, float logp) {  // 1 - e^-x is 0.63 x or more up to x = 1, and more than 0.63 from there on
    return fabsf(lse) * 0x1p-24f > ALLOWED<T> * 0.63f * fminf(-logp, 1.0f);
}

// ---- rows in 16-byte pieces -------------------------------------------------------------------------------------------------
// A row is taken apart at 16-byte boundaries of its address: whole pieces, and the few elements in front of the first and behind the last one, which go to
// one thread each. So a row may begin anywhere, and the gradient's row anywhere else: the hardware stores a piece where its elements may lie.

template <typename T>
struct Piece;
template <>
struct Piece<uint16_t> {
    static constexpr int N = 8;
    u32x4 v;
    template <typename F>
    __device__ void each(F&& f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f(__uint_as_float(v[i] << 16));
            f(__uint_as_float(v[i] & 0xFFFF0000u));
        }
    }
    template <typename F>
    __device__ Piece map(F&& f) const {
        Piece r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[i] = pack_bf16(f(2 * i, __uint_as_float(v[i] << 16)), f(2 * i + 1, __uint_as_float(v[i] & 0xFFFF0000u)));
        return r;
    }
    __device__ static Piece nothing() { return Piece{{0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u}}; }
};
template <>
struct Piece<float> {
    static constexpr int N = 4;
    u32x4 v;
    template <typename F>
    __device__ void each(F&& f) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) f(__uint_as_float(v[i]));
    }
    template <typename F>
    __device__ Piece map(F&& f) const {
        Piece r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[i] = __float_as_uint(f(i, __uint_as_float(v[i])));
        return r;
    }
    __device__ static Piece nothing() { return Piece{{0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u}}; }
};
template <typename T>
struct Cut {  // a row's pieces
    int head, pieces, edges;
    __device__ Cut(const T* x, int V) {
        constexpr int N = Piece<T>::N;
        const int past = static_cast<int>(reinterpret_cast<uintptr_t>(x) / sizeof(T)) & (N - 1);
        head = min((N - past) & (N - 1), V);
        pieces = (V - head) / N;
        edges = V - pieces * N;
    }
    __device__ int edge(int i) const { return i < head ? i : i + pieces * Piece<T>::N; }
    // which of `threads`, dealt the pieces (from `from` on) in turn and the edges one each, holds word j; -1: none, as of a word that there is not
    __device__ int holder(int j, int threads, int from = 0) const {
        const int p = (j - head) / Piece<T>::N;
        if (j < head) return j;
        if (p >= pieces) return p > pieces || j - pieces * Piece<T>::N >= edges ? -1 : j - pieces * Piece<T>::N;
        return (p - from) % threads;
    }
};

// A piece read for the last time, or written, past the last-level cache or through it.
template <bool PAST, typename T>
__device__ inline Piece<T> load_piece(const T* x) {
    const u32x4* p = reinterpret_cast<const u32x4*>(x);
    if constexpr (PAST)
        return Piece<T>{__builtin_nontemporal_load(p)};
    else
        return Piece<T>{*p};
}
typedef u32x4 u32x4_any __attribute__((aligned(2)));
template <bool PAST, typename T>
__device__ inline void store_piece(T* x, const Piece<T>& v) {
    u32x4_any* p = reinterpret_cast<u32x4_any*>(x);
    if constexpr (PAST)
        __builtin_nontemporal_store(v.v, p);
    else
        *p = v.v;
}

// A row that does not count: not read, its results zeros.
template <Mode MODE>
__device__ inline void no_row(const Loss& a, int64_t r) {
    a.logp[r] = 0.0f;
    if (a.lse) a.lse[r] = 0.0f;
    if (MODE == POLICY) {
        a.row_loss[r] = 0.0;
        if (a.coef_out) a.coef_out[r * a.coef_step] = 0.0f;
    }
}
template <typename T, int NT, bool PAST>
__device__ inline void zero_row(T* dx, const Cut<T>& cut, int tid) {
    for (int p = tid; p < cut.pieces; p += NT) store_piece<PAST>(dx + cut.head + p * Piece<T>::N, Piece<T>{{0, 0, 0, 0}});
    if (tid < cut.edges) put(dx, cut.edge(tid), 0.0f);
}
// The gradient of a piece as if none of its words were the target; the thread that holds the target's piece writes that element over afterwards.
template <typename T>
__device__ inline Piece<T> gradient(const Piece<T>& x, float s2, const RowOut& o) {
    return x.map([&](int, float v) { return o.other(v, s2); });
}

// Between two walks over a row the pieces stay as they are: the compiler would keep every element of the first walk in a register of its own.
template <typename T, int PER>
__device__ inline void keep_packed(Piece<T> (&held)[PER]) {
    if constexpr (Piece<T>::N == 8) {
#pragma unroll
        for (int k = 0; k < PER; ++k) asm volatile("" : "+v"(held[k].v));
    }
}

// ROW_NT threads hold a row, PER pieces each, so that the logits are read once. One exchange through LDS joins the wavefronts; the first one works out the
// row's scalars in 64 bits and hands them round.
template <typename T, Mode MODE, int ROW_NT, int PER, bool PAST>
__global__ __launch_bounds__(ROW_NT) void rows_held(Loss a) {
    constexpr int WAVES = ROW_NT / 64, N = Piece<T>::N;
    __shared__ float sh_m[WAVES];
    __shared__ double sh_s[WAVES];
    __shared__ RowOut sh_o;
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, V = a.vocab, t = a.targets[r];
    const T* x = static_cast<const T*>(a.logits) + r * a.ld;
    T* dx = MODE == LOGP ? nullptr : static_cast<T*>(a.dlogits) + r * a.dld;
    const Cut<T> cut(x, V);
    if (MODE == LOGP && a.clear && tid == 0) a.clear[r] = 0.0f;
    if (t < 0 || (MODE == POLICY && a.weights[r] == 0.0f)) {
        if (tid == 0) no_row<MODE>(a, r);
        if (MODE != LOGP) zero_row<T, ROW_NT, PAST>(dx, cut, tid);
        return;
    }
    Piece<T> held[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int p = tid + k * ROW_NT;
        held[k] = p < cut.pieces ? load_piece<PAST>(x + cut.head + p * N) : Piece<T>::nothing();
    }
    const float edge = tid < cut.edges ? elem(x, cut.edge(tid)) : -INFINITY;
    const float xt = t < V ? elem(x, t) : NAN;  // read before the row is written over; a token that is no word has no probability
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
    // Where one word has most of the row its log-probability is little more than the sum's own rounding, 2^-24: added up in 64 bits then, which for every row would cost
    // the log-probabilities of 8192 x 32000 bf16 99.6 -> 111.8 us.
    if (s != 0.0 && s < 1.25) {
        s = power_of(a, edge, ref);
        keep_packed(held);
#pragma unroll
        for (int k = 0; k < PER; ++k) held[k].each([&](float v) { s += power_of(a, v, ref); });
        s = lanes_sum(s);
    }
    RowOut o;
    if constexpr (WAVES == 1) {
        o = finish<MODE>(a, r, xt, row_sum(ref, s), tid == 0);
    } else {
        if ((tid & 63) == 0) sh_m[tid >> 6] = s == 0.0 ? -INFINITY : ref, sh_s[tid >> 6] = s;
        __syncthreads();
        if (tid < 64) {
            o = finish<MODE>(a, r, xt, sum_of_row<WAVES>(a, sh_m, sh_s), tid == 0);
            if (tid == 0) sh_o = o;
        }
        if constexpr (MODE == LOGP) return;
        __syncthreads();
        o = sh_o;
    }
    if constexpr (MODE != LOGP) {
        if (o.coef == 0.0f) return zero_row<T, ROW_NT, PAST>(dx, cut, tid);  // clipped
        const float s2 = a.scale * LOG2E;
        keep_packed(held);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int p = tid + k * ROW_NT;
            if (p < cut.pieces) store_piece<PAST>(dx + cut.head + p * N, gradient(held[k], s2, o));
        }
        if (tid < cut.edges) put(dx, cut.edge(tid), o.other(edge, s2));
        if (tid == cut.holder(t, ROW_NT)) put(dx, t, o.target);
    }
}

// Rows that no workgroup holds are read in strides, with a running maximum and sum, and again for the gradient.
constexpr int LONG_U = 4;
template <typename T, int NT>
__device__ inline void running(const Loss& a, const T* x, const Cut<T>& cut, int from, int to, float edge, float* sh_m, double* sh_s) {
    constexpr int N = Piece<T>::N;
    const int tid = threadIdx.x;
    float m = edge;
    double s = edge == -INFINITY ? 0.0 : static_cast<double>(power_of(a, edge, edge));
    for (int p0 = from + tid; p0 < to; p0 += LONG_U * NT) {
        Piece<T> v[LONG_U];
#pragma unroll
        for (int u = 0; u < LONG_U; ++u) {
            const int p = p0 + u * NT;
            v[u] = p < to ? load_piece<false>(x + cut.head + p * N) : Piece<T>::nothing();
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < LONG_U; ++u) v[u].each([&](float y) { top = fmaxf(top, y); });
        const float ref = top == -INFINITY ? 0.0f : top;
        if (s != 0.0) s *= power_of(a, m, ref);
#pragma unroll
        for (int u = 0; u < LONG_U; ++u) v[u].each([&](float y) { s += power_of(a, y, ref); });
        m = top;
    }
    // lanes, then wavefronts
    float top = m;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    s = lanes_sum(s == 0.0 ? 0.0 : s * power_of(a, m, top));
    if ((tid & 63) == 0) sh_m[tid >> 6] = s == 0.0 ? -INFINITY : top, sh_s[tid >> 6] = s;
    __syncthreads();
}

constexpr int LONG_NT = 1024;
template <typename T, Mode MODE, bool PAST>
__global__ __launch_bounds__(LONG_NT) void rows_long(Loss a) {
    constexpr int WAVES = LONG_NT / 64, N = Piece<T>::N;
    __shared__ float sh_m[WAVES];
    __shared__ double sh_s[WAVES];
    __shared__ RowOut sh_o;
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, V = a.vocab, t = a.targets[r];
    const T* x = static_cast<const T*>(a.logits) + r * a.ld;
    T* dx = MODE == LOGP ? nullptr : static_cast<T*>(a.dlogits) + r * a.dld;
    const Cut<T> cut(x, V);
    if (MODE == LOGP && a.clear && tid == 0) a.clear[r] = 0.0f;
    if (t < 0 || (MODE == POLICY && a.weights[r] == 0.0f)) {
        if (tid == 0) no_row<MODE>(a, r);
        if (MODE != LOGP) zero_row<T, LONG_NT, PAST>(dx, cut, tid);
        return;
    }
    const float edge = tid < cut.edges ? elem(x, cut.edge(tid)) : -INFINITY, xt = t < V ? elem(x, t) : NAN;
    running<T, LONG_NT>(a, x, cut, 0, cut.pieces, edge, sh_m, sh_s);
    RowOut o;
    if (tid < 64) {
        o = finish<MODE>(a, r, xt, sum_of_row<WAVES>(a, sh_m, sh_s), tid == 0);
        if (tid == 0) sh_o = o;
    }
    if constexpr (MODE != LOGP) {
        __syncthreads();
        o = sh_o;
        if (o.coef == 0.0f) return zero_row<T, LONG_NT, PAST>(dx, cut, tid);
        const float s2 = a.scale * LOG2E;
        for (int p = tid; p < cut.pieces; p += LONG_NT) {
            const int j0 = cut.head + p * N;
            store_piece<PAST>(dx + j0, gradient(load_piece<PAST>(x + j0), s2, o));
        }
        if (tid < cut.edges) put(dx, cut.edge(tid), o.other(edge, s2));
        if (tid == cut.holder(t, LONG_NT)) put(dx, t, o.target);
    }
}

// A few such rows are dealt to several workgroups, `per` pieces each, which leave the largest logit and the sum of their part; a wavefront joins a row's.
constexpr int PART_NT = 512, MOST_PARTS = 32, FEW_ROWS = 128;
template <typename T, Mode MODE>
__global__ __launch_bounds__(PART_NT) void rows_part(Loss a, int per, float2* parts) {
    constexpr int WAVES = PART_NT / 64;
    __shared__ float sh_m[WAVES];
    __shared__ double sh_s[WAVES];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x;
    if (a.targets[r] < 0 || (MODE == POLICY && a.weights[r] == 0.0f)) return;
    const T* x = static_cast<const T*>(a.logits) + r * a.ld;
    const Cut<T> cut(x, a.vocab);
    const int from = static_cast<int>(blockIdx.y) * per, to = min(cut.pieces, from + per);
    const float edge = blockIdx.y == 0 && tid < cut.edges ? elem(x, cut.edge(tid)) : -INFINITY;
    running<T, PART_NT>(a, x, cut, from, to, edge, sh_m, sh_s);
    if (tid != 0) return;
    float top = sh_m[0];
    double s = 0.0;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, sh_m[w]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s += sh_s[w] == 0.0 ? 0.0 : sh_s[w] * power_of(a, sh_m[w], top);
    parts[r * gridDim.y + blockIdx.y] = make_float2(top, static_cast<float>(s - 1.0));  // the part's largest word is 1 of it: what the others are keeps its bits
}
template <typename T, Mode MODE>
__global__ __launch_bounds__(64) void rows_join(Loss a, int count, const float2* parts) {
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x, t = a.targets[r];
    if (a.clear && lane == 0) a.clear[r] = 0.0f;
    if (t < 0 || (MODE == POLICY && a.weights[r] == 0.0f)) {
        if (lane == 0) no_row<MODE>(a, r);
        return;
    }
    const float2 v = lane < count ? parts[r * count + lane] : make_float2(-INFINITY, -1.0f);
    float top = v.x;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    double sum = v.y == -1.0f ? 0.0 : (1.0 + v.y) * power_of(a, v.x, top);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    const T* x = static_cast<const T*>(a.logits) + r * a.ld;
    if (lane == 0) finish<MODE>(a, r, t < a.vocab ? elem(x, t) : NAN, row_sum(top, sum));
}

// ---- pairs of sequences -----------------------------------------------------------------------------------------------------
struct Pairs {
    const int* starts;  // 2 pairs + 1
    const int* targets;
    const float *logp, *low;  // a log-probability is their sum
    const float* ref;
    float *coef, *margins;
    double* losses;
    int64_t rows;
    int pairs;
    float beta, smoothing, upstream;
};
struct PairOut {
    double margin, loss;
    float slope;  // of the chosen answer's log-probability; the rejected one's is its negative
};
__device__ inline PairOut pair_terms(const Pairs& a, double chosen, double rejected) {
    const double u = a.beta * (chosen - rejected), e = a.smoothing;
    const double small = exp(-fabs(u)), up = 1.0 / (1.0 + small), down = small / (1.0 + small);  // sigma(|u|), sigma(-|u|)
    const double yes = u >= 0.0 ? up : down, no = u >= 0.0 ? down : up;                          // sigma(u), sigma(-u); no number stays none
    const double tail = log1p(small), lost_no = fmax(-u, 0.0) + tail, lost_yes = fmax(u, 0.0) + tail;  // -log sigma(u), -log sigma(-u)
    // a weight of zero drops its term, also an infinite one (a word without probability in an answer)
    return PairOut{u, u != u ? u : (e < 1.0 ? (1.0 - e) * lost_no : 0.0) + (e > 0.0 ? e * lost_yes : 0.0),
                   static_cast<float>((e * yes - (1.0 - e) * no) * a.beta * a.upstream / a.pairs)};
}
__device__ inline int64_t start_of(const Pairs& a, int seq) { return min(max(static_cast<int64_t>(a.starts[seq]), int64_t{0}), a.rows); }  // offsets that lie are held to the rows there are
// What a sequence's rows from `begin` on give to its sum, to lane l of n; U rows' loads on their way together.
template <int U>
__device__ inline double sequence_part(const Pairs& a, int64_t begin, int64_t end, int l, int n) {
    double s = 0.0;
    for (int64_t r0 = begin + l; r0 < end; r0 += U * n) {
        float logp[U], low[U], ref[U];
        bool counts[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int64_t r = min(r0 + k * n, end - 1);
            counts[k] = a.targets[r] >= 0 && r0 + k * n < end, logp[k] = a.logp[r], low[k] = a.low[r], ref[k] = a.ref[r];
        }
#pragma unroll
        for (int k = 0; k < U; ++k) s += counts[k] ? static_cast<double>(logp[k]) + low[k] - static_cast<double>(ref[k]) : 0.0;
    }
    return s;
}
__device__ inline double wave_sum(double s) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    return s;
}
// A few short pairs are formed by who wants them: a wavefront, or a workgroup.
__device__ inline PairOut pair_of_wave(const Pairs& a, int pair) {
    const int lane = threadIdx.x & 63;
    const double chosen = sequence_part<4>(a, start_of(a, pair), start_of(a, pair + 1), lane, 64);
    const double rejected = sequence_part<4>(a, start_of(a, a.pairs + pair), start_of(a, a.pairs + pair + 1), lane, 64);
    return pair_terms(a, wave_sum(chosen), wave_sum(rejected));
}
// Row r's sequence, or -1.
__device__ inline int sequence_of(const Pairs& a, int64_t r) {
    const int lane = threadIdx.x & 63;
    const uint64_t in = __ballot(lane < 2 * a.pairs && start_of(a, lane) <= r && r < start_of(a, lane < 2 * a.pairs ? lane + 1 : 0));
    return in ? 63 - __builtin_clzll(in) : -1;
}
template <int NT>
__device__ inline void few_pairs_mean(const Pairs& a, float* mean) {
    __shared__ double sh[NT / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double s = 0.0;
    for (int p = wave; p < a.pairs; p += NT / 64) {
        const PairOut o = pair_of_wave(a, p);
        if (lane == 0) a.margins[p] = static_cast<float>(o.margin);
        s += o.loss;
    }
    if (lane == 0) sh[wave] = s;
    __syncthreads();
    s = sh[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) s += sh[w];
    if (threadIdx.x == 0) *mean = static_cast<float>(s / a.pairs);
}

// ---- the gradient of rows whose sums are known --------------------------------------------------------------------------------
// Every element by itself, so a row may be dealt to several workgroups (grid.y, `per` pieces each) and written over.
// What they are known by: the log of the sum that a caller keeps (DEALT: and several workgroups take a row), or the sum itself; PAIRS: the sum, and the rows' coefficients are formed
// here, from the pairs.
enum Known { LSE, DEALT, SUMS, PAIRS };
constexpr int GRAD_U = 8;
template <typename T, int GRAD_NT, bool PAST, Known BY>
__global__ __launch_bounds__(GRAD_NT) void rows_grad(Loss a, int per, Pairs pairs) {
    constexpr int N = Piece<T>::N;
    __shared__ float sh_m[GRAD_NT / 64];
    __shared__ double sh_s[GRAD_NT / 64];
    if (blockIdx.x == a.rows) {
        if (blockIdx.y != 0) return;
        if constexpr (BY == PAIRS)
            few_pairs_mean<GRAD_NT>(pairs, a.loss);
        else
            losses_sum<GRAD_NT>(a);
        return;
    }
    const int64_t r = a.rows - 1 - blockIdx.x;  // the last rows first: they are what the pass before has left in the last-level cache
    const int tid = threadIdx.x, V = a.vocab, t = a.targets[r];
    const T* x = static_cast<const T*>(a.logits) + r * a.ld;
    T* dx = static_cast<T*>(a.dlogits) + r * a.dld;
    const Cut<T> cut(x, V);
    const int from = static_cast<int>(blockIdx.y) * per, to = min(cut.pieces, from + per);
    const bool edges = blockIdx.y == 0 && tid < cut.edges;
    float given = 0.0f;
    if constexpr (BY == PAIRS) {
        const int seq = t < 0 ? -1 : sequence_of(pairs, r);
        if (seq >= 0) {
            const bool rejected = seq >= pairs.pairs;
            const float slope = pair_of_wave(pairs, rejected ? seq - pairs.pairs : seq).slope;
            given = (rejected ? -slope : slope) * a.scale;
        }
    } else {
        given = a.coef[r * a.coef_step] * a.scale;
    }
    const float s2 = a.scale * LOG2E;
    if (t < 0 || given == 0.0f) {
        for (int p = from + tid; p < to; p += GRAD_NT) store_piece<PAST>(dx + cut.head + p * N, Piece<T>{{0, 0, 0, 0}});
        if (edges) put(dx, cut.edge(tid), 0.0f);
        return;
    }
    constexpr bool GIVEN = BY == LSE || BY == DEALT;
    const float lse = GIVEN ? a.lse_in[r] : 0.0f;
    if (GIVEN && far<T>(lse)) {  // one workgroup forms the sum again, before it writes over the row
        if (blockIdx.y != 0) return;
        const float edge = tid < cut.edges ? elem(x, cut.edge(tid)) : -INFINITY, xt = t < V ? elem(x, t) : NAN;
        running<T, GRAD_NT>(a, x, cut, 0, cut.pieces, edge, sh_m, sh_s);
        const RowOut o = summed_row(a, given, xt, sum_of_row<GRAD_NT / 64>(a, sh_m, sh_s), t < V);
        for (int p = tid; p < cut.pieces; p += GRAD_NT) store_piece<PAST>(dx + cut.head + p * N, gradient(load_piece<PAST>(x + cut.head + p * N), s2, o));
        if (tid < cut.edges) put(dx, cut.edge(tid), o.other(edge, s2));
        if (tid == cut.holder(t, GRAD_NT)) put(dx, t, o.target);
        return;
    }
    // the target's piece, or -1, and who holds its element; read before they are written over
    const int in_piece = t < V && t >= cut.head ? (t - cut.head) / N : -1, pt = in_piece < cut.pieces ? in_piece : -1, word = t - cut.head - pt * N;
    const bool held_here = pt >= 0 ? pt >= from && pt < to : blockIdx.y == 0, holds = held_here && tid == cut.holder(t, GRAD_NT, from);
    Piece<T> beside = Piece<T>::nothing();
    const bool all_know = GIVEN && GRAD_NT > 64 && t < V && a.dlogits != a.logits;  // the target's logit: but for its holder it may be written over
    float xt = 0.0f;
    if (GIVEN && holds && pt >= 0) beside = load_piece<false>(x + cut.head + pt * N);
    if (GIVEN && (holds || all_know)) xt = elem(x, t);
    const RowOut o = GIVEN ? given_row(a, lse, given, t < V) : known_row(a, r, given, t < V);
    float others = 0.0f;  // LSE: what the words of other pieces than the target's come to, to a lane
    if (edges) {
        const int j = cut.edge(tid);
        const float e = o.probability(elem(x, j), s2);
        if (BY == LSE && j != t) others = e;
        put(dx, j, -o.coef * e);
    }
    for (int p0 = from + tid; p0 < to; p0 += GRAD_U * GRAD_NT) {
        Piece<T> v[GRAD_U];
#pragma unroll
        for (int u = 0; u < GRAD_U; ++u) {
            const int p = p0 + u * GRAD_NT;
            if (p < to) v[u] = load_piece<PAST>(x + cut.head + p * N);
        }
        float round = 0.0f;
#pragma unroll
        for (int u = 0; u < GRAD_U; ++u) {
            const int p = p0 + u * GRAD_NT;
            if (p >= to) continue;
            float sum = 0.0f;
            store_piece<PAST>(dx + cut.head + p * N, v[u].map([&](int, float y) {
                const float e = o.probability(y, s2);
                if (BY == LSE) sum += e;
                return -o.coef * e;
            }));
            if (BY == LSE) round += p == pt ? 0.0f : sum;
        }
        if (BY == LSE) others += round;
    }
    if constexpr (!GIVEN) {
        if (holds) put(dx, t, o.target);
        return;
    }
    const float logp = static_cast<float>(static_cast<double>(xt) * a.scale - lse);
    const bool dim = (holds || all_know) && faint<T>(lse, logp);
    if (GRAD_NT == 64 ? !__ballot(dim) : all_know && !dim) {
        if (holds) put(dx, t, o.coef * -expm1f(logp));
        return;
    }
    if (BY == DEALT && !held_here) return;  // the holder's workgroup reads the others again
    if constexpr (BY == DEALT) {
        if (tid < cut.edges && cut.edge(tid) != t) others = o.probability(elem(x, cut.edge(tid)), s2);
        for (int p0 = tid; p0 < cut.pieces; p0 += GRAD_U * GRAD_NT) {
            Piece<T> v[GRAD_U];
#pragma unroll
            for (int u = 0; u < GRAD_U; ++u) {
                const int p = p0 + u * GRAD_NT;
                v[u] = p < cut.pieces && p != pt ? load_piece<false>(x + cut.head + p * N) : Piece<T>::nothing();
            }
            float round = 0.0f;
#pragma unroll
            for (int u = 0; u < GRAD_U; ++u) v[u].each([&](float y) { round += o.probability(y, s2); });
            others += round;
        }
    }
    if (dim && holds) {
        int i = 0;
        beside.each([&](float y) { others += i++ == word ? 0.0f : o.probability(y, s2); });
    }
    float rest = group_sum<64>(others);
    if constexpr (GRAD_NT > 64) {
        if ((tid & 63) == 0) sh_m[tid >> 6] = rest;
        __syncthreads();
        rest = 0.0f;
        for (int w = 0; w < GRAD_NT / 64; ++w) rest += sh_m[w];
    }
    if (holds) put(dx, t, o.coef * (dim ? rest : -expm1f(logp)));
}

__global__ __launch_bounds__(1024) void loss_sum(const double* x, int64_t n, float* out) {
    const double s = sum_of<1024>(x, n);
    if (threadIdx.x == 0) *out = static_cast<float>(s);
}

// A workgroup takes a pair: both sequences' sums, the pair's loss, and for every row of the two what its gradient is multiplied by.
constexpr int PAIR_NT = 1024;
__global__ __launch_bounds__(PAIR_NT) void pair_loss(Pairs a) {
    __shared__ double sh[2][PAIR_NT / 64];
    const int tid = threadIdx.x, seq[2] = {static_cast<int>(blockIdx.x), a.pairs + static_cast<int>(blockIdx.x)};
    int64_t begin[2], end[2];
    double sum[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        begin[k] = start_of(a, seq[k]), end[k] = start_of(a, seq[k] + 1);
        sum[k] = wave_sum(sequence_part<1>(a, begin[k], end[k], tid, PAIR_NT));
        if ((tid & 63) == 0) sh[k][tid >> 6] = sum[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        sum[k] = 0.0;
        for (int w = 0; w < PAIR_NT / 64; ++w) sum[k] += sh[k][w];
    }
    const PairOut o = pair_terms(a, sum[0], sum[1]);
    if (tid == 0) a.margins[blockIdx.x] = static_cast<float>(o.margin), a.losses[blockIdx.x] = o.loss;
#pragma unroll
    for (int k = 0; k < 2; ++k)
        for (int64_t r = begin[k] + tid; r < end[k]; r += PAIR_NT) a.coef[r] = k ? -o.slope : o.slope;
}

// From here on logits and gradient do not stay in the 256 MB of the last-level cache together. A gradient that passes it by leaves it to the logits, which the
// preference loss reads again (197 MB of logits 120.7 -> 100.0 us; 524 MB 308 -> 271), and takes less time to write (policy loss 81.3 -> 72.0; 204 -> 181). The
// product behind the loss then finds less of a small one there: loss and product of 33 MB 120.7 -> 128.7 us, 66 MB 172.8 -> 185.3, 98 MB 228.6 -> 229.3, 131 MB
// 254.0 -> 251.9, 262 MB 392.5 -> 387.2.
constexpr int64_t PAST_BYTES = int64_t{96} << 20;
constexpr int HELD_PIECES = 8192;
// Threads and pieces for a row. Policy loss over 262 to 131 MB of bf16 logits, the neighbours in brackets: 1000 words 73 us (a wavefront for two pieces; 90 on two wavefronts),
// 2000 words 106 (118 on 128 threads), 4000 words 100 (104 on 256, 106 on 64), 8000 words 91.5 (95 on 128, 100 on 512), 16000 words 90 (96 on 256), 32000 words 94 (94 on 1024), 64000
// words 98.8 (97.7 read twice), 128000 words 101 (101 held by 1024 threads, 16 pieces each, whose log-probabilities took 54.4 instead of 46.7).
template <typename T, Mode MODE, bool PAST>
void launch_held(const Loss& a, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>(a.rows));
    const int pieces = a.vocab / Piece<T>::N;
    if (pieces <= 64) return rows_held<T, MODE, 64, 1, PAST><<<grid, 64, 0, st>>>(a);
    if (pieces <= 128) return rows_held<T, MODE, 64, 2, PAST><<<grid, 64, 0, st>>>(a);
    if (pieces <= 256) return rows_held<T, MODE, 64, 4, PAST><<<grid, 64, 0, st>>>(a);
    if (pieces <= 512) return rows_held<T, MODE, 128, 4, PAST><<<grid, 128, 0, st>>>(a);
    if (pieces <= 1024) return rows_held<T, MODE, 256, 4, PAST><<<grid, 256, 0, st>>>(a);
    if (pieces <= 2048) return rows_held<T, MODE, 512, 4, PAST><<<grid, 512, 0, st>>>(a);
    if (pieces <= 4096) return rows_held<T, MODE, 512, 8, PAST><<<grid, 512, 0, st>>>(a);
    if (pieces <= HELD_PIECES) return rows_held<T, MODE, 1024, 8, PAST><<<grid, 1024, 0, st>>>(a);
    rows_long<T, MODE, PAST><<<grid, LONG_NT, 0, st>>>(a);
}
// Workgroups that a row is dealt to: one, but for a few rows that none holds. bf16, log-probabilities whole and dealt out: one row of 128000 words 8.7 and 5.6 us, 64 of
// them 9.5 and 6.9, one of 200000 12.6 and 5.7, 64 13.6 and 8.8; a held row of 32000 words takes 4.1, less than the two launches. The policy loss, with a pass of its own for the
// gradient: one row of 34000 words 10.3 and 9.0, 31 of them 10.8 and 10.3, 127 11.9 and 13.1; one of 134000 20.2 and 9.2, 64 23.9 and 18.1, 250 36 and 41.
int parts_of_rows(Mode mode, int64_t rows, int64_t vocab, int64_t es) {
    const int64_t pieces = vocab * es / 16, held = mode == POLICY && rows <= 32 ? 4096 : HELD_PIECES;
    if (rows < 1 || rows >= (mode == POLICY ? 65 : FEW_ROWS) || pieces <= held) return 1;
    return static_cast<int>(std::min<int64_t>(std::min<int64_t>(MOST_PARTS, 512 / rows), pieces / (2 * PART_NT)));
}
template <typename T, Mode MODE>
void launch_dealt(const Loss& a, int parts, hipStream_t st) {
    const int pieces = a.vocab / Piece<T>::N, per = (pieces + parts - 1) / parts;
    rows_part<T, MODE><<<dim3(static_cast<unsigned>(a.rows), static_cast<unsigned>(parts)), PART_NT, 0, st>>>(a, per, a.parts);
    rows_join<T, MODE><<<dim3(static_cast<unsigned>(a.rows)), 64, 0, st>>>(a, parts, a.parts);
}
template <typename T, int NT, bool PAST, Known BY>
void launch_grad(const Loss& a, const Pairs& pairs, hipStream_t st) {
    // Few rows are dealt out, one load to a thread, as far as that fills the chip: one row of 128000 words bf16 11.0 -> 3.2 us, 64 of them 13.6 -> 7.1, 128 16.3 -> 12.4. From the log of a
    // sum not to two, nor rows that a workgroup reads in one round: they gain little (192 rows 18.9 and 17.4, 64 of 10007 words 3.9 and 3.6), and where a target's element is what the others come to,
    // whoever holds it reads the others' parts as well (192 rows 23.7, 64 of 10007 words 5.2; one row of 128000 words 10.1). Nor rows that are written over, of which it would read what others have
    // written (one row of 128000 words 3.3 -> 10.9).
    const int pieces = a.vocab / Piece<T>::N, most = static_cast<int>(std::max<int64_t>(1, 512 / std::max<int64_t>(a.rows, 1)));
    const bool whole = BY == LSE && (most < 3 || pieces <= GRAD_U * NT || a.dlogits == a.logits);
    const int parts = whole ? 1 : std::min(most, std::max(1, pieces / NT)), per = (pieces + parts - 1) / parts;
    const dim3 grid(static_cast<unsigned>(a.rows + (a.loss ? 1 : 0)), static_cast<unsigned>(parts));
    if constexpr (BY == LSE && NT == 512) {
        if (parts > 1) return rows_grad<T, NT, PAST, DEALT><<<grid, NT, 0, st>>>(a, per, pairs);
    }
    rows_grad<T, NT, PAST, BY><<<grid, NT, 0, st>>>(a, per, pairs);
}
// Threads for a row: bf16, 65536 rows of 1000 words 48 us by 64 threads (57 by 128, 72 by 256, 122 by 512), 32768 of 2000 48 (48, 49, 70), 16384 of 4000 49 (48, 46,
// 49), 8192 of 8000 49 (45, 44, 42), 8192 of 32000 208 (205, 193, 180). The pairs' mean is a workgroup's too: thousands of pairs want a large one.
template <typename T, Known BY>
void launch_grads(const Loss& a, bool past, hipStream_t st) {
    const int pieces = a.vocab / Piece<T>::N;
    if (pieces <= 256 && a.terms <= 4096) return past ? launch_grad<T, 64, true, BY>(a, Pairs{}, st) : launch_grad<T, 64, false, BY>(a, Pairs{}, st);
    if (pieces <= 512 && a.terms <= 4096) return past ? launch_grad<T, 256, true, BY>(a, Pairs{}, st) : launch_grad<T, 256, false, BY>(a, Pairs{}, st);
    past ? launch_grad<T, 512, true, BY>(a, Pairs{}, st) : launch_grad<T, 512, false, BY>(a, Pairs{}, st);
}
template <typename T, Mode MODE>
void launch_typed(const Loss& a, const Pairs* pairs, hipStream_t st) {
    const bool past = a.rows * a.vocab * static_cast<int64_t>(sizeof(T)) >= PAST_BYTES;
    const dim3 grid(static_cast<unsigned>(a.rows + (a.loss ? 1 : 0)));
    if constexpr (MODE == LOGP) {
        const int parts = a.parts ? parts_of_rows(LOGP, a.rows, a.vocab, sizeof(T)) : 1;
        if (parts == 1) return launch_held<T, MODE, false>(a, st);  // the logits are read again for their gradient: not past the cache
        launch_dealt<T, MODE>(a, parts, st);
    } else {
        if constexpr (MODE == GRAD) {
            if (pairs) return launch_grad<T, 512, false, PAIRS>(a, *pairs, st);
            a.sums ? launch_grads<T, SUMS>(a, past, st) : launch_grads<T, LSE>(a, past, st);
        } else if (a.parts)
            launch_dealt<T, MODE>(a, parts_of_rows(POLICY, a.rows, a.vocab, sizeof(T)), st);
        else
            past ? launch_held<T, MODE, true>(a, st) : launch_held<T, MODE, false>(a, st);
    }
}
// A launch has fewer than 2^32 threads, 1024 for a row at most: more rows than that allows go in runs.
constexpr int64_t MOST_ROWS = (1 << 22) - 2;
template <Mode MODE>
int launch_rows(const Loss& all, int dtype, hipStream_t st, const Pairs* pairs = nullptr) {
    if (all.rows == 0 && !all.loss) return PK_OK;
    for (int64_t r = 0; r == 0 || r < all.rows; r += MOST_ROWS) {
        const auto on = [r](auto*& p, int64_t ld = 1) { p = p ? p + r * ld : p; };
        const int64_t es = elem_size(dtype);
        Loss a = all;
        a.rows = std::min(MOST_ROWS, all.rows - r);
        if (r + MOST_ROWS < all.rows) a.loss = nullptr;  // the last run's
        a.logits = static_cast<const char*>(a.logits) + r * a.ld * es;
        if (a.dlogits) a.dlogits = static_cast<char*>(a.dlogits) + r * a.dld * es;
        on(a.targets), on(a.logp), on(a.lse), on(a.lse_in), on(a.coef, a.coef_step), on(a.clear), on(a.low), on(a.sums), on(a.old_logp), on(a.ref_logp), on(a.adv), on(a.weights);
        on(a.row_loss), on(a.coef_out, a.coef_step);
        if (dtype == PK_BF16)
            launch_typed<uint16_t, MODE>(a, pairs, st);
        else
            launch_typed<float, MODE>(a, pairs, st);
        if (int rc = launched()) return rc;
    }
    return PK_OK;
}

// What every entry asks of its logits; dlogits only where it writes them: over the logits, row for row, or clear of them.
int check(const char* who, const void* logits, int64_t ld, const int* targets, int64_t rows, int64_t vocab, float scale, int dtype, bool writes,
          const void* dlogits, int64_t dld) {
    const std::string w(who);
    if (rows < 0 || rows >= INT32_MAX || vocab <= 0 || vocab > (1 << 30)) return fail(PK_ERR_SHAPE, w + ": shape mismatch (rows or vocabulary out of range)");
    if (!known_dtype(dtype)) return fail(PK_ERR_ARGUMENT, w + ": dtype must be PK_F32 or PK_BF16");
    if (!(scale >= 0x1p-64f && scale <= 0x1p64f)) return fail(PK_ERR_ARGUMENT, w + ": scale must lie between 2^-64 and 2^64");  // both parts of its product with log2(e) are numbers
    if (ld < 0 || (writes && rows > 1 && dld < vocab)) return fail(PK_ERR_SHAPE, w + ": rows of logits overlap");
    if (rows == 0) return PK_OK;
    if (!logits || !targets || (writes && !dlogits)) return fail(PK_ERR_ARGUMENT, w + ": null pointer");
    if (writes && !(logits == dlogits && (ld == dld || rows == 1))) {
        const uintptr_t es = static_cast<uintptr_t>(elem_size(dtype)), x = reinterpret_cast<uintptr_t>(logits), y = reinterpret_cast<uintptr_t>(dlogits);
        const uintptr_t xe = x + ((rows - 1) * ld + vocab) * es, ye = y + ((rows - 1) * dld + vocab) * es;
        // two matrices may lie in one another's gaps; what no gap can hold is refused
        if (x < ye && y < xe && !(ld == dld && ld >= 2 * vocab && (y > x ? y - x : x - y) % (ld * es) >= vocab * es &&
                                  (y > x ? y - x : x - y) % (ld * es) <= (ld - vocab) * es))
            return fail(PK_ERR_ARGUMENT, w + ": dlogits may lie where the logits do, row for row, or clear of them");
    }
    return PK_OK;
}

// Few pairs of few rows are formed by the gradient's own wavefronts, each the pair it wants: a launch less. bf16, with a launch of their own and without: 8 pairs of 4 + 4 rows of
// 1000 words 10.6 and 7.9 us, one of 256 + 256 of 32000 25.5 and 23.5, 8 of 32 + 32 of 8000 13.6 and 12.7; past that 31 pairs of 4 + 4 11.5 and 14.4, one of 512 + 512 18.0 and 21.6.
constexpr int MOST_FEW_PAIRS = 8, FEW_PAIRS_ROWS = 512;
static_assert(2 * MOST_FEW_PAIRS < 64, "their starts fit into a wavefront");
size_t pad(size_t bytes) { return (bytes + 255) & ~size_t{255}; }

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" {

size_t pk_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int dtype) {
    if (rows < 0 || vocab <= 0 || !known_dtype(dtype)) return 0;
    const int parts = parts_of_rows(LOGP, rows, vocab, elem_size(dtype));
    return parts == 1 ? 0 : sizeof(float2) * static_cast<size_t>(rows * parts);
}

int pk_token_logprobs_fwd(const void* logits, int64_t ld, const int* targets, int64_t rows, int64_t vocab, float scale, float* logp, float* lse,
                          void* workspace, size_t workspace_bytes, int dtype, void* stream) {
    return c_entry([&] {
        if (int rc = check("pk_token_logprobs_fwd", logits, ld, targets, rows, vocab, scale, dtype, false, nullptr, 0)) return rc;
        if (rows > 0 && !logp) return fail(PK_ERR_ARGUMENT, "pk_token_logprobs_fwd: null pointer");
        if (workspace && (workspace_bytes < pk_token_logprobs_workspace_bytes(rows, vocab, dtype) || !aligned(workspace, 8)))
            return fail(PK_ERR_WORKSPACE, "pk_token_logprobs_fwd: workspace too small (pk_token_logprobs_workspace_bytes)");
        touch({logits, targets, logp, lse, workspace}, stream);
        Loss a{};
        a.parts = static_cast<float2*>(workspace);
        a.logits = logits, a.ld = ld, a.targets = targets, a.rows = rows, a.vocab = static_cast<int>(vocab), a.logp = logp, a.lse = lse;
        set_scale(a, scale);
        return launch_rows<LOGP>(a, dtype, static_cast<hipStream_t>(stream));
    });
}

int pk_token_logprobs_bwd(const void* logits, int64_t ld, const int* targets, const float* lse, const float* dlogp, int64_t rows, int64_t vocab,
                          float scale, void* dlogits, int64_t dld, int dtype, void* stream) {
    return c_entry([&] {
        if (int rc = check("pk_token_logprobs_bwd", logits, ld, targets, rows, vocab, scale, dtype, true, dlogits, dld)) return rc;
        if (rows > 0 && (!lse || !dlogp)) return fail(PK_ERR_ARGUMENT, "pk_token_logprobs_bwd: null pointer");
        touch({logits, targets, lse, dlogp, dlogits}, stream);
        Loss a{};
        a.logits = logits, a.ld = ld, a.targets = targets, a.rows = rows, a.vocab = static_cast<int>(vocab);
        set_scale(a, scale);
        a.dlogits = dlogits, a.dld = dld, a.lse_in = lse, a.coef = dlogp, a.coef_step = 1;
        return launch_rows<GRAD>(a, dtype, static_cast<hipStream_t>(stream));
    });
}

size_t pk_policy_loss_workspace_bytes(int64_t rows, int64_t vocab, int dtype) {
    if (rows < 0 || vocab <= 0 || !known_dtype(dtype)) return 0;
    const int parts = parts_of_rows(POLICY, rows, vocab, elem_size(dtype));
    return parts == 1 ? 0 : (sizeof(float2) * parts + 2 * sizeof(float)) * static_cast<size_t>(rows);
}

int pk_policy_loss(const pk_policy_config* c, const void* logits, int64_t ld, const int* targets, const float* old_logp, const float* ref_logp,
                   const float* advantages, const float* weights, int64_t rows, int64_t vocab, void* dlogits, int64_t dld, float* logp,
                   double* row_loss, float* loss, void* workspace, size_t workspace_bytes, int dtype, void* stream) {
    return c_entry([&] {
        if (!c || !loss) return fail(PK_ERR_ARGUMENT, "pk_policy_loss: null pointer");
        if (int rc = check("pk_policy_loss", logits, ld, targets, rows, vocab, c->scale, dtype, true, dlogits, dld)) return rc;
        if (rows > 0 && (!old_logp || !advantages || !weights || !logp || !row_loss)) return fail(PK_ERR_ARGUMENT, "pk_policy_loss: null pointer");
        if (!(c->clip_low >= 0.0f) || !(c->clip_high >= 0.0f)) return fail(PK_ERR_ARGUMENT, "pk_policy_loss: the clip's widths must not be negative");
        if (!std::isfinite(c->kl_coef) || !std::isfinite(c->upstream)) return fail(PK_ERR_ARGUMENT, "pk_policy_loss: kl_coef and upstream must be finite");
        if (c->kl_coef != 0.0f && !ref_logp && rows > 0) return fail(PK_ERR_ARGUMENT, "pk_policy_loss: a KL term needs ref_logp");
        if (workspace && (workspace_bytes < pk_policy_loss_workspace_bytes(rows, vocab, dtype) || !aligned(workspace, 8)))
            return fail(PK_ERR_WORKSPACE, "pk_policy_loss: workspace too small (pk_policy_loss_workspace_bytes)");
        touch({logits, targets, old_logp, ref_logp, advantages, weights, dlogits, logp, row_loss, loss, workspace}, stream);
        hipStream_t st = static_cast<hipStream_t>(stream);
        Loss a{};
        a.logits = logits, a.ld = ld, a.targets = targets, a.rows = rows, a.vocab = static_cast<int>(vocab);
        set_scale(a, c->scale);
        a.dlogits = dlogits, a.dld = dld, a.logp = logp, a.row_loss = row_loss;
        a.old_logp = old_logp, a.ref_logp = c->kl_coef != 0.0f ? ref_logp : nullptr, a.adv = advantages, a.weights = weights;
        a.clip_low = c->clip_low, a.clip_high = c->clip_high, a.kl = c->kl_coef, a.upstream = c->upstream;
        const int parts = workspace ? parts_of_rows(POLICY, rows, vocab, elem_size(dtype)) : 1;
        if (parts > 1) {  // the gradient in a pass of its own, once the rows' parts are joined
            a.parts = static_cast<float2*>(workspace), a.sums = a.parts + rows * parts;
            a.coef_out = &a.parts->x, a.coef_step = 2 * parts;  // a row's takes the place of its first part once that is read
            if (int rc = launch_rows<POLICY>(a, dtype, st)) return rc;
            a.parts = nullptr, a.coef = a.coef_out, a.losses = row_loss, a.terms = rows, a.divisor = 1.0, a.loss = loss;
            return launch_rows<GRAD>(a, dtype, st);
        }
        if (int rc = launch_rows<POLICY>(a, dtype, st)) return rc;
        loss_sum<<<1, 1024, 0, st>>>(row_loss, rows, loss);
        return launched();
    });
}

size_t pk_preference_loss_workspace_bytes(int64_t rows, int64_t pairs) {
    if (rows < 0 || pairs < 0) return 0;
    return 2 * pad(sizeof(float) * static_cast<size_t>(rows)) + pad(sizeof(double) * static_cast<size_t>(rows)) + pad(sizeof(double) * static_cast<size_t>(pairs)) +
           (rows < FEW_ROWS ? pad(sizeof(float2) * static_cast<size_t>(rows) * MOST_PARTS) : 0);
}

int pk_preference_loss(const pk_preference_config* c, const void* logits, int64_t ld, const int* targets, const int* seq_start, int64_t pairs,
                       const float* ref_logp, int64_t rows, int64_t vocab, void* dlogits, int64_t dld, float* logp, float* margins, float* loss,
                       void* workspace, size_t workspace_bytes, int dtype, void* stream) {
    return c_entry([&] {
        if (!c || !loss || !margins || !seq_start) return fail(PK_ERR_ARGUMENT, "pk_preference_loss: null pointer");
        if (pairs < 1 || pairs > MOST_ROWS) return fail(PK_ERR_SHAPE, "pk_preference_loss: shape mismatch (at least one pair is wanted)");
        if (int rc = check("pk_preference_loss", logits, ld, targets, rows, vocab, c->scale, dtype, true, dlogits, dld)) return rc;
        if (rows > 0 && (!ref_logp || !logp)) return fail(PK_ERR_ARGUMENT, "pk_preference_loss: null pointer");
        if (!std::isfinite(c->beta) || !std::isfinite(c->upstream)) return fail(PK_ERR_ARGUMENT, "pk_preference_loss: beta and upstream must be finite");
        if (!(c->label_smoothing >= 0.0f && c->label_smoothing <= 1.0f))
            return fail(PK_ERR_ARGUMENT, "pk_preference_loss: label_smoothing must lie between 0 and 1");
        if (!workspace || workspace_bytes < pk_preference_loss_workspace_bytes(rows, pairs) || !aligned(workspace, 8))
            return fail(PK_ERR_WORKSPACE, "pk_preference_loss: workspace too small (pk_preference_loss_workspace_bytes)");
        touch({logits, targets, seq_start, ref_logp, dlogits, logp, margins, loss, workspace}, stream);
        hipStream_t st = static_cast<hipStream_t>(stream);
        char* ws = static_cast<char*>(workspace);
        const size_t singles = pad(sizeof(float) * static_cast<size_t>(rows)), doubles = pad(sizeof(double) * static_cast<size_t>(rows));
        float *low = reinterpret_cast<float*>(ws), *coef = reinterpret_cast<float*>(ws + singles);
        float2* sums = reinterpret_cast<float2*>(ws + 2 * singles);
        double* losses = reinterpret_cast<double*>(ws + 2 * singles + doubles);
        Loss a{};
        a.logits = logits, a.ld = ld, a.targets = targets, a.rows = rows, a.vocab = static_cast<int>(vocab);
        set_scale(a, c->scale);
        a.logp = logp, a.low = low, a.sums = sums, a.clear = coef;
        if (rows < FEW_ROWS) a.parts = reinterpret_cast<float2*>(ws + 2 * singles + doubles + pad(sizeof(double) * static_cast<size_t>(pairs)));
        if (int rc = launch_rows<LOGP>(a, dtype, st)) return rc;
        const Pairs p{seq_start, targets, logp, low, ref_logp, coef, margins, losses, rows, static_cast<int>(pairs), c->beta, c->label_smoothing, c->upstream};
        a.dlogits = dlogits, a.dld = dld;
        const bool few = rows <= FEW_PAIRS_ROWS && pairs <= MOST_FEW_PAIRS;
        if (!few) {
            pair_loss<<<dim3(static_cast<unsigned>(pairs)), PAIR_NT, 0, st>>>(p);
            if (int rc = launched()) return rc;
        }
        a.coef = coef, a.coef_step = 1, a.losses = losses, a.terms = pairs, a.divisor = static_cast<double>(pairs), a.loss = loss;
        return launch_rows<GRAD>(a, dtype, st, few ? &p : nullptr);
    });
}

}  // extern "C"
