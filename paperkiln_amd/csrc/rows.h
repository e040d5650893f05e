// Rows of storage elements in 16-byte pieces, and sums over a wavefront in 64 bits: what the kernels of token_loss.hip, distill_loss.hip and layernorm.hip share.
#pragma once
#include "post.h"

namespace pk {

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
// Between two walks over a row the pieces stay as they are: the compiler would keep every element of the first walk in a register of its own.
template <typename T, int PER>
__device__ inline void keep_packed(Piece<T> (&held)[PER]) {
    if constexpr (Piece<T>::N == 8) {
#pragma unroll
        for (int k = 0; k < PER; ++k) asm volatile("" : "+v"(held[k].v));
    }
}

template <typename T, int NT, bool PAST>
__device__ inline void zero_row(T* dx, const Cut<T>& cut, int tid) {
    for (int p = tid; p < cut.pieces; p += NT) store_piece<PAST>(dx + cut.head + p * Piece<T>::N, Piece<T>{{0, 0, 0, 0}});
    if (tid < cut.edges) put(dx, cut.edge(tid), 0.0f);
}

// ---- exponentials and sums of a row ----

constexpr float LOG2E = 1.44269504088896340736f;
constexpr double LN2 = 0.693147180559945309417;

// 2^(s2 (x - m)). The difference is taken before the product, so a row of the type's lowest value has its probabilities too. The exponent from both parts of s2: rounded to 32
// bits it would turn every row's log-probability by up to 6e-8 times its logits, always the same way, and a preference loss adds up hundreds of them (margins
// 4e-7 off, 1e-7 so). A logit of -inf stays one: the low part is not zero nor negative.
template <typename A>
__device__ inline float power_of(const A& a, float x, float m) {
    const float d = x - m;
    return __builtin_amdgcn_exp2f(fmaf(d, a.s2_hi, d * a.s2_lo));
}
template <typename A>  // A: a kernel's arguments, with scale, s2, per_s2, s2_hi and s2_lo
void set_scale(A& a, double scale) {
    a.scale = static_cast<float>(scale);
    a.s2 = scale * 1.4426950408889634074;
    a.per_s2 = 1.0 / a.s2;
    a.s2_hi = static_cast<float>(a.s2);
    if (static_cast<double>(a.s2_hi) >= a.s2) a.s2_hi = std::nextafter(a.s2_hi, 0.0f);
    a.s2_lo = static_cast<float>(a.s2 - static_cast<double>(a.s2_hi));
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
struct RowTotal {
    float top;
    double sum;  // of 2^(s2 (x - top))
};
template <typename A, int WAVES>
__device__ inline RowTotal total_of_row(const A& a, const float (&m)[WAVES], const double (&s)[WAVES]) {
    float top = m[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, m[w]);
    double sum = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += s[w] == 0.0 ? 0.0 : s[w] * power_of(a, m[w], top);
    return RowTotal{top, sum};
}
template <typename A, int WAVES>
__device__ inline RowSum sum_of_row(const A& a, const float (&m)[WAVES], const double (&s)[WAVES]) {
    const RowTotal t = total_of_row(a, m, s);
    return row_sum(t.top, t.sum);
}

// Rows that no workgroup holds are read in strides, with a running maximum and sum, and again for the gradient.
constexpr int LONG_U = 4;
template <typename T, int NT, typename A>
__device__ inline void running(const A& a, const T* x, const Cut<T>& cut, int from, int to, float edge, float* sh_m, double* sh_s) {
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

}  // namespace pk
