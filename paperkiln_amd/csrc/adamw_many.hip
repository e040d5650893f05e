// One AdamW step over a list of tensors, with the global gradient norm's clip in front of it, the moments in 32 bits or in 8.
//
//   g' = g min(1, max_norm / |g|)    m' = b1 m + (1 - b1) g'    v' = b2 v + (1 - b2) g'^2    p -= lr ((m' / c1) / (sqrt(v' / c2) + eps) + wd p)
//
// In 8 bits m is e4m3 and v e5m2 with a power of two for every 256 elements of a tensor, the smallest that keeps the block's largest value inside the
// format. The powers are the device's powf(2, e), which torch.ldexp is on this GPU too (one step of 32 bits under 2^e for about a sixth of the exponents): a state
// that a program packs or unpacks with torch's operations has the bits that it has here. v' moves by a thousandth of itself in a step, far less than the 1/8 between neighbours of its format, so
// rounding to the nearest would leave it where it is for ever; both moments are rounded up with the probability that the bits dropped stand for,
// from a hash of the seed, the tensor's place in the list and the element's place in it. The same call gives the same bits. A v that is not zero
// does not become zero: m / sqrt(v) would have no bound. A block that holds a value which is not finite becomes NaN as a whole.
//
// Nothing is formed with fused operations (each product and sum is rounded by itself): a state in 8 bits is then one function of its inputs in
// any program that follows these formulas, and not of how a compiler contracts them, and so is a whole step with moments in 32 bits.
//
// What bounds it: memory. An element of 32-bit moments reads p, m, v and the gradient, 14 to 16 bytes, with a clip the gradient once more, and writes 12; with 8-bit moments it
// reads 8 to 10 and writes 6; a copy is 2 more.
#include "post.h"

#include <algorithm>
#include <vector>

#pragma clang fp contract(off)

namespace pk {
namespace {

constexpr int BLOCK = 256, NT = 256, WAVES = NT / 64;  // elements that share a scale; a wavefront takes a block

struct One {
    float* p;
    const void* g;
    void *m, *v;
    float *ms, *vs;
    uint16_t* copy;
    int64_t n;
};
// The list travels in the kernel's arguments, 4 KB at most, addresses in 48 bits: 126 tensors with moments in 32 bits, 58 in whole words (a launch is 4 us of the
// host's: 96 tensors 13.8 -> 11.0 us).
template <int PTRS>  // addresses of a tensor
struct Table {
    static constexpr int MOST = (4096 - 64) / (8 + 4 * PTRS + 4 * ((PTRS + 1) / 2));
    uint64_t size[MOST];  // elements, 40 bits; the tensor's first workgroup above
    uint32_t low[MOST][PTRS], high[MOST][(PTRS + 1) / 2];
    int count, place;  // tensors, the first one's place in the caller's list
    uint32_t seed;
    int per;  // blocks of a workgroup
    void put(int j, int64_t n, int64_t first, std::initializer_list<const void*> at) {
        size[j] = static_cast<uint64_t>(n) | static_cast<uint64_t>(first) << 40;
        int k = 0;
        for (const void* p : at) {
            const uint64_t u = reinterpret_cast<uint64_t>(p);
            const uint32_t top = static_cast<uint32_t>(u >> 32);
            low[j][k] = static_cast<uint32_t>(u);
            high[j][k / 2] = k % 2 ? high[j][k / 2] | top << 16 : top;
            ++k;
        }
    }
    __device__ int64_t elements(int j) const { return static_cast<int64_t>(size[j] & ((uint64_t{1} << 40) - 1)); }
    __device__ int first(int j) const { return static_cast<int>(size[j] >> 40); }
    template <typename T>
    __device__ T* at(int j, int k) const {
        return reinterpret_cast<T*>(static_cast<uint64_t>(low[j][k]) | static_cast<uint64_t>(high[j][k / 2] >> (k % 2 * 16) & 0xFFFFu) << 32);
    }
    // The tensor that a workgroup belongs to: the last one whose first workgroup is not behind it (one without elements has no workgroup of its own).
    __device__ int tensor_of(int group) const {
        int lo = 0, hi = count - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (first(mid) <= group)
                lo = mid;
            else
                hi = mid - 1;
        }
        return lo;
    }
};
constexpr int pointers(bool eight, bool copy) { return 4 + (eight ? 2 : 0) + (copy ? 1 : 0); }
struct Step {
    float lr, b1, b2, rest1, rest2, eps, wd, per_c1, per_c2;  // 1 / c1, 1 / c2
    const float* factor;                                       // what the gradients are multiplied by, or null
};
static_assert(sizeof(Table<4>) + sizeof(Step) <= 4096 && sizeof(Table<5>) + sizeof(Step) <= 4096 && sizeof(Table<6>) + sizeof(Step) <= 4096 &&
                  sizeof(Table<7>) + sizeof(Step) <= 4096 && sizeof(Table<1>) + 8 <= 4096,
              "kernel arguments");

// The low 32 bits scrambled: two multiplications by the fractions of the square roots of 3 and 2, shifts between them.
__host__ __device__ inline uint32_t mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0xBB67AE85u;
    x ^= x >> 15;
    x *= 0x6A09E667u;
    return x ^ (x >> 16);
}

// the largest of all lanes
__device__ inline uint32_t wave_max(uint32_t x) {
    const auto h = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = max(h[0], h[1]);
    const auto q = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(q[0], q[1]);
    auto moved = [](uint32_t u, auto ctrl) { return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, u, decltype(ctrl)::value, 0xf, 0xf, true)); };
    x = max(x, moved(x, std::integral_constant<int, 0x128>{}));
    x = max(x, moved(x, std::integral_constant<int, 0x141>{}));
    x = max(x, moved(x, std::integral_constant<int, 0x4E>{}));
    return max(x, moved(x, std::integral_constant<int, 0xB1>{}));
}

// The exponent of a block's scale from the bits of its largest magnitude; TOP: the exponent of the format's largest value, 1.75 * 2^TOP.
template <int TOP>
__device__ inline int scale_power(uint32_t largest) {
    const int e = static_cast<int>(largest >> 23) - 127 + ((largest & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return max(e - TOP, -126);
}
// powf(2, e) for e in -126 .. 127 at e + 126, formed once by a workgroup: a call a block and wavefront would cost more than the block's update.
struct Powers {
    const float* at;
    __device__ float operator()(int e) const { return at[e + 126]; }
};
__device__ inline Powers powers(float (&table)[NT]) {
    table[threadIdx.x] = powf(2.0f, static_cast<float>(static_cast<int>(threadIdx.x) - 126));
    __syncthreads();
    return Powers{table};
}

// Into 8 bits: the magnitude moved to where the format's exponent range begins at 32 bits' own, random bits added below the last kept one.
__device__ inline uint32_t to_e4m3(float y, uint32_t chance) {
    return ((__float_as_uint(fabsf(y) * 0x1p-120f) + (chance << 4) + 8u) >> 20) | ((__float_as_uint(y) >> 24) & 0x80u);
}
__device__ inline uint32_t to_e5m2(float y, uint32_t chance) { return (__float_as_uint(y * 0x1p-112f) + (chance << 5) + 16u) >> 21; }
__device__ inline float of_e4m3(uint32_t c) {
    const float x = (c & 0x7Fu) == 0x7Fu ? NAN : __uint_as_float((c & 0x7Fu) << 20) * 0x1p120f;
    return c & 0x80u ? -x : x;
}
__device__ inline float of_e5m2(uint32_t c) { return c > 0x7Cu ? NAN : c == 0x7Cu ? INFINITY : __uint_as_float(c << 21) * 0x1p112f; }

// sqrt of x >= 0 to a step of 32 bits; small x are scaled into the range of the instruction
__device__ inline float root(float x) {
    const bool small = x < 0x1p-100f;
    const float r = __builtin_amdgcn_sqrtf(small ? x * 0x1p100f : x);
    return small ? r * 0x1p-50f : r;
}
// m', v' and, with moments in 32 bits, p' by the formula's own roundings, the corrections as products with their reciprocals. With moments in 8 bits, which know their values to a
// sixteenth, the root and the quotient are the instructions', a step each: as the others' they would cost 35 M elements 89 -> 100 us, 5.8 M 18 -> 21. In 32 bits
// memory hides them (35 M 143 us, 5.8 M 26.4 either way; 0.5 M 3.6 -> 3.8).
template <bool EIGHT>
__device__ inline void update(const Step& s, float& p, float g, float& m, float& v) {
    const float a = s.b1 * m, b = s.rest1 * g, c = s.b2 * v, d = s.rest2 * g, e = d * g;
    m = a + b;
    v = c + e;
    float upd;
    if constexpr (EIGHT)
        upd = (m * s.per_c1) * __builtin_amdgcn_rcpf(root(v * s.per_c2) + s.eps);
    else
        upd = (m * s.per_c1) / (sqrtf(v * s.per_c2) + s.eps);
    p -= s.lr * (upd + s.wd * p);
}

// A wavefront takes what a tensor has behind its last whole block of 256 elements, a lane its elements lane, lane + 64, lane + 128 and lane + 192.
template <typename G, bool EIGHT>
__device__ inline void block_any(const One& t, const Step& s, uint32_t key, int64_t block, float gs, Powers power_of_two) {
    const int lane = threadIdx.x & 63;
    const int64_t base = block * BLOCK;
    float p[4], m[4], v[4];
    bool in[4];
    float ms = 0.0f, vs = 0.0f;
    if (EIGHT) ms = t.ms[block], vs = t.vs[block];
    uint32_t mm = 0, vm = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t i = base + lane + 64 * k;
        in[k] = i < t.n;
        p[k] = m[k] = v[k] = 0.0f;
        if (!in[k]) continue;
        const float g = elem(static_cast<const G*>(t.g), i) * gs;
        p[k] = t.p[i];
        if (EIGHT) {
            m[k] = of_e4m3(static_cast<const uint8_t*>(t.m)[i]) * ms;
            v[k] = of_e5m2(static_cast<const uint8_t*>(t.v)[i]) * vs;
        } else {
            m[k] = static_cast<const float*>(t.m)[i];
            v[k] = static_cast<const float*>(t.v)[i];
        }
        update<EIGHT>(s, p[k], g, m[k], v[k]);
        t.p[i] = p[k];
        if (t.copy) put(t.copy, i, p[k]);
        if (EIGHT) {
            mm = max(mm, __float_as_uint(m[k]) & 0x7FFFFFFFu);
            vm = max(vm, __float_as_uint(v[k]) & 0x7FFFFFFFu);
        } else {
            static_cast<float*>(t.m)[i] = m[k];
            static_cast<float*>(t.v)[i] = v[k];
        }
    }
    if (!EIGHT) return;
    mm = wave_max(mm), vm = wave_max(vm);
    const bool m_fine = mm < 0x7F800000u, v_fine = vm < 0x7F800000u;
    const int me = scale_power<8>(mm), ve = scale_power<15>(vm);
    if (lane == 0) {
        t.ms[block] = m_fine ? power_of_two(me) : NAN;
        t.vs[block] = v_fine ? power_of_two(ve) : NAN;
    }
    const float mi = power_of_two(-me), vi = power_of_two(-ve);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t i = base + lane + 64 * k;
        if (!in[k]) continue;
        const uint32_t h = mix(static_cast<uint32_t>(i) ^ key);
        static_cast<uint8_t*>(t.m)[i] = static_cast<uint8_t>(m_fine ? to_e4m3(m[k] * mi, h & 0xFFFFu) : 0x7Fu);
        static_cast<uint8_t*>(t.v)[i] = static_cast<uint8_t>(v_fine ? max(to_e5m2(v[k] * vi, h >> 16), v[k] > 0.0f ? 1u : 0u) : 0x7Fu);
    }
}

// The same for whole blocks: a lane takes four neighbours, 16 bytes of 32-bit tensors and four of 8-bit ones, which the hardware moves from where the elements may lie. Parameters and moments are not
// read again before the next step and pass by the last-level cache, which keeps the gradients from the norm's pass and the copies for the next
// products (35 M parameters, 8-bit moments, clip and copies 155.7 -> 141.7 us; one element off 221 element by element,
// 137 so).
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef uint32_t u32_any __attribute__((aligned(1)));
template <typename V>
__device__ inline V load_past(const void* p) { return __builtin_nontemporal_load(static_cast<const V*>(p)); }
template <typename V>
__device__ inline void store_past(void* p, V v) { __builtin_nontemporal_store(v, static_cast<V*>(p)); }
__device__ inline f32x4 four(const float* p, int64_t i) { return *reinterpret_cast<const f32x4_any*>(p + i); }
__device__ inline f32x4 four(const uint16_t* p, int64_t i) {
    const u32x2 r = *reinterpret_cast<const u32x2_any*>(p + i);
    return f32x4{__uint_as_float(r[0] << 16), __uint_as_float(r[0] & 0xFFFF0000u), __uint_as_float(r[1] << 16), __uint_as_float(r[1] & 0xFFFF0000u)};
}
template <typename G, bool EIGHT>
__device__ inline void block_whole(const One& t, const Step& s, uint32_t key, int64_t block, float gs, Powers power_of_two) {
    const int lane = threadIdx.x & 63;
    const int64_t i = block * BLOCK + lane * 4;
    const f32x4 g = four(static_cast<const G*>(t.g), i);
    f32x4 p = load_past<f32x4_any>(t.p + i), m, v;
    if constexpr (EIGHT) {
        const uint32_t mc = load_past<u32_any>(static_cast<const uint8_t*>(t.m) + i), vc = load_past<u32_any>(static_cast<const uint8_t*>(t.v) + i);
        const float ms = t.ms[block], vs = t.vs[block];
        const auto m0 = __builtin_amdgcn_cvt_pk_f32_fp8(mc, false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8(mc, true);
        const auto v0 = __builtin_amdgcn_cvt_pk_f32_bf8(vc, false), v1 = __builtin_amdgcn_cvt_pk_f32_bf8(vc, true);
        m = f32x4{m0[0] * ms, m0[1] * ms, m1[0] * ms, m1[1] * ms};
        v = f32x4{v0[0] * vs, v0[1] * vs, v1[0] * vs, v1[1] * vs};
    } else {
        m = load_past<f32x4_any>(static_cast<const float*>(t.m) + i);
        v = load_past<f32x4_any>(static_cast<const float*>(t.v) + i);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float pk = p[k], mk = m[k], vk = v[k];
        update<EIGHT>(s, pk, g[k] * gs, mk, vk);
        p[k] = pk, m[k] = mk, v[k] = vk;
    }
    store_past<f32x4_any>(t.p + i, p);
    if (t.copy) *reinterpret_cast<u32x2_any*>(t.copy + i) = u32x2{pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3])};
    if constexpr (!EIGHT) {
        store_past<f32x4_any>(static_cast<float*>(t.m) + i, m);
        store_past<f32x4_any>(static_cast<float*>(t.v) + i, v);
    } else {
        uint32_t mm = 0, vm = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            mm = max(mm, __float_as_uint(m[k]) & 0x7FFFFFFFu);
            vm = max(vm, __float_as_uint(v[k]) & 0x7FFFFFFFu);
        }
        mm = wave_max(mm), vm = wave_max(vm);
        const bool m_fine = mm < 0x7F800000u, v_fine = vm < 0x7F800000u;
        const int me = scale_power<8>(mm), ve = scale_power<15>(vm);
        if (lane == 0) {
            t.ms[block] = m_fine ? power_of_two(me) : NAN;
            t.vs[block] = v_fine ? power_of_two(ve) : NAN;
        }
        const float mi = power_of_two(-me), vi = power_of_two(-ve);
        uint32_t mc = 0, vc = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t h = mix((static_cast<uint32_t>(i) + k) ^ key);
            mc |= to_e4m3(m[k] * mi, h & 0xFFFFu) << (8 * k);
            vc |= max(to_e5m2(v[k] * vi, h >> 16), v[k] > 0.0f ? 1u : 0u) << (8 * k);
        }
        store_past<u32_any>(static_cast<uint8_t*>(t.m) + i, m_fine ? mc : 0x7F7F7F7Fu);
        store_past<u32_any>(static_cast<uint8_t*>(t.v) + i, v_fine ? vc : 0x7F7F7F7Fu);
    }
}
__host__ __device__ inline uint32_t key_of(uint32_t seed, int place) { return mix(seed * 0x9E3779B9u + mix(static_cast<uint32_t>(place) + 0x3C6EF373u)); }

template <typename G, bool EIGHT, bool COPY>
__global__ __launch_bounds__(NT) void adamw_many_k(Table<pointers(EIGHT, COPY)> tab, Step s) {
    const int group = blockIdx.x, j = tab.tensor_of(group);
    One t{tab.template at<float>(j, 0), tab.template at<const void>(j, 1), tab.template at<void>(j, 2), tab.template at<void>(j, 3), nullptr, nullptr, nullptr, tab.elements(j)};
    if constexpr (EIGHT) t.ms = tab.template at<float>(j, 4), t.vs = tab.template at<float>(j, 5);
    if constexpr (COPY) t.copy = tab.template at<uint16_t>(j, EIGHT ? 6 : 4);
    const int64_t blocks = (t.n + BLOCK - 1) / BLOCK, whole = t.n / BLOCK;
    const int64_t begin = static_cast<int64_t>(group - tab.first(j)) * tab.per, end = min(begin + tab.per, blocks);
    const uint32_t key = key_of(tab.seed, tab.place + j);
    const float gs = s.factor ? *s.factor : 1.0f;
    __shared__ float table[EIGHT ? NT : 1];
    Powers p2{table};
    if constexpr (EIGHT) p2 = powers(table);
    for (int64_t k = begin + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); k < end; k += WAVES) {
        if (k < whole)
            block_whole<G, EIGHT>(t, s, key, k, gs, p2);
        else
            block_any<G, EIGHT>(t, s, key, k, gs, p2);
    }
}

// Sums of the gradients' squares in 64 bits, one to a workgroup.
constexpr int SQ_ELEMS = 16384;  // of one tensor that a workgroup takes
template <typename G>
__global__ __launch_bounds__(NT) void squares_k(Table<1> tab, double* part) {
    constexpr int N = 16 / sizeof(G), U = 4;
    __shared__ double sh[WAVES];
    const int group = blockIdx.x, j = tab.tensor_of(group);
    const int64_t begin = static_cast<int64_t>(group - tab.first(j)) * SQ_ELEMS;
    const int count = static_cast<int>(min(tab.elements(j) - begin, static_cast<int64_t>(SQ_ELEMS)));
    const G* g = tab.template at<const G>(j, 0) + begin;
    double q[4] = {0.0, 0.0, 0.0, 0.0};  // chains of additions
    // 16 bytes a lane, four loads on their way
    for (int p0 = threadIdx.x; p0 < count / N; p0 += U * NT) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = p0 + u * NT < count / N ? *reinterpret_cast<const u32x4_any*>(g + (p0 + u * NT) * N) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (N == 4) {
                    const double x = __uint_as_float(v[u][e]);
                    q[e] = fma(x, x, q[e]);
                } else {
                    const double x = __uint_as_float(v[u][e] << 16), y = __uint_as_float(v[u][e] & 0xFFFF0000u);
                    q[e] = fma(y, y, fma(x, x, q[e]));
                }
            }
        }
    }
    for (int i = count / N * N + threadIdx.x; i < count; i += NT) {
        const double x = elem(g, i);
        q[0] = fma(x, x, q[0]);
    }
    double s = (q[0] + q[1]) + (q[2] + q[3]);
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[group] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}
__global__ __launch_bounds__(1024) void factor_k(const double* part, int64_t parts, float max_norm, float* factor, float* norm) {
    __shared__ double sh[16];
    double s = 0.0;
    for (int64_t i0 = threadIdx.x; i0 < parts; i0 += 4 * 1024) {
        double v[4];  // on their way together
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = i0 + k * 1024 < parts ? part[i0 + k * 1024] : 0.0;
        s += (v[0] + v[1]) + (v[2] + v[3]);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
#pragma unroll
    for (int w = 1; w < 16; ++w) s += sh[w];
    const double total = sqrt(s), limit = max_norm;
    *factor = total > limit && total > 0.0 ? static_cast<float>(limit / total) : 1.0f;
    *norm = static_cast<float>(total);
}

int64_t parts_of(const pk_adamw_tensor* t, int count) {
    int64_t n = 0;
    for (int i = 0; i < count; ++i) n += t[i].n > 0 ? (t[i].n + SQ_ELEMS - 1) / SQ_ELEMS : 0;
    return n;
}

// What is wrong with where a list's tensors lie, or null: two of those that are written have memory in common, or a gradient lies over one of them otherwise than over its own
// parameter's, element for element (there a lane reads it before it writes).
const char* misplaced(const pk_adamw_tensor* t, int count, bool eight, size_t grad_size) {
    struct Span {
        uintptr_t from, to;
        int tensor;
        size_t size;  // of an element, 0: scales
        bool operator<(const Span& o) const { return from < o.from; }
    };
    const auto written = [&](int i, int k) {  // nothing: from 0 to 0
        const void* const p = k == 0 ? t[i].p : k == 1 ? t[i].m : k == 2 ? t[i].v : k == 3 ? t[i].m_scale : k == 4 ? t[i].v_scale : t[i].copy;
        if (t[i].n == 0 || !p || ((k == 3 || k == 4) && !eight)) return Span{0, 0, i, 0};
        const size_t size = k == 0 ? 4 : k < 3 ? eight ? 1 : 4 : k < 5 ? 0 : 2;
        const uintptr_t n = static_cast<uintptr_t>(t[i].n), at = reinterpret_cast<uintptr_t>(p);
        return Span{at, at + (size ? size * n : 4 * ((n + BLOCK - 1) / BLOCK)), i, size};
    };
    const auto grad = [&](int i) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(t[i].g);
        return Span{at, at + static_cast<uintptr_t>(t[i].n) * grad_size, i, grad_size};
    };
    // Each list one slab, or in the order of an allocator: the lists' ends say all, where they are apart.
    Span lists[7];
    int n = 0;
    bool clear = true;
    for (int k = 0; k < 6 && clear; ++k) {
        Span all{0, 0, 0, 0};
        for (int i = 0; i < count; ++i) {
            const Span s = written(i, k);
            if (s.to == 0) continue;
            clear = clear && all.to <= s.from;
            all = {all.to ? all.from : s.from, s.to, 0, 0};
        }
        if (all.to) lists[n++] = all;
    }
    Span grads{UINTPTR_MAX, 0, 0, 0};
    for (int i = 0; i < count; ++i)
        if (t[i].n) grads.from = std::min(grads.from, grad(i).from), grads.to = std::max(grads.to, grad(i).to);
    if (clear) {
        if (grads.to) lists[n++] = grads;
        std::sort(lists, lists + n);
        for (int i = 1; i < n; ++i) clear = clear && lists[i - 1].to <= lists[i].from;
    }
    if (clear) return nullptr;
    std::vector<Span> all;
    all.reserve(static_cast<size_t>(count) * 6);
    for (int k = 0; k < 6; ++k)
        for (int i = 0; i < count; ++i)
            if (const Span s = written(i, k); s.to) all.push_back(s);
    std::sort(all.begin(), all.end());
    for (size_t i = 1; i < all.size(); ++i)
        if (all[i].from < all[i - 1].to) return "a parameter, state or copy is in the list twice";
    for (int i = 0; i < count; ++i) {
        if (!t[i].n) continue;
        const Span g = grad(i);
        for (auto w = std::lower_bound(all.begin(), all.end(), g.from, [](const Span& s, uintptr_t from) { return s.to <= from; }); w != all.end() && w->from < g.to; ++w)
            if (w->tensor != i || w->from != g.from || w->size != g.size) return "a gradient lies over a parameter, state or copy otherwise than element for element over its own";
    }
    return nullptr;
}

// Blocks that a workgroup takes. In 32 bits one to a wavefront: 96 tensors of 60000 elements 25.2 us, by 16 27.5; 35 M elements 147 and 154. In 8 bits a workgroup forms the
// powers first, so it takes more where there are enough: 0.5 M elements 8.7 us by 4, 12.5 by 16; 5.8 M 22.9 by 4, 22.1 by 8, 25.5 by 16; 8 M 22.8 by 8, 23.0 by 16;
// 35 M 99, 88 and 85; 120 M 328, 291 and 280.
template <bool EIGHT>
int blocks_of_group(int64_t blocks) {
    if (!EIGHT) return blocks < (1 << 25) ? 4 : 16;  // a launch's threads are counted in 32 bits
    return blocks <= 4 * 4096 ? 4 : blocks <= 8 * 4096 ? 8 : 16;
}
template <typename G, bool EIGHT, bool COPY>
int launch(const pk_adamw_tensor* t, int count, uint32_t seed, const Step& s, hipStream_t st) {
    int64_t blocks = 0;
    for (int i = 0; i < count; ++i) blocks += (t[i].n + BLOCK - 1) / BLOCK;
    const int per = blocks_of_group<EIGHT>(blocks);
    for (int i = 0; i < count;) {
        using List = Table<pointers(EIGHT, COPY)>;
        List tab;
        int64_t groups = 0;
        tab.place = i, tab.seed = seed, tab.per = per;
        for (tab.count = 0; i < count && tab.count < List::MOST; ++i, ++tab.count) {
            const pk_adamw_tensor& x = t[i];
            if constexpr (EIGHT && COPY)
                tab.put(tab.count, x.n, groups, {x.p, x.g, x.m, x.v, x.m_scale, x.v_scale, x.copy});
            else if constexpr (EIGHT)
                tab.put(tab.count, x.n, groups, {x.p, x.g, x.m, x.v, x.m_scale, x.v_scale});
            else if constexpr (COPY)
                tab.put(tab.count, x.n, groups, {x.p, x.g, x.m, x.v, x.copy});
            else
                tab.put(tab.count, x.n, groups, {x.p, x.g, x.m, x.v});
            groups += (x.n + BLOCK * per - 1) / (BLOCK * per);
        }
        if (groups == 0) continue;
        adamw_many_k<G, EIGHT, COPY><<<dim3(static_cast<unsigned>(groups)), NT, 0, st>>>(tab, s);
        if (int rc = launched()) return rc;
    }
    return PK_OK;
}
template <typename G>
int run(const pk_adamw_tensor* t, int count, const pk_adamw_config* c, void* workspace, float* norm, hipStream_t st) {
    Step s;
    s.lr = c->lr, s.b1 = c->b1, s.b2 = c->b2, s.eps = c->eps, s.wd = c->wd;
    s.rest1 = 1.0f - c->b1, s.rest2 = 1.0f - c->b2;
    s.per_c1 = static_cast<float>(1.0 / (1.0 - std::pow(static_cast<double>(c->b1), c->t)));
    s.per_c2 = static_cast<float>(1.0 / (1.0 - std::pow(static_cast<double>(c->b2), c->t)));
    s.factor = nullptr;
    if (c->max_norm > 0.0f) {
        float* factor = static_cast<float*>(workspace);
        double* part = reinterpret_cast<double*>(static_cast<char*>(workspace) + 256);
        int64_t parts = 0;
        for (int i = 0; i < count;) {
            Table<1> q;
            int64_t groups = 0;
            for (q.count = 0; i < count && q.count < Table<1>::MOST; ++i, ++q.count) {
                q.put(q.count, t[i].n, groups, {t[i].g});
                groups += (t[i].n + SQ_ELEMS - 1) / SQ_ELEMS;
            }
            if (groups == 0) continue;
            squares_k<G><<<dim3(static_cast<unsigned>(groups)), NT, 0, st>>>(q, part + parts);
            if (int rc = launched()) return rc;
            parts += groups;
        }
        factor_k<<<1, 1024, 0, st>>>(part, parts, c->max_norm, factor, norm);
        if (int rc = launched()) return rc;
        s.factor = factor;
    }
    bool copies = false;
    for (int i = 0; i < count; ++i) copies = copies || t[i].copy;
    if (c->state_bits == 8) return copies ? launch<G, true, true>(t, count, c->seed, s, st) : launch<G, true, false>(t, count, c->seed, s, st);
    return copies ? launch<G, false, true>(t, count, c->seed, s, st) : launch<G, false, false>(t, count, c->seed, s, st);
}

}  // namespace
}  // namespace pk

using namespace pk;

extern "C" {

size_t pk_adamw_many_workspace_bytes(const pk_adamw_tensor* tensors, int count, const pk_adamw_config* c) {
    if (!c || count < 0 || (count > 0 && !tensors) || !(c->max_norm > 0.0f)) return 0;
    return 256 + sizeof(double) * static_cast<size_t>(parts_of(tensors, count));
}

int pk_adamw_many(const pk_adamw_tensor* t, int count, const pk_adamw_config* c, void* workspace, size_t workspace_bytes, float* norm, void* stream) {
    return c_entry([&] {
        if (!c || count < 0 || (count > 0 && !t)) return fail(PK_ERR_ARGUMENT, "pk_adamw_many: null table");
        if (c->t < 1) return fail(PK_ERR_ARGUMENT, "pk_adamw_many: step count starts at 1");
        if (c->state_bits != 8 && c->state_bits != 32) return fail(PK_ERR_ARGUMENT, "pk_adamw_many: states are held in 8 or in 32 bits");
        if (!known_dtype(c->grad_dtype)) return fail(PK_ERR_ARGUMENT, "pk_adamw_many: dtype must be PK_F32 or PK_BF16");
        if (!(c->b1 >= 0.0f && c->b1 < 1.0f && c->b2 >= 0.0f && c->b2 < 1.0f)) return fail(PK_ERR_ARGUMENT, "pk_adamw_many: b1 and b2 lie in [0, 1)");
        if (c->max_norm != c->max_norm) return fail(PK_ERR_ARGUMENT, "pk_adamw_many: max_norm is no number");
        const bool clip = c->max_norm > 0.0f;
        int64_t total = 0;  // a launch has fewer than 2^32 threads, 16 elements each
        for (int i = 0; i < count; ++i) {
            total += t[i].n > 0 ? t[i].n : 0;
            if (t[i].n < 0 || total > (int64_t{1} << 35)) return fail(PK_ERR_SHAPE, "pk_adamw_many: a tensor's size is out of range");
            if (t[i].n > 0 && (!t[i].p || !t[i].g || !t[i].m || !t[i].v || (c->state_bits == 8 && (!t[i].m_scale || !t[i].v_scale))))
                return fail(PK_ERR_ARGUMENT, "pk_adamw_many: null pointer");
            for (const void* p : {static_cast<const void*>(t[i].p), t[i].g, static_cast<const void*>(t[i].m), static_cast<const void*>(t[i].v), static_cast<const void*>(t[i].m_scale),
                                  static_cast<const void*>(t[i].v_scale), static_cast<const void*>(t[i].copy)})
                if (reinterpret_cast<uint64_t>(p) >> 48) return fail(PK_ERR_ARGUMENT, "pk_adamw_many: an address past 48 bits");
        }
        if (const char* why = misplaced(t, count, c->state_bits == 8, static_cast<size_t>(elem_size(c->grad_dtype)))) return fail(PK_ERR_ARGUMENT, std::string("pk_adamw_many: ") + why);
        if (clip && !norm) return fail(PK_ERR_ARGUMENT, "pk_adamw_many: a clip writes the norm");
        if (clip && (!workspace || !aligned(workspace, 8) || workspace_bytes < pk_adamw_many_workspace_bytes(t, count, c)))
            return fail(PK_ERR_WORKSPACE, "pk_adamw_many: workspace too small (pk_adamw_many_workspace_bytes)");
        std::vector<const void*> used;
        used.reserve(7 * static_cast<size_t>(count) + 2);
        for (int i = 0; i < count; ++i) used.insert(used.end(), {t[i].p, t[i].g, t[i].m, t[i].v, t[i].m_scale, t[i].v_scale, t[i].copy});
        used.insert(used.end(), {workspace, norm});
        dev_touch(used.data(), used.size(), stream);
        hipStream_t st = static_cast<hipStream_t>(stream);
        return c->grad_dtype == PK_BF16 ? run<uint16_t>(t, count, c, workspace, norm, st) : run<float>(t, count, c, workspace, norm, st);
    });
}

}  // extern "C"
