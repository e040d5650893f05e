// One AdamW step over a list of tensors, with the global gradient norm's clip in front of it, the moments in 32 bits or in 8.
//
//   g' = g min(1, max_norm / |g|)    m' = b1 m + (1 - b1) g'    v' = b2 v + (1 - b2) g'^2    p -= lr ((m' / c1) / (sqrt(v' / c2) + eps) + wd p)
//
// In 8 bits m is e4m3 and v e5m2 with a power of two for every 256 elements of a tensor, the largest that keeps the block's largest value inside the
// format: scaling then rounds nothing. v' moves by a thousandth of itself in a step, far less than the 1/8 between neighbours of its format, so
// rounding to the nearest would leave it where it is for ever; both moments are rounded up with the probability that the bits dropped stand for,
// from a hash of the seed, the tensor's place in the list and the element's place in it. The same call gives the same bits. A v that is not zero
// does not become zero: m / sqrt(v) would have no bound. A block that holds a value which is not finite becomes NaN as a whole.
//
// m' and v' are formed without fused operations (each product and sum rounded by itself): a state in 8 bits is then one function of its inputs in
// any program that follows these formulas, and not of how a compiler contracts them.
//
// What bounds it: memory: 4 to 6 words read and 3 written an element with moments in 32 bits, 16 bytes in all with those in 8.
#include "post.h"

#include <algorithm>
#include <vector>

#pragma clang fp contract(off)

namespace pk {
namespace {

constexpr int BLOCK = 256, NT = 256, WAVES = NT / 64;  // elements that share a scale; a wavefront takes a block
constexpr int MAX_TENSORS = 48;                         // of one launch: the table travels in the kernel's arguments (4 KB at most)
constexpr int BLOCKS_PER_WG = 16;

struct One {
    float* p;
    const void* g;
    void *m, *v;
    float *ms, *vs;
    uint16_t* copy;
    int64_t n;
};
struct Table {
    int first[MAX_TENSORS + 1];  // a tensor's first workgroup
    uint32_t key[MAX_TENSORS];
    One t[MAX_TENSORS];
};
static_assert(sizeof(Table) + 128 <= 4096, "kernel arguments");
struct Step {
    float lr, b1, b2, rest1, rest2, eps, wd, c1, c2;
    const float* factor;  // what the gradients are multiplied by, or null
};

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
__device__ inline float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

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

__device__ inline void update(const Step& s, float& p, float g, float& m, float& v) {
    const float a = s.b1 * m, b = s.rest1 * g, c = s.b2 * v, d = s.rest2 * g, e = d * g;
    m = a + b;
    v = c + e;
    p -= s.lr * ((m / s.c1) / (sqrtf(v / s.c2) + s.eps) + s.wd * p);
}

// A wavefront takes a block of 256 elements, a lane its elements lane, lane + 64, lane + 128 and lane + 192.
template <typename G, bool EIGHT>
__device__ inline void block_any(const One& t, const Step& s, uint32_t key, int64_t block, float gs) {
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
        update(s, p[k], g, m[k], v[k]);
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

// The tensor that a workgroup belongs to: the last one whose first workgroup is not behind it.
__device__ inline int tensor_of(const int* first, int count, int group) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (first[mid] <= group)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

template <typename G, bool EIGHT>
__global__ __launch_bounds__(NT) void adamw_many_k(Table tab, Step s, int count) {
    const int group = blockIdx.x, j = tensor_of(tab.first, count, group);
    const One t = tab.t[j];
    const int64_t blocks = (t.n + BLOCK - 1) / BLOCK, begin = static_cast<int64_t>(group - tab.first[j]) * BLOCKS_PER_WG;
    const float gs = s.factor ? *s.factor : 1.0f;
    for (int k = threadIdx.x >> 6; k < BLOCKS_PER_WG && begin + k < blocks; k += WAVES) block_any<G, EIGHT>(t, s, tab.key[j], begin + k, gs);
}

// Sums of the gradients' squares in 64 bits, one to a workgroup.
constexpr int SQ_ELEMS = 16384;  // of one tensor that a workgroup takes
struct Squares {
    int first[MAX_TENSORS + 1];
    const void* g[MAX_TENSORS];
    int64_t n[MAX_TENSORS];
};
template <typename G>
__global__ __launch_bounds__(NT) void squares_k(Squares tab, int count, double* part) {
    __shared__ double sh[WAVES];
    const int group = blockIdx.x, j = tensor_of(tab.first, count, group);
    const int64_t begin = static_cast<int64_t>(group - tab.first[j]) * SQ_ELEMS, end = min(tab.n[j], begin + SQ_ELEMS);
    const G* g = static_cast<const G*>(tab.g[j]);
    double s = 0.0;
    for (int64_t i = begin + threadIdx.x; i < end; i += NT) {
        const double x = elem(g, i);
        s += x * x;
    }
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[group] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}
__global__ __launch_bounds__(1024) void factor_k(const double* part, int64_t parts, float max_norm, float* factor, float* norm) {
    __shared__ double sh[16];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < parts; i += 1024) s += part[i];
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
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

template <typename G>
int run(const pk_adamw_tensor* t, int count, const pk_adamw_config* c, void* workspace, float* norm, hipStream_t st) {
    Step s;
    s.lr = c->lr, s.b1 = c->b1, s.b2 = c->b2, s.eps = c->eps, s.wd = c->wd;
    s.rest1 = 1.0f - c->b1, s.rest2 = 1.0f - c->b2;
    s.c1 = static_cast<float>(1.0 - std::pow(static_cast<double>(c->b1), c->t));
    s.c2 = static_cast<float>(1.0 - std::pow(static_cast<double>(c->b2), c->t));
    s.factor = nullptr;
    if (c->max_norm > 0.0f) {
        float* factor = static_cast<float*>(workspace);
        double* part = reinterpret_cast<double*>(static_cast<char*>(workspace) + 256);
        int64_t parts = 0;
        for (int i = 0; i < count;) {
            Squares q;
            int used = 0, groups = 0;
            for (; i < count && used < MAX_TENSORS; ++i) {
                if (t[i].n == 0) continue;
                const int64_t more = (t[i].n + SQ_ELEMS - 1) / SQ_ELEMS;
                q.first[used] = groups, q.g[used] = t[i].g, q.n[used] = t[i].n;
                groups += static_cast<int>(more), ++used;
            }
            if (!used) break;
            squares_k<G><<<dim3(groups), NT, 0, st>>>(q, used, part + parts);
            if (int rc = launched()) return rc;
            parts += groups;
        }
        factor_k<<<1, 1024, 0, st>>>(part, parts, c->max_norm, factor, norm);
        if (int rc = launched()) return rc;
        s.factor = factor;
    }
    for (int i = 0; i < count;) {
        Table tab;
        int used = 0;
        int64_t groups = 0;
        for (; i < count && used < MAX_TENSORS; ++i) {
            if (t[i].n == 0) continue;
            tab.first[used] = static_cast<int>(groups);
            tab.key[used] = mix(static_cast<uint32_t>(c->seed) * 0x9E3779B9u + mix(static_cast<uint32_t>(i) + 0x3C6EF373u));
            tab.t[used] = One{t[i].p, t[i].g, t[i].m, t[i].v, t[i].m_scale, t[i].v_scale, static_cast<uint16_t*>(t[i].copy), t[i].n};
            groups += (t[i].n + BLOCK * BLOCKS_PER_WG - 1) / (BLOCK * BLOCKS_PER_WG), ++used;
        }
        if (!used) break;
        if (c->state_bits == 8)
            adamw_many_k<G, true><<<dim3(static_cast<unsigned>(groups)), NT, 0, st>>>(tab, s, used);
        else
            adamw_many_k<G, false><<<dim3(static_cast<unsigned>(groups)), NT, 0, st>>>(tab, s, used);
        if (int rc = launched()) return rc;
    }
    return PK_OK;
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
        const bool clip = c->max_norm > 0.0f;
        std::vector<std::pair<uintptr_t, uintptr_t>> written;
        written.reserve(3 * static_cast<size_t>(count));
        for (int i = 0; i < count; ++i) {
            if (t[i].n < 0 || t[i].n > (int64_t{1} << 40)) return fail(PK_ERR_SHAPE, "pk_adamw_many: a tensor's size is out of range");
            if (t[i].n == 0) continue;
            if (!t[i].p || !t[i].g || !t[i].m || !t[i].v || (c->state_bits == 8 && (!t[i].m_scale || !t[i].v_scale)))
                return fail(PK_ERR_ARGUMENT, "pk_adamw_many: null pointer");
            const uintptr_t n = static_cast<uintptr_t>(t[i].n), e = n * (c->state_bits / 8);
            const uintptr_t p = reinterpret_cast<uintptr_t>(t[i].p), m = reinterpret_cast<uintptr_t>(t[i].m), v = reinterpret_cast<uintptr_t>(t[i].v);
            written.push_back({p, p + 4 * n}), written.push_back({m, m + e}), written.push_back({v, v + e});
        }
        std::sort(written.begin(), written.end());
        for (size_t i = 1; i < written.size(); ++i)
            if (written[i].first < written[i - 1].second) return fail(PK_ERR_ARGUMENT, "pk_adamw_many: a parameter or state is in the list twice");
        if (clip && !norm) return fail(PK_ERR_ARGUMENT, "pk_adamw_many: a clip writes the norm");
        if (clip && (!workspace || !aligned(workspace, 8) || workspace_bytes < pk_adamw_many_workspace_bytes(t, count, c)))
            return fail(PK_ERR_WORKSPACE, "pk_adamw_many: workspace too small (pk_adamw_many_workspace_bytes)");
        for (int i = 0; i < count; ++i)
            for (const void* p : {static_cast<const void*>(t[i].p), t[i].g, static_cast<const void*>(t[i].m), static_cast<const void*>(t[i].v),
                                  static_cast<const void*>(t[i].m_scale), static_cast<const void*>(t[i].v_scale), static_cast<const void*>(t[i].copy)})
                if (p) dev_touch(p, stream);
        hipStream_t st = static_cast<hipStream_t>(stream);
        return c->grad_dtype == PK_BF16 ? run<uint16_t>(t, count, c, workspace, norm, st) : run<float>(t, count, c, workspace, norm, st);
    });
}

}  // extern "C"
