// Queries and keys on their way into attention: every head's row normalised by its root mean square, multiplied by a weight of the head size and
// turned pair by pair by its token's position, in one pass over both tensors, and the gradients of that.
//
//   r = 1 / sqrt(mean_j x_j^2 + eps)      u_j = x_j r w_j      (y_a, y_b) = (u_a cos t - u_b sin t, u_a sin t + u_b cos t),  t = pos theta^(-2i/R)
//   du = y's gradient turned back         dw_j = sum over rows of du_j x_j r       dx_j = r (w_j du_j - x_j r^2 mean_i(w_i du_i x_i))
//
// What bounds it: memory. The forward reads and writes each element once, the backward reads two and writes one; r is formed again there instead of
// being kept, because the row is in registers anyway. The angle is formed in 64 bits, in turns, and its whole turns are dropped there: at position
// 10^6 an angle in 32 bits is 0.06 rad off. Rounded to 32 bits after that it is 1e-7 rad off up to position 2^26, 1.6e-7 at 2^28, 4.3e-7 at 2^31 (theta 10^4 to 10^6, 64 to 256 columns).
#include "post.h"

#include <algorithm>

namespace pk {
namespace {

// Workgroups of a launch. Forward of 16384 tokens, 32 heads of 128: 53.3 us on 1024, 51.3 on 2048, 47.5 on 4096. Each of the backward's leaves sums of dw, and four to a
// CU fill its registers: backward of 8192 tokens, 14 + 2 heads of 64, four tokens to a wavefront, 16.9 us on 512, 15.2 on 1024, 15.3 on 2048; 16 + 16 heads of 64, a token to a
// wavefront, 24.2, 21.7 and 23.5; 16384 tokens, 16 + 16 heads of 128 90.7, 83.0 and 85.0.
constexpr int FWD_MOST = 4096, BWD_MOST = 1024;
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
    int pack;             // row kernels: a wavefront takes 2^pack tokens at a time
    float eps, per_dk;        // 1 / dk
    // Turns that a position moves pair p by, theta^(-2p/R) / 2 pi, as coarse[p / 8] * fine[p % 8]: two factors that are rounded once each.
    double coarse[MAX_PAIRS / 8], fine[8];
};

__device__ inline double turns_of(const Qk& a, int pair) { return a.coarse[pair >> 3] * a.fine[pair & 7]; }

// cos and sin of a position's angle. The angle is taken to the nearest quarter turn, r eighths of a turn and less from it (both exact), and the two series
// run there: their first terms left out are (pi/4)^11 / 11! = 2e-9 and (pi/4)^10 / 10! = 2.5e-8, under half a step of 32 bits. Half of the instructions of
// sincospif.
__device__ inline void cos_sin(int pos, double turns, float& c, float& s) {
    const double t = pos * turns;
    const float f = static_cast<float>(t - rint(t)), q = rintf(4.0f * f);
    const float x = fmaf(-0.25f, q, f) * 6.28318530717958647693f, z = x * x;
    const float sine = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), x);
    const float cosine = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 40320, -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const int k = static_cast<int>(q);  // quarter turns, -2 .. 2
    const bool swap = k & 1;
    c = swap ? sine : cosine, s = swap ? cosine : sine;
    c = __uint_as_float(__float_as_uint(c) ^ (static_cast<uint32_t>(k + 1) & 2u) << 30);
    s = __uint_as_float(__float_as_uint(s) ^ (static_cast<uint32_t>(k) & 2u) << 30);
}
// 1 / sqrt(x), x >= 0, to a step of 32 bits; small x are scaled into the range of the instruction
__device__ inline float inverse_root(float x) {
    const bool small = x < 0x1p-100f;
    const float r = __builtin_amdgcn_rsqf(small ? x * 0x1p100f : x);
    return small ? r * 0x1p50f : r;
}

// The two columns of pair p: of the first `rotary` ones neighbours, or one from each half; behind them neighbours, which are not turned.
__device__ inline void columns(int p, int rotary, bool halves, int& a, int& b) {
    const bool turned = halves && p < rotary / 2;
    a = turned ? p : 2 * p;
    b = turned ? p + rotary / 2 : 2 * p + 1;
}

// What the row kernels below do not serve: a wavefront takes a row, a lane its pairs lane and lane + 64.
template <typename T>
__global__ __launch_bounds__(NT) void qk_fwd_any(Qk a) {
    const int lane = threadIdx.x & 63, heads = a.Hq + a.Hkv, pairs = a.dk / 2;
    const int64_t items = static_cast<int64_t>(a.B) * a.T * heads, stride = static_cast<int64_t>(gridDim.x) * WAVES;
    const double turns[2] = {turns_of(a, lane), turns_of(a, lane + 64)};
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
        const float r = inverse_root(group_sum<64>(ss) * a.per_dk + a.eps);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int p = lane + 64 * k;
            if (p >= pairs) continue;
            const float ua = xa[k] * r * a.w[which][ca[k]], ub = xb[k] * r * a.w[which][cb[k]];
            if (p < a.rotary / 2) {
                float c, s;
                cos_sin(pos, turns[k], c, s);
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
    const double turns[2] = {turns_of(a, lane), turns_of(a, lane + 64)};
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
                cos_sin(pos, turns[k], c, s);
                ga[k] = da * c + db * s;
                gb[k] = db * c - da * s;
            }
            ss += xa[k] * xa[k] + xb[k] * xb[k];
            sg += wa[k] * ga[k] * xa[k] + wb[k] * gb[k] * xb[k];
        }
        const float r = inverse_root(group_sum<64>(ss) * a.per_dk + a.eps), m = r * r * (group_sum<64>(sg) * a.per_dk);
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

// ---- rows in 16-byte pieces ------------------------------------------------------------------------------------------
// A group of G lanes takes a head's row, a lane eight of its columns as four pairs (a[i], b[i]): columns 8l .. 8l+7, or, where pairs come from two
// halves, columns 4l .. and R/2 + 4l .., so that a pair never leaves its lane. A wavefront holds 64 / G rows of one token, or of a few, at a time and walks the
// token's heads, queries and keys as one list. The angles are the token's: 64 lanes form one pair's each and hand them round through a strip of LDS.

struct Eight {  // vectors: as arrays the compiler kept half of one in LDS, by an offset that it read from the launch's packet in the host's memory (gqa forward 8.5 -> 22 us)
    f32x4 a, b;
};
// Vectors that lie where their elements may. The hardware takes them anywhere; what it costs stands at `serve`.
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
template <typename T, bool HALVES, bool LOOSE>
struct Cols;  // how a lane's columns are moved: two runs of four, c0 and c1 bytes behind the base
template <bool HALVES, bool LOOSE>
struct Cols<uint16_t, HALVES, LOOSE> {
    using Four = std::conditional_t<LOOSE, u32x4_any, u32x4>;
    using Two = std::conditional_t<LOOSE, u32x2_any, u32x2>;
    struct Raw {
        u32x4 v;
    };
    __device__ static Raw load(const char* row, uint32_t c0, uint32_t c1) {
        if constexpr (HALVES) {
            const u32x2 x = *reinterpret_cast<const Two*>(row + c0), y = *reinterpret_cast<const Two*>(row + c1);
            return Raw{{x[0], x[1], y[0], y[1]}};
        } else {
            return Raw{*reinterpret_cast<const Four*>(row + c0)};
        }
    }
    __device__ static Eight unpack(const Raw& r) {
        Eight e;
        const auto lo = [](uint32_t u) { return __uint_as_float(u << 16); };
        const auto hi = [](uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (HALVES) {
                e.a[i] = i & 1 ? hi(r.v[i / 2]) : lo(r.v[i / 2]);
                e.b[i] = i & 1 ? hi(r.v[2 + i / 2]) : lo(r.v[2 + i / 2]);
            } else {
                e.a[i] = lo(r.v[i]), e.b[i] = hi(r.v[i]);
            }
        }
        return e;
    }
    __device__ static void store(char* row, uint32_t c0, uint32_t c1, const Eight& e) {
        if constexpr (HALVES) {
            *reinterpret_cast<Two*>(row + c0) = u32x2{pack_bf16(e.a[0], e.a[1]), pack_bf16(e.a[2], e.a[3])};
            *reinterpret_cast<Two*>(row + c1) = u32x2{pack_bf16(e.b[0], e.b[1]), pack_bf16(e.b[2], e.b[3])};
        } else {
            const u32x4 v = {pack_bf16(e.a[0], e.b[0]), pack_bf16(e.a[1], e.b[1]), pack_bf16(e.a[2], e.b[2]), pack_bf16(e.a[3], e.b[3])};
            if constexpr (LOOSE)
                *reinterpret_cast<Four*>(row + c0) = v;
            else
                store_through(reinterpret_cast<u32x4*>(row + c0), v);  // whole lines: rows of 64 columns and more
        }
    }
};
template <bool HALVES, bool LOOSE>
struct Cols<float, HALVES, LOOSE> {
    using Four = std::conditional_t<LOOSE, f32x4_any, f32x4>;
    struct Raw {
        f32x4 x, y;
    };
    __device__ static Raw load(const char* row, uint32_t c0, uint32_t c1) {
        return Raw{*reinterpret_cast<const Four*>(row + c0), *reinterpret_cast<const Four*>(row + c1)};
    }
    __device__ static Eight unpack(const Raw& r) {
        Eight e;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (HALVES)
                e.a[i] = r.x[i], e.b[i] = r.y[i];
            else
                e.a[i] = i < 2 ? r.x[2 * i] : r.y[2 * i - 4], e.b[i] = i < 2 ? r.x[2 * i + 1] : r.y[2 * i - 3];
        }
        return e;
    }
    __device__ static void store(char* row, uint32_t c0, uint32_t c1, const Eight& e) {
        if constexpr (HALVES) {
            *reinterpret_cast<Four*>(row + c0) = f32x4{e.a[0], e.a[1], e.a[2], e.a[3]};
            *reinterpret_cast<Four*>(row + c1) = f32x4{e.b[0], e.b[1], e.b[2], e.b[3]};
        } else {
            *reinterpret_cast<Four*>(row + c0) = f32x4{e.a[0], e.b[0], e.a[1], e.b[1]};
            *reinterpret_cast<Four*>(row + c1) = f32x4{e.a[2], e.b[2], e.a[3], e.b[3]};
        }
    }
};
// What lane l of a row's group holds: two runs of four columns from c0 and c1 on, pairs p0 .. p0 + 3 where they are turned.
//
// LOOSE: any even head size from 8 on, any number of turned columns. A run that would pass its end is moved back to it, so the lane holds columns of its neighbour's, too:
// those count in no sum (ka, kb 0), and are not stored. With pairs of halves the turned columns and those behind them are dealt out one after the other.
template <bool LOOSE>
struct Share {
    int c0, c1, p0;
    bool mine;
};
template <>
struct Share<true> : Share<false> {
    f32x4 ka, kb;
    bool whole;
};
__host__ __device__ inline int turned_lanes(int rotary) { return (rotary + 7) / 8; }
__host__ __device__ inline int lanes_wanted(int dk, int rotary, bool halves) { return halves ? turned_lanes(rotary) + (dk - rotary + 7) / 8 : (dk + 7) / 8; }
template <int G, bool HALVES, bool LOOSE>
__device__ inline Share<LOOSE> share(int l, int dk, int rotary) {
    Share<LOOSE> r;
    if constexpr (!LOOSE) {
        r.mine = 8 * l < dk;
        l = r.mine ? l : 0;
        const bool turned = HALVES && 8 * l < rotary;
        r.c0 = turned ? 4 * l : 8 * l;
        r.c1 = turned ? rotary / 2 + 4 * l : 8 * l + 4;
        r.p0 = 4 * l;
    } else {
        r.mine = l < lanes_wanted(dk, rotary, HALVES);
        const int half = rotary / 2, turned = turned_lanes(rotary);
        if (HALVES && l < turned) {
            r.p0 = max(0, min(4 * l, half - 4));
            r.c0 = r.p0, r.c1 = half + r.p0;
#pragma unroll
            for (int i = 0; i < 4; ++i) r.ka[i] = r.kb[i] = r.p0 + i >= 4 * l && r.p0 + i < half ? 1.0f : 0.0f;
        } else {
            const int from = HALVES ? rotary + 8 * (l - turned) : 8 * l;
            r.c0 = min(from, dk - 8), r.c1 = r.c0 + 4;
            r.p0 = HALVES ? 4 * G - 4 : r.c0 / 2;  // with halves the last four angles of the strip, which are none
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                r.ka[i] = r.c0 + (HALVES ? i : 2 * i) >= from ? 1.0f : 0.0f;
                r.kb[i] = r.c0 + (HALVES ? 4 + i : 2 * i) >= from ? 1.0f : 0.0f;
            }
        }
        r.whole = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!r.mine) r.ka[i] = r.kb[i] = 0.0f;
            r.whole = r.whole && r.ka[i] != 0.0f && r.kb[i] != 0.0f;
        }
        if (!r.mine) r.c0 = r.p0 = 0, r.c1 = 4;
    }
    return r;
}
// Column of a[i] and of b[i].
template <bool HALVES>
__device__ inline int column_a(int c0, int c1, int i) { return HALVES ? c0 + i : i < 2 ? c0 + 2 * i : c1 + 2 * i - 4; }
template <bool HALVES>
__device__ inline int column_b(int c0, int c1, int i) { return HALVES ? c1 + i : i < 2 ? c0 + 2 * i + 1 : c1 + 2 * i - 3; }
// The cosines and sines of a lane's four pairs, p0 and on; a pair that is not turned has 1 and 0.
struct Angles {
    f32x4 c, s;
};
// `pos`: the position of the wavefront's first token. A lane forms pairs of all its tokens in turn; p0 counts over all of them.
template <int G, bool PACKED>
__device__ inline Angles angles(const Qk& a, const int* pos, int tokens, int p0, double near, double far, float2* strip) {
    const int lane = threadIdx.x & 63;
    __builtin_amdgcn_wave_barrier();
    if constexpr (!PACKED) {
        const int at = *pos;
#pragma unroll
        for (int k = 0; k < (G + 15) / 16; ++k) {  // 4 G pairs, 64 lanes
            const int p = lane + 64 * k;
            float c = 1.0f, s = 0.0f;
            if (p < a.rotary / 2) cos_sin(at, k ? far : near, c, s);
            if (p < 4 * G) strip[p] = make_float2(c, s);
        }
    } else {
        const int p = lane % (4 * G);
#pragma unroll 1
        for (int k = 0; 64 * k < 4 * G << a.pack; ++k) {
            const int e = lane + 64 * k, token = e / (4 * G);
            float c = 1.0f, s = 0.0f;
            if ((G > 16 ? e % (4 * G) : p) < a.rotary / 2) cos_sin(pos[min(token, tokens - 1)], G > 16 && (k & 1) ? far : near, c, s);
            if (e < 4 * G << a.pack) strip[e] = make_float2(c, s);
        }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();  // the strip is this wavefront's, whose LDS operations are in order
    Angles r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = strip[p0 + i];
        r.c[i] = v.x, r.s[i] = v.y;
    }
    return r;
}
template <bool HALVES>
__device__ inline Eight weights_of(const float* w, int c0, int c1) {
    Eight e;
#pragma unroll
    for (int i = 0; i < 4; ++i) e.a[i] = w[column_a<HALVES>(c0, c1, i)], e.b[i] = w[column_b<HALVES>(c0, c1, i)];
    return e;
}

// A wavefront takes 2^a.pack tokens, neighbours in a sequence, and of each a list of rows, 64 / G to a step over all of them, the queries' steps first, then the keys'. What
// a step needs is the wavefront's (scalars) but for the lane's offset, and the next step's loads are on their way while one is worked on: with four steps unrolled the
// compiler formed every address ahead of the loop, 2600 instructions in place of 500. Scalars that do not fit pass through lanes of vector registers: none or a few of the forward's, 13 to 31 of the
// backward's, 55 to 78 of it where a wavefront takes several tokens.
template <typename T, int G, bool HALVES, bool LOOSE, bool PACKED>
struct List : Share<LOOSE> {
    using C = Cols<T, HALVES, LOOSE>;
    using Share<LOOSE>::c0;
    using Share<LOOSE>::c1;
    static constexpr int ROWS = 64 / G;
    static constexpr uint32_t SIZE = sizeof(T);
    int row, token, each, q_steps, steps;  // the lane's place in a step; rows of a token in it
    __device__ List(const Qk& a) : Share<LOOSE>(share<G, HALVES, LOOSE>((threadIdx.x & 63) % G, a.dk, a.rotary)) {
        const int g = (threadIdx.x & 63) / G;
        const int bits = (G == 4 ? 4 : G == 8 ? 3 : G == 16 ? 2 : 1) - (PACKED ? a.pack : 0);  // each is a power of two
        each = 1 << bits;
        token = PACKED ? g >> bits : 0, row = g & (each - 1);
        q_steps = (a.Hq + each - 1) >> bits;
        steps = q_steps + ((a.Hkv + each - 1) >> bits);
    }
    struct Step {
        bool key;
        int head;   // its first
        bool live;  // whether the lane's group has a row in it
    };
    __device__ Step step(const Qk& a, int s, int tokens) const {
        const bool key = s >= q_steps;
        const int head = (key ? s - q_steps : s) * each;
        return Step{key, head, head + row < (key ? a.Hkv : a.Hq) && (!PACKED || token < tokens)};
    }
    // What a lane's row lies behind the step's first one by, in bytes, in queries and keys. With one token it is formed where it is used: two registers fewer a tensor.
    struct Lane {
        uint32_t q, k;
    };
    template <typename P>
    __device__ Lane lane(const P (&x)[2]) const {
        if constexpr (!PACKED) return Lane{0, 0};
        return Lane{(row * static_cast<uint32_t>(x[0].sh) + token * static_cast<uint32_t>(x[0].st)) * SIZE,
                    (row * static_cast<uint32_t>(x[1].sh) + token * static_cast<uint32_t>(x[1].st)) * SIZE};
    }
    // the lane's row; groups without one take the step's first
    template <typename P>
    __device__ const char* at(const P (&x)[2], const Step& s, int64_t oq, int64_t ok, const Lane& lane, uint32_t& off) const {
        const int64_t sh = s.key ? x[1].sh : x[0].sh;
        if constexpr (PACKED)
            off = s.live ? s.key ? lane.k : lane.q : 0u;
        else
            off = s.live ? static_cast<uint32_t>(row) * static_cast<uint32_t>(sh * SIZE) : 0u;
        return static_cast<const char*>(s.key ? x[1].p : x[0].p) + ((s.key ? ok : oq) + s.head * sh) * static_cast<int64_t>(SIZE);
    }
    __device__ typename C::Raw load(const Rows (&x)[2], const Step& s, int64_t oq, int64_t ok, const Lane& lane) const {
        uint32_t off;
        const char* base = at(x, s, oq, ok, lane, off);
        return C::load(base, off + c0 * SIZE, off + c1 * SIZE);
    }
    __device__ void store(const RowsOut (&y)[2], const Step& s, int64_t oq, int64_t ok, const Lane& lane, const Eight& e) const {
        uint32_t off;
        char* base = const_cast<char*>(at(y, s, oq, ok, lane, off));
        if constexpr (LOOSE) {
            T* to = reinterpret_cast<T*>(base + off);
            if (!this->whole) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (this->ka[i] != 0.0f) put(to, column_a<HALVES>(c0, c1, i), e.a[i]);
                    if (this->kb[i] != 0.0f) put(to, column_b<HALVES>(c0, c1, i), e.b[i]);
                }
            }
            if (this->whole) {
                C::store(base, off + c0 * SIZE, off + c1 * SIZE, e);
                asm volatile("s_nop 1");  // no path needs it: the check of 16-byte stores reads the kernel's text in order, and the block behind the branch writes the data's registers
            }
        } else {
            C::store(base, off + c0 * SIZE, off + c1 * SIZE, e);
        }
    }
};

// grid.x: wavefronts' tokens, WAVES to a workgroup, in strides of the grid; grid.y: `per` steps of a token's list each.
template <typename T, int G, bool HALVES, bool LOOSE, bool PACKED>
__global__ __launch_bounds__(NT) void qk_fwd_rows(Qk a, int per) {
    using L = List<T, G, HALVES, LOOSE, PACKED>;
    __shared__ float2 strips[WAVES][PACKED ? 256 : 4 * G];  // 64 / G tokens at most
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), stride = static_cast<int>(gridDim.x) * WAVES;
    const L list(a);
    const Eight wq = weights_of<HALVES>(a.w[0], list.c0, list.c1), wk = weights_of<HALVES>(a.w[1], list.c0, list.c1);
    const auto lx = list.lane(a.x), ly = list.lane(a.y);
    const double near = turns_of(a, lane % (4 * G)), far = G > 16 ? turns_of(a, lane + 64) : 0.0;
    const int first = static_cast<int>(blockIdx.y) * per, last = min(first + per, list.steps), pack = PACKED ? a.pack : 0, runs = (a.T + (1 << pack) - 1) >> pack, items = a.B * runs;
#pragma unroll 1
    for (int item = blockIdx.x * WAVES + wave; item < items; item += stride) {
        const int b = a.B == 1 ? 0 : __builtin_amdgcn_readfirstlane(item / runs), t = (item - b * runs) << pack, tokens = min(1 << pack, a.T - t);
        const int64_t xq = b * a.x[0].sb + t * a.x[0].st, xk = b * a.x[1].sb + t * a.x[1].st, yq = b * a.y[0].sb + t * a.y[0].st, yk = b * a.y[1].sb + t * a.y[1].st;
        auto at = list.step(a, first, tokens);
        typename L::C::Raw raw = list.load(a.x, at, xq, xk, lx);
        const Angles turn = angles<G, PACKED>(a, a.pos + b * a.pos_sb + t, tokens, list.token * 4 * G + list.p0, near, far, strips[wave]);
#pragma unroll 1
        for (int s = first; s < last; ++s) {
            const auto now = at;
            const Eight x = L::C::unpack(raw);
            if (s + 1 < last) at = list.step(a, s + 1, tokens), raw = list.load(a.x, at, xq, xk, lx);
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (LOOSE)
                    ss += list.ka[i] * (x.a[i] * x.a[i]) + list.kb[i] * (x.b[i] * x.b[i]);
                else
                    ss += x.a[i] * x.a[i] + x.b[i] * x.b[i];
            }
            const float r = inverse_root(group_sum<G>(list.mine ? ss : 0.0f) * a.per_dk + a.eps);
            Eight y;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float ua = x.a[i] * r * (now.key ? wk.a[i] : wq.a[i]), ub = x.b[i] * r * (now.key ? wk.b[i] : wq.b[i]);
                y.a[i] = ua * turn.c[i] - ub * turn.s[i];
                y.b[i] = ua * turn.s[i] + ub * turn.c[i];
            }
            if (list.mine && now.live) list.store(a.y, now, yq, yk, ly, y);
        }
    }
}

template <typename T, int G, bool HALVES, bool LOOSE, bool PACKED>
__global__ __launch_bounds__(NT) void qk_bwd_rows(Qk a, int per) {
    using L = List<T, G, HALVES, LOOSE, PACKED>;
    __shared__ float2 strips[WAVES][PACKED ? 256 : 4 * G];  // 64 / G tokens at most
    __shared__ __align__(16) float sh[WAVES * L::ROWS * 2 * 8 * G];  // 16 KB
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), stride = static_cast<int>(gridDim.x) * WAVES;
    const L list(a);
    const Eight wq = weights_of<HALVES>(a.w[0], list.c0, list.c1), wk = weights_of<HALVES>(a.w[1], list.c0, list.c1);
    const auto lx = list.lane(a.x), lg = list.lane(a.dy), ly = list.lane(a.y);
    const double near = turns_of(a, lane % (4 * G)), far = G > 16 ? turns_of(a, lane + 64) : 0.0;
    const int first = static_cast<int>(blockIdx.y) * per, last = min(first + per, list.steps), pack = PACKED ? a.pack : 0, runs = (a.T + (1 << pack) - 1) >> pack, items = a.B * runs;
    Eight dwq = {}, dwk = {};
#pragma unroll 1
    for (int item = blockIdx.x * WAVES + wave; item < items; item += stride) {
        const int b = a.B == 1 ? 0 : __builtin_amdgcn_readfirstlane(item / runs), t = (item - b * runs) << pack, tokens = min(1 << pack, a.T - t);
        const int64_t xq = b * a.x[0].sb + t * a.x[0].st, xk = b * a.x[1].sb + t * a.x[1].st, yq = b * a.y[0].sb + t * a.y[0].st, yk = b * a.y[1].sb + t * a.y[1].st;
        const int64_t gq = b * a.dy[0].sb + t * a.dy[0].st, gk = b * a.dy[1].sb + t * a.dy[1].st;
        auto at = list.step(a, first, tokens);
        typename L::C::Raw rx = list.load(a.x, at, xq, xk, lx), rg = list.load(a.dy, at, gq, gk, lg);
        const Angles turn = angles<G, PACKED>(a, a.pos + b * a.pos_sb + t, tokens, list.token * 4 * G + list.p0, near, far, strips[wave]);
#pragma unroll 1
        for (int s = first; s < last; ++s) {
            const auto now = at;
            const Eight x = L::C::unpack(rx), dy = L::C::unpack(rg);
            if (s + 1 < last) at = list.step(a, s + 1, tokens), rx = list.load(a.x, at, xq, xk, lx), rg = list.load(a.dy, at, gq, gk, lg);
            Eight wdu, dux;
            float ss = 0.0f, sg = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float da = dy.a[i] * turn.c[i] + dy.b[i] * turn.s[i], db = dy.b[i] * turn.c[i] - dy.a[i] * turn.s[i];
                wdu.a[i] = da * (now.key ? wk.a[i] : wq.a[i]), wdu.b[i] = db * (now.key ? wk.b[i] : wq.b[i]);
                dux.a[i] = da * x.a[i], dux.b[i] = db * x.b[i];
                if constexpr (LOOSE) {
                    ss += list.ka[i] * (x.a[i] * x.a[i]) + list.kb[i] * (x.b[i] * x.b[i]);
                    sg += list.ka[i] * (wdu.a[i] * x.a[i]) + list.kb[i] * (wdu.b[i] * x.b[i]);
                } else {
                    ss += x.a[i] * x.a[i] + x.b[i] * x.b[i];
                    sg += wdu.a[i] * x.a[i] + wdu.b[i] * x.b[i];
                }
            }
            const float r = inverse_root(group_sum<G>(list.mine ? ss : 0.0f) * a.per_dk + a.eps);
            const float m = r * r * (group_sum<G>(list.mine ? sg : 0.0f) * a.per_dk);
            if (!list.mine || !now.live) continue;
            Eight dx;
#pragma unroll
            for (int i = 0; i < 4; ++i) dx.a[i] = r * (wdu.a[i] - x.a[i] * m), dx.b[i] = r * (wdu.b[i] - x.b[i] * m);
            if (now.key) {
#pragma unroll
                for (int i = 0; i < 4; ++i) dwk.a[i] += dux.a[i] * r, dwk.b[i] += dux.b[i] * r;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) dwq.a[i] += dux.a[i] * r, dwq.b[i] += dux.b[i] * r;
            }
            list.store(a.y, now, yq, yk, ly, dx);
        }
    }
    // the sums of all groups of all wavefronts, columns in their order, then added up column by column
    constexpr int PITCH = 2 * 8 * G;
    float* const own = sh + (wave * L::ROWS + lane / G) * PITCH;
    if (list.mine) {
        auto lay = [&](float* to, const Eight& d) {
            if constexpr (LOOSE) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (list.ka[i] != 0.0f) to[column_a<HALVES>(list.c0, list.c1, i)] = d.a[i];
                    if (list.kb[i] != 0.0f) to[column_b<HALVES>(list.c0, list.c1, i)] = d.b[i];
                }
                return;
            }
            *reinterpret_cast<f32x4*>(to + list.c0) = HALVES ? d.a : f32x4{d.a[0], d.b[0], d.a[1], d.b[1]};
            *reinterpret_cast<f32x4*>(to + list.c1) = HALVES ? d.b : f32x4{d.a[2], d.b[2], d.a[3], d.b[3]};
        };
        lay(own, dwq);
        lay(own + 8 * G, dwk);
    }
    __syncthreads();
    const int64_t group = blockIdx.y * static_cast<int64_t>(gridDim.x) + blockIdx.x;
    for (int i = threadIdx.x; i < PITCH; i += NT) {
        const int col = i & (8 * G - 1);
        if (col >= a.dk) continue;
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < WAVES * L::ROWS; ++k) s += sh[k * PITCH + i];
        a.part[group * (2 * a.dk) + (i >= 8 * G ? a.dk : 0) + col] = s;
    }
}

// The workgroups' sums of dw added up in a fixed order: 16 columns to a workgroup, four to a thread, 256 threads to a column, whose loads are all on their way
// together.
constexpr int SUM_NT = 1024;
__global__ __launch_bounds__(SUM_NT) void qk_dw_sum(const float* part, int parts, int dk, float* dwq, float* dwk) {
    __shared__ f32x4 sh[SUM_NT / 64][4];
    const int c = threadIdx.x & 3, slice = threadIdx.x >> 2, col = static_cast<int>(blockIdx.x) * 16 + 4 * c, cols = 2 * dk;  // cols is a multiple of 4
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (col < cols) {
        f32x4 v[BWD_MOST / (SUM_NT / 4)];
#pragma unroll
        for (int k = 0; k < BWD_MOST / (SUM_NT / 4); ++k) {
            const int i = slice + k * (SUM_NT / 4);
            v[k] = i < parts ? *reinterpret_cast<const f32x4*>(part + i * static_cast<int64_t>(cols) + col) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int k = 0; k < BWD_MOST / (SUM_NT / 4); ++k) s += v[k];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        for (int o = 4; o < 64; o *= 2) s[e] += __shfl_xor(s[e], o);
    if ((threadIdx.x & 63) < 4) sh[threadIdx.x >> 6][c] = s;
    __syncthreads();
    if (threadIdx.x >= 16) return;
    const int at = static_cast<int>(threadIdx.x), to = static_cast<int>(blockIdx.x) * 16 + at;
    float r = 0.0f;
#pragma unroll
    for (int i = 0; i < SUM_NT / 64; ++i) r += sh[i][at >> 2][at & 3];
    if (to < cols) (to < dk ? dwq[to] : dwk[to - dk]) = r;
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
// Where a tensor's rows lie: three dimensions of runs of `run` bytes, those of size 1 left out.
struct Place {
    int64_t at, run;   // the first byte of all, strides taken by their size
    int64_t n[3], stride[3];
    bool back[3], repeats = false;  // which strides lead backwards; whether one leads nowhere
    int dims = 0;
    void add(int64_t count, int64_t bytes) {
        if (count < 2) return;
        if (bytes == 0) {
            repeats = true;
            return;
        }
        if ((back[dims] = bytes < 0)) at += (count - 1) * bytes, bytes = -bytes;
        n[dims] = count, stride[dims++] = bytes;
    }
    int64_t span(int64_t under = INT64_MAX) const {  // of the runs that strides smaller than this join
        int64_t bytes = run;
        for (int i = 0; i < dims; ++i) bytes += stride[i] < under ? (n[i] - 1) * stride[i] : 0;
        return bytes;
    }
    bool in_steps_of(int64_t step) const {  // all other strides are whole numbers of steps
        return std::all_of(stride, stride + dims, [&](int64_t s) { return s < step || s % step == 0; });
    }
    int64_t widest() const { return dims ? *std::max_element(stride, stride + dims) : 0; }
    int64_t drop(int64_t step) {  // one repetition of what repeats in these steps is left, the first: how many there were
        for (int i = 0; i < dims; ++i)
            if (stride[i] == step) {
                const int64_t count = n[i];
                --dims, n[i] = n[dims], stride[i] = stride[dims];
                return count;
            }
        return 1;
    }
    bool single() const {  // no byte is in two runs
        return !repeats && std::all_of(stride, stride + dims, [&](int64_t s) { return s >= span(s) && std::count(stride, stride + dims, s) == 1; });
    }
};
Place place_of(const pk_tensor4* t, const pk_qk_shape* s, int heads) {
    const int64_t es = elem_size(s->dtype);
    Place p;
    p.at = static_cast<int64_t>(reinterpret_cast<uintptr_t>(t->ptr)), p.run = s->dk * es;
    p.add(s->B, t->stride_b * es), p.add(s->T, t->stride_t * es), p.add(heads, t->stride_h * es);
    return p;
}
Place place_of(const void* v, int64_t n, int64_t rows = 1, int64_t stride = 0) {  // n words
    Place p;
    p.at = static_cast<int64_t>(reinterpret_cast<uintptr_t>(v)), p.run = 4 * n;
    p.add(rows, 4 * stride);
    return p;
}
bool same(const Place& a, const Place& b) {  // element for element
    return a.at == b.at && a.run == b.run && a.dims == b.dims && a.repeats == b.repeats && std::equal(a.n, a.n + a.dims, b.n) && std::equal(a.stride, a.stride + a.dims, b.stride) &&
           std::equal(a.back, a.back + a.dims, b.back);
}
// Whether two have no byte in common for sure: one behind the other, or, as heads, tokens or sequences of one buffer, in different parts of a step that both repeat in,
// or so in every distance that what the outermost step repeats can come to.
bool apart(const Place& a, const Place& b) {
    if (a.at + a.span() <= b.at || b.at + b.span() <= a.at) return true;
    const auto in_gaps_of = [&](int64_t step) {
        if (!a.in_steps_of(step) || !b.in_steps_of(step)) return false;
        const int64_t ahead = ((b.at - a.at) % step + step) % step;
        return a.span(step) <= ahead && ahead + b.span(step) <= step;
    };
    if (std::any_of(a.stride, a.stride + a.dims, in_gaps_of) || std::any_of(b.stride, b.stride + b.dims, in_gaps_of)) return true;
    Place u = a, v = b;
    const int64_t step = std::max(u.widest(), v.widest());
    if (step == 0) return false;
    const int64_t ahead = u.drop(step) - 1, behind = v.drop(step) - 1;  // u's repetition less v's lies from -behind to ahead
    const auto down = [step](int64_t x) { return x >= 0 ? x / step : -((step - 1 - x) / step); };
    const int64_t first = std::max(-behind, down(v.at - u.at - u.span()) + 1), last = std::min(ahead, -down(u.at - v.at - v.span()) - 1);
    if (last - first > 2) return false;  // repetitions that lie over one another
    for (int64_t d = first; d <= last; ++d) {
        u.at = a.at + d * step;
        if (!apart(u, v)) return false;
    }
    return true;
}
// What every row of a result may be written over is its own input, element for element: rows are read and written by different wavefronts. Refused: a result over the other
// one or over what that is made of, over the weights or positions, over its own input in any other way, over itself.
int overlapping(const char* who, const pk_qk_shape* s, const pk_tensor4* q, const pk_tensor4* k, std::initializer_list<const pk_tensor4*> read_for_q,
                std::initializer_list<const pk_tensor4*> read_for_k, const float* wq, const float* wk, const int* pos) {
    const auto refuse = [who](const char* why) { return fail(PK_ERR_ARGUMENT, std::string(who) + why); };
    const Place results[2] = {place_of(q, s, s->Hq), place_of(k, s, s->Hkv)};
    if (!apart(results[0], results[1])) return refuse(": a result lies over the other one's tensor");
    const Place words[3] = {place_of(wq, s->dk), place_of(wk, s->dk), s->pos_stride_b ? place_of(pos, s->T, s->B, s->pos_stride_b) : place_of(pos, s->T)};
    for (int i = 0; i < 2; ++i) {
        for (const pk_tensor4* x : i ? read_for_q : read_for_k)
            if (!apart(results[i], place_of(x, s, i ? s->Hq : s->Hkv))) return refuse(": a result lies over the other one's tensor");
        for (const pk_tensor4* x : i ? read_for_k : read_for_q)
            if (const Place own = place_of(x, s, i ? s->Hkv : s->Hq); !same(results[i], own) && !apart(results[i], own))
                return refuse(": a result may lie where its own input does, element for element, or clear of it");
        for (const Place& w : words)
            if (!apart(results[i], w)) return refuse(": a result lies over the weights or the positions");
    }
    for (const Place& r : results)
        if (!r.single()) return refuse(": a result's elements share memory");
    return PK_OK;
}

void fill(Qk& a, const pk_qk_shape* s) {
    a.B = s->B, a.T = s->T, a.Hq = s->Hq, a.Hkv = s->Hkv, a.dk = s->dk, a.rotary = s->rotary ? s->rotary : s->dk, a.halves = s->halves != 0;
    a.eps = s->eps, a.per_dk = 1.0f / static_cast<float>(s->dk), a.pos_sb = s->pos_stride_b, a.part = nullptr, a.pack = 0;
    for (int i = 0; i < MAX_PAIRS / 8; ++i) a.coarse[i] = i == 0 ? 1.0 : 16 * i < a.rotary ? std::pow(s->theta, -16.0 * i / a.rotary) : 0.0;
    for (int i = 0; i < 8; ++i) a.fine[i] = std::pow(s->theta, -2.0 * i / a.rotary) / 6.283185307179586476925;
}
Rows rows_of(const pk_tensor4* t) { return Rows{t->ptr, t->stride_b, t->stride_t, t->stride_h}; }
RowsOut out_of(const pk_tensor4* t) { return RowsOut{t->ptr, t->stride_b, t->stride_t, t->stride_h}; }

int64_t items_of(const pk_qk_shape* s) { return static_cast<int64_t>(s->B) * s->T * (s->Hq + s->Hkv); }

// Whether a tensor's rows are whole pieces that the row kernels move: 16 bytes, or 8 where bf16 pairs come from two halves.
bool pieces(const void* p, int64_t sb, int64_t st, int64_t sh, const pk_qk_shape* s) {
    const int64_t es = elem_size(s->dtype), to = s->dtype == PK_BF16 && s->halves ? 8 : 16;
    return aligned(p, to) && sb * es % to == 0 && st * es % to == 0 && sh * es % to == 0;
}
// Which kernels take a call: the row kernels on whole aligned pieces, the row kernels on any rows, or those that take a wavefront for a row (head sizes under 8, the last few
// up to 256 where two remainders want a lane each, strides that are negative or past 2^24). 8192 tokens, 14 + 2 heads, bf16, a token to a wavefront, forward and backward: 64 columns aligned
// 7.9 and 15.8 us, the same as any rows 9.6 and 17.6, one element off 10.2 and 17.6, a wavefront for a row 59 and 80; 62 columns 10.1 and 18.5 (60 and 80), 100 columns of fp32
// 18.9 and 31 (64 and 84); 16456 tokens, 8 + 8 heads of 104 columns, 92 turned from halves, 27 and 39 (121 and 151).
enum Serve { ALIGNED, LOOSE, ANY };
Serve serve(const Qk& a, const pk_qk_shape* s, bool backward) {
    if (a.dk < 8 || lanes_wanted(a.dk, a.rotary, a.halves) > 32 || static_cast<int64_t>(s->B) * s->T > (1 << 30)) return ANY;
    bool whole = a.dk % 8 == 0 && !(a.halves && a.rotary % 8);
    for (int i = 0; i < 2; ++i) {
        whole = whole && pieces(a.x[i].p, a.x[i].sb, a.x[i].st, a.x[i].sh, s) && pieces(a.y[i].p, a.y[i].sb, a.y[i].st, a.y[i].sh, s);
        whole = whole && (!backward || pieces(a.dy[i].p, a.dy[i].sb, a.dy[i].st, a.dy[i].sh, s));
        for (const int64_t sh : {a.x[i].sh, a.y[i].sh, backward ? a.dy[i].sh : 0})  // a lane's offset inside a step is held in 32 bits
            if (sh < 0 || sh > (1 << 24)) return ANY;
    }
    return whole ? ALIGNED : LOOSE;
}
// Tokens of all sequences as one run, where every tensor has them so: no division in the kernel.
void flatten(Qk& a, bool backward) {
    if (a.pos_sb != a.T && a.B > 1) return;
    for (int i = 0; i < 2; ++i)
        if (a.x[i].sb != a.T * a.x[i].st || a.y[i].sb != a.T * a.y[i].st || (backward && a.dy[i].sb != a.T * a.dy[i].st)) return;
    a.T *= a.B, a.B = 1;
}
// of a row's group
int lanes_of(const Qk& a) {
    const int lanes = lanes_wanted(a.dk, a.rotary, a.halves);
    return lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : 32;
}

int steps_of(const Qk& a) {
    const int rows = (64 / lanes_of(a)) >> a.pack;
    return (a.Hq + rows - 1) / rows + (a.Hkv + rows - 1) / rows;
}
int64_t runs_of(const Qk& a) { return a.B * ((static_cast<int64_t>(a.T) + (1 << a.pack) - 1) >> a.pack); }
// Tokens that a wavefront takes at a time, as a power of two. With few heads most of a token's steps are groups without a row; dealt to several tokens they are none, and a step's
// 130 instructions are what bounds such shapes. Forward and backward, bf16: 32768 tokens, 1 + 1 heads of 64 by one token 18.0 and 32.0 us, by eight 6.0 and 11.8; 75348 tokens, 4 + 1
// heads of 32 37.6 and 64.5, by sixteen 10.4 and 21; 8192 tokens, 14 + 2 heads of 64 8.0 and 15.9, by four 6.9 and 14.4; 74251, 8 + 2 of 72 50 and 95, by two 45 and 93. The
// rows of a step lie further apart then, and not for nothing: steps that only become a fifth fewer cost fp32, whose bytes are twice as many, 2 %, and unaligned fp32 15 %.
int pack_of(Qk a, int dtype, bool backward) {
    for (int i = 0; i < 2; ++i)
        for (const int64_t st : {a.x[i].st, a.y[i].st, backward ? a.dy[i].st : 0})  // with the heads' strides a lane's offset, in 32 bits
            if (st < 0 || st > (1 << 24)) return 0;
    const double alone = static_cast<double>(steps_of(a)) * runs_of(a), enough = dtype == PK_BF16 ? 1.15 : 1.6;
    int best = 0;
    double least = alone;
    for (a.pack = 1; (64 / lanes_of(a)) >> a.pack; ++a.pack) {
        if (runs_of(a) < 2048) break;  // wavefronts
        const double steps = static_cast<double>(steps_of(a)) * runs_of(a);
        if (steps < least && steps * enough <= alone) best = a.pack, least = steps;
    }
    return best;
}

// A launch of the row kernels: workgroups over tokens, parts that a token's heads are dealt to, `most` workgroups in all.
struct Plan {
    int groups, parts, per;
};
// A token's heads stay with one wavefront, which forms the angles once, where the tokens alone fill the chip; fewer tokens are dealt out, to 4096 wavefronts.
// Forward, 32 heads of 128: 4 tokens 5.7 us by a wavefront each, 2.4 dealt out; 2048 tokens 8.6 and 7.9, dealt to 16384 wavefronts 10.1; 4096 tokens 12.5 either way.
Plan plan_of(const Qk& a, int most) {
    const int steps = steps_of(a);
    const int64_t tokens = runs_of(a), want = 4096;
    int parts = 1;
    while (parts < steps && parts < most && tokens * parts < want) ++parts;
    Plan p;
    p.per = (steps + parts - 1) / parts;
    p.parts = (steps + p.per - 1) / p.per;
    const int64_t groups = (tokens + WAVES - 1) / WAVES, cap = most / p.parts > 0 ? most / p.parts : 1;
    p.groups = static_cast<int>(groups < cap ? groups : cap);
    return p;
}

template <typename T, int G, bool HALVES, bool LOOSE>
void launch_rows(const Qk& a, const Plan& p, bool backward, hipStream_t st) {
    const dim3 grid(p.groups, p.parts);
    if (a.pack)
        backward ? qk_bwd_rows<T, G, HALVES, LOOSE, true><<<grid, NT, 0, st>>>(a, p.per) : qk_fwd_rows<T, G, HALVES, LOOSE, true><<<grid, NT, 0, st>>>(a, p.per);
    else
        backward ? qk_bwd_rows<T, G, HALVES, LOOSE, false><<<grid, NT, 0, st>>>(a, p.per) : qk_fwd_rows<T, G, HALVES, LOOSE, false><<<grid, NT, 0, st>>>(a, p.per);
}
template <typename T, bool HALVES, bool LOOSE>
void launch_rows(const Qk& a, const Plan& p, bool backward, hipStream_t st) {
    switch (lanes_of(a)) {
        case 4: return launch_rows<T, 4, HALVES, LOOSE>(a, p, backward, st);
        case 8: return launch_rows<T, 8, HALVES, LOOSE>(a, p, backward, st);
        case 16: return launch_rows<T, 16, HALVES, LOOSE>(a, p, backward, st);
        default: return launch_rows<T, 32, HALVES, LOOSE>(a, p, backward, st);
    }
}
template <typename T>
void launch_rows(const Qk& a, const Plan& p, bool backward, bool loose, hipStream_t st) {
    if (loose)
        a.halves ? launch_rows<T, true, true>(a, p, backward, st) : launch_rows<T, false, true>(a, p, backward, st);
    else
        a.halves ? launch_rows<T, true, false>(a, p, backward, st) : launch_rows<T, false, false>(a, p, backward, st);
}
void launch_rows(const Qk& a, const Plan& p, bool backward, bool loose, int dtype, hipStream_t st) {
    if (dtype == PK_BF16)
        launch_rows<uint16_t>(a, p, backward, loose, st);
    else
        launch_rows<float>(a, p, backward, loose, st);
}
// workgroups of the backward that takes any row
int any_groups(const pk_qk_shape* s) {
    const int64_t want = (items_of(s) + WAVES - 1) / WAVES;
    return static_cast<int>(want < 1 ? 1 : want > BWD_MOST ? BWD_MOST : want);
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
        if (int rc = overlapping("pk_qk_norm_rope_fwd", s, yq, yk, {q}, {k}, wq, wk, pos)) return rc;
        Qk a;
        fill(a, s);
        a.x[0] = rows_of(q), a.x[1] = rows_of(k), a.y[0] = out_of(yq), a.y[1] = out_of(yk), a.dy[0] = a.dy[1] = Rows{nullptr, 0, 0, 0};
        a.w[0] = wq, a.w[1] = wk, a.pos = pos;
        touch({q->ptr, k->ptr, yq->ptr, yk->ptr, wq, wk, pos}, stream);
        hipStream_t st = static_cast<hipStream_t>(stream);
        if (const Serve by = serve(a, s, false); by != ANY) {
            flatten(a, false);
            a.pack = pack_of(a, s->dtype, false);
            launch_rows(a, plan_of(a, FWD_MOST), false, by == LOOSE, s->dtype, st);
            return launched();
        }
        const int64_t want = (items_of(s) + WAVES - 1) / WAVES;
        const dim3 grid(static_cast<unsigned>(want < 65536 ? want : 65536));
        if (s->dtype == PK_BF16)
            qk_fwd_any<uint16_t><<<grid, NT, 0, st>>>(a);
        else
            qk_fwd_any<float><<<grid, NT, 0, st>>>(a);
        return launched();
    });
}

size_t pk_qk_norm_rope_bwd_workspace_bytes(const pk_qk_shape* s) {
    if (check(s, "pk_qk_norm_rope_bwd_workspace_bytes")) return 0;
    Qk a;
    fill(a, s);
    const Plan p = plan_of(a, BWD_MOST);
    return sizeof(float) * static_cast<size_t>(std::max(any_groups(s), p.groups * p.parts)) * 2 * s->dk;
}

int pk_qk_norm_rope_bwd(const pk_qk_shape* s, const pk_tensor4* dyq, const pk_tensor4* dyk, const pk_tensor4* q, const pk_tensor4* k, const float* wq,
                        const float* wk, const int* pos, const pk_tensor4* dq, const pk_tensor4* dk, float* dwq, float* dwk, void* workspace,
                        size_t workspace_bytes, void* stream) {
    return c_entry([&] {
        if (int rc = check(s, "pk_qk_norm_rope_bwd")) return rc;
        if (!wq || !wk || !dwq || !dwk) return fail(PK_ERR_ARGUMENT, "pk_qk_norm_rope_bwd: null tensor");
        const bool none = static_cast<int64_t>(s->B) * s->T == 0;
        if (!none && (bad(dyq) || bad(dyk) || bad(q) || bad(k) || bad(dq) || bad(dk) || !pos)) return fail(PK_ERR_ARGUMENT, "pk_qk_norm_rope_bwd: null tensor");
        if (!workspace || workspace_bytes < pk_qk_norm_rope_bwd_workspace_bytes(s) || !aligned(workspace, 16))
            return fail(PK_ERR_WORKSPACE, "pk_qk_norm_rope_bwd: workspace too small (pk_qk_norm_rope_bwd_workspace_bytes)");
        if (!none)
            if (int rc = overlapping("pk_qk_norm_rope_bwd", s, dq, dk, {q, dyq}, {k, dyk}, wq, wk, pos)) return rc;
        hipStream_t st = static_cast<hipStream_t>(stream);
        Qk a;
        fill(a, s);
        a.part = static_cast<float*>(workspace);
        a.w[0] = wq, a.w[1] = wk, a.pos = pos;
        int groups = any_groups(s);
        touch({wq, wk, dwq, dwk, pos, workspace}, stream);
        if (!none) {
            a.x[0] = rows_of(q), a.x[1] = rows_of(k), a.dy[0] = rows_of(dyq), a.dy[1] = rows_of(dyk), a.y[0] = out_of(dq), a.y[1] = out_of(dk);
            touch({q->ptr, k->ptr, dyq->ptr, dyk->ptr, dq->ptr, dk->ptr}, stream);
            if (const Serve by = serve(a, s, true); by != ANY) {
                flatten(a, true);
                a.pack = pack_of(a, s->dtype, true);
                const Plan p = plan_of(a, BWD_MOST);
                groups = p.groups * p.parts;
                launch_rows(a, p, true, by == LOOSE, s->dtype, st);
            } else if (s->dtype == PK_BF16)
                qk_bwd_any<uint16_t><<<dim3(groups), NT, 0, st>>>(a);
            else
                qk_bwd_any<float><<<dim3(groups), NT, 0, st>>>(a);
            if (int rc = launched()) return rc;
        }
        qk_dw_sum<<<dim3((2 * s->dk + 15) / 16), SUM_NT, 0, st>>>(a.part, none ? 0 : groups, s->dk, dwq, dwk);
        return launched();
    });
}

}  // extern "C"
