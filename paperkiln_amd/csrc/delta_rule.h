// What the kernels of the gated delta rule share (delta_rule.hip forward, delta_rule_bwd.hip backward).
//
// Chunks of 64 tokens. With G the sum of a chunk's log-decays up to a token, D_ij = exp(G_i - G_j) for j <= i, gamma_i = exp(G_i), delta_j = exp(G_63 - G_j):
//   M_ij = beta_i D_ij k_i.k_j (j < i)     T = (I + M)^-1     A_ij = scale D_ij q_i.k_j (j <= i)
//   R = beta (V - gamma K S)     U = T R     O = scale gamma Q S + A U     S' = gamma_63 S + K^T (delta U)
//
// Everything but q, k, v (and do) is a value of 32 bits that enters matrix products: it goes in as bf16 parts, x = x0 + x1 + x2 with 8 bits each, and a product
// of two such values is the sum of the six products of parts whose places add up to 2 at most. What is left out is 2^-24 of a term, the rounding that a
// product in 32 bits has; the matrix cores take 16 such products in the time of one in fp32. Tensors of bf16 are one part, tensors of fp32 three.
//
// A matrix instruction runs whatever lanes are switched on, so a branch around one has to be the wavefront's own: wavefront numbers are read into scalars.
// v_mfma_f32_16x16x32_bf16, lane l = 16 g + c: A row c, k = 8g .. 8g+7; B column c, k = 8g .. 8g+7; C column c, rows 4g .. 4g+3.
// A and B are alike, so a product is formed in the orientation that its result is wanted in: a lane's four values are neighbours there, in a row of memory or in what LDS keeps
// for the next product, whose operands are read along k in pieces of 16 bytes. The states in LDS are [columns][rows], R, U and their like [columns][tokens]; only K^T and Q^T are read
// by transposing reads.
#pragma once
#include <algorithm>

#include "post.h"

namespace pk {
namespace delta {

constexpr int C = 64;       // tokens of a chunk
// Columns of the state that a workgroup of a walk has are 16 or 32 (VB). Rows in LDS are 8 values past a multiple of 32, so that reads of 16 bytes down 16 rows meet every bank once.
constexpr int CP = C + 8;
constexpr int GB = 32;  // columns that go by at a time in the backward's last launch

inline int chunks(int T) { return (T + C - 1) / C; }
inline int blocks(int dv, int vb) { return (dv + vb - 1) / vb; }

typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));

__device__ inline f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Two values as N bf16 parts each, packed.
template <int N>
__device__ inline void split2(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        p[i] = pack_bf16(x, y);
        if (i + 1 < N) x -= __uint_as_float(p[i] << 16), y -= __uint_as_float(p[i] & 0xFFFF0000u);
    }
}
template <int N>
__device__ inline void split4(const f32x4& x, u32x2 (&p)[N]) {
    uint32_t a[N], b[N];
    split2(x[0], x[1], a), split2(x[2], x[3], b);
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = u32x2{a[i], b[i]};
}
// Eight values along k as an operand's parts.
template <int N>
struct Operand {
    bf16x8 part[N];
};
template <int N>
__device__ inline Operand<N> split8(const f32x4& lo, const f32x4& hi) {
    u32x2 a[N], b[N];
    split4(lo, a), split4(hi, b);
    Operand<N> o;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const u32x4 v = {a[i][0], a[i][1], b[i][0], b[i][1]};
        o.part[i] = *reinterpret_cast<const bf16x8*>(&v);
    }
    return o;
}
// c += a b: of two values in parts the products down to place MOST.
template <int MOST, int NA, int NB>
__device__ inline void product(const Operand<NA>& a, const Operand<NB>& b, f32x4& c) {
#pragma unroll
    for (int s = MOST; s >= 0; --s)  // the small ones first
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB) c = mfma16(a.part[i], b.part[s - i], c);
}

// The same into an accumulator for each place, so that no product waits for the one before it; their sum at the end.
template <int MOST, int NA, int NB>
__device__ inline void spread(const Operand<NA>& a, const Operand<NB>& b, f32x4 (&c)[MOST + 1]) {
#pragma unroll
    for (int s = MOST; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB) c[s] = mfma16(a.part[i], b.part[s - i], c[s]);
}
template <int N>
__device__ inline f32x4 gather(const f32x4 (&c)[N]) {
    f32x4 x = c[N - 1];
#pragma unroll
    for (int i = N - 2; i >= 0; --i) x += c[i];
    return x;
}

// ---- operands from LDS: N parts of a matrix of R rows, one behind the other ----
// rows r0 .. r0+15, k along a row from k0 on
template <int N, int R, int P>
__device__ inline Operand<N> rows_of(const uint16_t* m, int r0, int k0, int lane) {
    Operand<N> o;
    const uint16_t* p = m + (r0 + (lane & 15)) * P + k0 + 8 * (lane >> 4);
#pragma unroll
    for (int i = 0; i < N; ++i) o.part[i] = lds_read8(p + i * R * P);
    return o;
}
// columns c0 .. c0+15, k down the rows from k0 on
template <int N, int R, int P>
__device__ inline Operand<N> cols_of(const uint16_t* m, int k0, int c0, int lane) {
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    Operand<N> o;
    const int g = lane >> 4, j = lane & 15;
    const uint16_t* p = m + (k0 + 8 * g + (j >> 2)) * P + c0 + 4 * (j & 3);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const s16x4 lo = lds_read_tr4(p + i * R * P), hi = lds_read_tr4(p + i * R * P + 4 * P);
        const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        o.part[i] = *reinterpret_cast<const bf16x8*>(&v);
    }
    return o;
}
// four values of row r from column c0 on
template <int N, int R, int P>
__device__ inline void put4(uint16_t* m, int r, int c0, const f32x4& x) {
    u32x2 p[N];
    split4(x, p);
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<u32x2*>(m + (i * R + r) * P + c0) = p[i];
}

// ---- from memory ----
template <typename T>
constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
// Eight values of a row of n from column c on, zeros past its end.
__device__ inline Operand<1> load8(const uint16_t* row, int c, int n) {
    u32x4 v = {0, 0, 0, 0};
    if (c + 8 <= n) {
        v = *reinterpret_cast<const u32x4_any*>(row + c);
    } else {
        for (int i = 0; i < 8; ++i)
            if (c + i < n) {
                const uint32_t e = static_cast<uint32_t>(row[c + i]) << (16 * (i & 1));
                if (i < 2) v[0] |= e;
                else if (i < 4) v[1] |= e;
                else if (i < 6) v[2] |= e;
                else v[3] |= e;
            }
    }
    Operand<1> o;
    o.part[0] = *reinterpret_cast<const bf16x8*>(&v);
    return o;
}
// Four values of a row of n from column c on, as they are.
__device__ inline f32x4 load4(const float* row, int c, int n) {
    if (c + 4 <= n) return *reinterpret_cast<const f32x4_any*>(row + c);
    return f32x4{c < n ? row[c] : 0.0f, c + 1 < n ? row[c + 1] : 0.0f, c + 2 < n ? row[c + 2] : 0.0f, 0.0f};
}
__device__ inline f32x4 load4(const uint16_t* row, int c, int n) {
    const auto f = [](uint32_t x) { return __uint_as_float(x << 16); };
    if (c + 4 <= n) {
        const u32x2 v = *reinterpret_cast<const u32x2_any*>(row + c);
        return f32x4{f(v[0]), __uint_as_float(v[0] & 0xFFFF0000u), f(v[1]), __uint_as_float(v[1] & 0xFFFF0000u)};
    }
    return f32x4{c < n ? f(row[c]) : 0.0f, c + 1 < n ? f(row[c + 1]) : 0.0f, c + 2 < n ? f(row[c + 2]) : 0.0f, 0.0f};
}
__device__ inline void store4(float* row, int c, int n, const f32x4& x) {
    if (c + 4 <= n) {
        *reinterpret_cast<f32x4_any*>(row + c) = x;
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (c + i < n) row[c + i] = x[i];
    }
}
__device__ inline void store4(uint16_t* row, int c, int n, const f32x4& x) {
    const u32x2 v = {pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
    if (c + 4 <= n) {
        *reinterpret_cast<u32x2_any*>(row + c) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (c + i < n) row[c + i] = static_cast<uint16_t>(v[i >> 1] >> (16 * (i & 1)));
    }
}
// The address space is named where an address is one of two: of any space the load would also count as one of LDS, and no load could be left on its way.
template <typename V>
__device__ inline V from_memory(const void* p) {
    return *(const __attribute__((address_space(1))) V*)(p);
}
// How rows of q, k and their like are read. ANY: by the functions above. EVEN: rows are whole pieces; without a branch, where a row has ended the address is that of zeros. EXACT: rows are
// as long as the kernel's own, so a piece lies at an offset of 32 bits from its chunk's first.
enum Rows { ANY, EVEN, EXACT };
__device__ const uint32_t no_values[8] = {};
template <Rows BY, typename T>
struct Eight;  // eight values as they lie in memory: row `r` (a pitch of st) of `base`, from column c on, of n
template <Rows BY>
struct Eight<BY, uint16_t> {
    u32x4 v;
    __device__ void load(const uint16_t* base, int64_t st, int r, int c, int n) {
        if constexpr (BY == EXACT) {
            v = from_memory<u32x4_any>(base + (static_cast<uint32_t>(r) * static_cast<uint32_t>(st) + static_cast<uint32_t>(c)));
        } else if constexpr (BY == EVEN) {
            v = from_memory<u32x4_any>(c < n ? base + r * st + c : reinterpret_cast<const uint16_t*>(no_values));
        } else {
            const Operand<1> o = load8(base + r * st, c, n);
            v = *reinterpret_cast<const u32x4*>(&o.part[0]);
        }
    }
    __device__ Operand<1> operand() const {
        Operand<1> o;
        o.part[0] = *reinterpret_cast<const bf16x8*>(&v);
        return o;
    }
};
template <Rows BY>
struct Eight<BY, float> {
    f32x4 lo, hi;
    __device__ void load(const float* base, int64_t st, int r, int c, int n) {
        if constexpr (BY == EXACT) {
            const uint32_t at = static_cast<uint32_t>(r) * static_cast<uint32_t>(st) + static_cast<uint32_t>(c);
            lo = from_memory<f32x4_any>(base + at), hi = from_memory<f32x4_any>(base + at + 4);
        } else if constexpr (BY == EVEN) {
            const float* p = c < n ? base + r * st + c : reinterpret_cast<const float*>(no_values);
            lo = from_memory<f32x4_any>(p), hi = from_memory<f32x4_any>(p + 4);
        } else {
            lo = load4(base + r * st, c, n), hi = load4(base + r * st, c + 4, n);
        }
    }
    __device__ Operand<3> operand() const { return split8<3>(lo, hi); }
};
// eight values as they are
template <Rows BY>
__device__ inline void values_of(const Eight<BY, uint16_t>& e, f32x4& lo, f32x4& hi) {
    lo = f32x4{__uint_as_float(e.v[0] << 16), __uint_as_float(e.v[0] & 0xFFFF0000u), __uint_as_float(e.v[1] << 16), __uint_as_float(e.v[1] & 0xFFFF0000u)};
    hi = f32x4{__uint_as_float(e.v[2] << 16), __uint_as_float(e.v[2] & 0xFFFF0000u), __uint_as_float(e.v[3] << 16), __uint_as_float(e.v[3] & 0xFFFF0000u)};
}
template <Rows BY>
__device__ inline void values_of(const Eight<BY, float>& e, f32x4& lo, f32x4& hi) { lo = e.lo, hi = e.hi; }
// Four values of a dense matrix [rows][cols] of 32 bits: row r from column c on; zeros outside of it.
template <Rows BY>
__device__ inline f32x4 dense4(const float* base, int r, int c, int rows, int cols) {
    if constexpr (BY == EXACT)
        return from_memory<f32x4_any>(base + static_cast<uint32_t>(r * cols + c));
    else if constexpr (BY == EVEN)
        return from_memory<f32x4_any>(r < rows && c < cols ? base + (r * cols + c) : reinterpret_cast<const float*>(no_values));
    else
        return load4(base + (r < rows ? r : 0) * cols, c, r < rows ? cols : 0);
}
template <Rows BY, typename T>
__device__ inline void write4(T* row, int c, int n, const f32x4& x) {
    if constexpr (BY == ANY) {
        store4(row, c, n, x);
    } else {
        if (BY == EVEN && c >= n) return;
        if constexpr (sizeof(T) == 4)
            *reinterpret_cast<f32x4_any*>(row + c) = x;
        else
            *reinterpret_cast<u32x2_any*>(row + c) = u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
    }
}
// What a thread of NT holds of a chunk's rows of q or k on their way to LDS.
template <Rows BY, typename T, int DK, int NT>
struct Tile {
    static constexpr int PER = DK / 8, COUNT = (C * PER + NT - 1) / NT;
    static constexpr bool WHOLE = C * PER % NT == 0;
    Eight<BY, T> e[COUNT];
    __device__ void load(const T* base, int64_t st, int n, int dk) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const int at = threadIdx.x + i * NT, r = at / PER, c = at % PER * 8;
            if (WHOLE || r < C) e[i].load(base, st, min(r, n - 1), c, dk);  // a token behind the last one is multiplied by zeros
        }
    }
    template <int P>
    __device__ void to_lds(uint16_t* m) const {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const int at = threadIdx.x + i * NT, r = at / PER, c = at % PER * 8;
            if (!WHOLE && r >= C) continue;
            const Operand<PARTS<T>> o = e[i].operand();
#pragma unroll
            for (int p = 0; p < PARTS<T>; ++p) *reinterpret_cast<bf16x8*>(m + (p * C + r) * P + c) = o.part[p];
        }
    }
};
// Four tokens' values of one column, as they lie in memory. Tokens behind the last one have its values, columns behind the last one the first one's: they are multiplied by zero or not stored.
template <Rows BY, typename T>
struct Tokens {
    T v[4];
    __device__ void load(const T* base, int64_t st, int t, int n, int c, int cols) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int at = min(t + r, n - 1);
            if constexpr (BY == EXACT)
                v[r] = from_memory<T>(base + (static_cast<uint32_t>(at) * static_cast<uint32_t>(st) + static_cast<uint32_t>(c)));
            else
                v[r] = from_memory<T>(base + at * st + (c < cols ? c : 0));
        }
    }
    __device__ f32x4 values() const {
        if constexpr (sizeof(T) == 4)
            return f32x4{v[0], v[1], v[2], v[3]};
        else
            return f32x4{elem(v, 0), elem(v, 1), elem(v, 2), elem(v, 3)};
    }
};
// A chunk's matrices in memory: lower triangles T and A (or, transposed, upper ones) as the operands that they are read as, 16 rows and 32 values of k to a block of 64 lanes of 16
// bytes, in whole lines; of the eight blocks the six that are not all zeros.
constexpr int BLOCK = 16 * 32, BLOCKS = 6;
template <bool UPPER>
__device__ constexpr int block_of(int tile, int kk) {
    return UPPER ? (tile < 2 ? 2 * tile + kk : tile + 2) : (tile < 2 ? tile : 2 * tile - 2 + kk);
}
template <int N, bool UPPER>
__device__ inline Operand<N> matrix_block(const uint16_t* m, int tile, int kk, int lane) {
    Operand<N> o;
    const uint16_t* p = m + block_of<UPPER>(tile, kk) * BLOCK + 8 * lane;
#pragma unroll
    for (int i = 0; i < N; ++i) o.part[i] = *reinterpret_cast<const bf16x8*>(p + i * BLOCKS * BLOCK);
    return o;
}
// four values of row `row` from k on
template <int N, bool UPPER>
__device__ inline void put_block4(uint16_t* m, int row, int k, const f32x4& x) {
    u32x2 p[N];
    split4(x, p);
    uint16_t* to = m + block_of<UPPER>(row >> 4, k >> 5) * BLOCK + ((k & 31) >> 3) * 128 + (row & 15) * 8 + (k & 7);
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<u32x2*>(to + i * BLOCKS * BLOCK) = p[i];
}

// A problem as the kernels see it. Strides are in elements.
struct View {
    void* ptr;
    int64_t sb, st, sh;
};
template <typename T>
__device__ inline T* head(const View& v, int b, int h) {
    return static_cast<T*>(v.ptr) + b * v.sb + h * v.sh;
}
struct Rule {
    View q, k, v, o;                // o: the forward's
    const float *g, *beta;          // [B][T][Hv]
    const float* state_in;          // [B][Hv][dk][dv], or null
    float* state_out;               // or null
    // for every unit (batch, head of v) and chunk:
    uint16_t *inverse, *attn;       // parts of T and A, six blocks each
    float* scalars;                 // gamma, delta and beta of its tokens, 64 each
    float *states, *puts;           // backward: the state that the chunk begins with, [dk][dv]; U, [64][dv]
    // backward
    View dout, dq, dk_, dv_;
    float *dg, *dbeta;
    const float* dstate_out;        // gradient of the state that the rule leaves, or null
    float* dstate_in;               // of the one that it begins with, or null
    uint16_t *inverse_t, *attn_t;   // transposed
    float *dstates, *dputs;         // the gradient of the state that the chunk leaves; of R
    int B, T, Hk, Hv, dk, dv, chunks;
    float scale;
};
inline Rows rows_by(const Rule& a, int row, int vb) {
    const auto near = [](const View& v) { return v.st >= 0 && v.st < (1 << 22); };
    if (a.dk == row && a.dv % vb == 0 && near(a.q) && near(a.k) && near(a.v) && near(a.dout)) return EXACT;
    return a.dk % 8 == 0 && a.dv % 8 == 0 ? EVEN : ANY;
}
template <typename F>
int by_rows(Rows r, F&& f) {
    return r == EXACT ? f(std::integral_constant<Rows, EXACT>{}) : r == EVEN ? f(std::integral_constant<Rows, EVEN>{}) : f(std::integral_constant<Rows, ANY>{});
}
template <typename F>
int by_size(int dk, F&& f) {
    return dk <= 32 ? f(std::integral_constant<int, 32>{}) : dk <= 64 ? f(std::integral_constant<int, 64>{}) : f(std::integral_constant<int, 128>{});
}
// Columns to a workgroup of a walk: 32 where that many workgroups fill the chip, and a unit's matrices, q and k are then fetched half as often; else 16, a chunk of which takes less time.
// Forward and backward of 1024 tokens, us in columns of 32 and of 16, 256 workgroups of 32 and 128 of them: bf16 at 128 73, 258 (77, 267) and 64, 160 (52, 143); at 64 72, 268 (75, 274) and
// 59, 149 (53, 139); at 32 93, 357 (98, 378) and 66, 186 (59, 178); fp32 at 128 125, 423 (154, 450) and 107, 224 (82, 217); at 64 94, 312 (116, 364) and 77, 186 (66, 170); at 32 117, 390
// (130, 439) and 74, 218 (67, 205).
inline bool wide(const Rule& a) { return static_cast<int64_t>(a.B) * a.Hv * blocks(a.dv, 32) >= 256; }
// Workgroups of one unit go to one XCD, whose L2 then has the unit's q, k and matrices for all of its blocks. Launch with grid.x = unit_grid.
inline unsigned unit_grid(int64_t units, int per) { return static_cast<unsigned>((units + 7) / 8 * 8 * per); }
__device__ inline bool unit_of(int id, int units, int per, int& unit, int& blk) {
    const int j = id >> 3;
    unit = quotient(j, per) * 8 + (id & 7), blk = j - quotient(j, per) * per;
    return unit < units;
}

// What the chunks are made of that does not depend on a state, for the forward or (transposed as well) for the backward.
int launch_chunks(const Rule& a, int dtype, bool backward, hipStream_t st);
// The states that the chunks begin with and what they put into them.
int launch_states(const Rule& a, int dtype, hipStream_t st);
int check(const char* who, const pk_delta_shape* s);
bool view_of(const pk_tensor4* t, View& v);
// Where a tensor lies, to refuse results on top of something else. Tensors of heads that have gaps may lie between one another in one buffer, so of two tensors of heads, one of
// them with gaps, only the same place is refused.
struct Span {
    uintptr_t from, to;
    bool heads, gaps;
};
Span span_of(const void* dense, size_t bytes);
Span span_of(const View& v, const pk_delta_shape* s, int heads, int width);
bool apart(std::initializer_list<Span> written, std::initializer_list<Span> read);
bool shares(const View& v, const pk_delta_shape* s, int heads);  // elements that are one in memory
inline size_t pad(size_t bytes) { return (bytes + 255) & ~size_t{255}; }
constexpr size_t MATRIX = BLOCKS * BLOCK * sizeof(uint16_t);

}  // namespace delta
}  // namespace pk
