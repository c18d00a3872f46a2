// nxg_adapter_rows.hip -- gfx950 low-rank adapters over packed rows, forward and backward, and their C ABI
// (include/nxg_rows.h).
//
// A document's rows go through two thin products, down to `rank` values and up again. The forward pass and dx are the same
// kernel: s = x A^T, y = base + s B^T, and g = dy B, dx = base + g A with the weights turned round beforehand. What is left are sums
// over rows, g^T x and s^T dy, for each adapter. Large calls are bound by HBM for 16-bit rows of ranks up to 64 and fp32 rows of up to 32,
// then by the weights' way from L2 and by loads, products and stores that take turns (fp32 rows of rank 64: 116 us for 32,768, where the
// bytes take 45 to 50 and the products 28). The matrix instructions are 16x16 ones (32 values of the contracted
// index in 16 bits, 4 in fp32). 32 documents of 32,935 fp32 rows, 8 adapters of rank 16, 1,024 to 1,024: 79 us, 5.0 TB/s.
//
// s and g stay fp32. Beside 16-bit rows they enter the next product as the sum of two bf16 values, which is off by at most
// 2^-16 of a value, beside a result's own rounding by 2^-8 (bf16) or 2^-11 (fp16). fp16 rows and weights are the sum of two bf16
// values exactly, and of the four products only that of both second parts is left out (2^-16 again); so no value
// below 3.39e38 leaves a type's range on the way. Beside fp32 rows every product is fp32.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "nxg_rows.h"
#include "nxg_internal.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int MAX_RANK = 128;

// Rows of type E as operands of a matrix instruction: a lane has V values of one row, 16 bytes.
template <class E> struct operand;
template <> struct operand<__bf16> {
    static constexpr int V = 8;
    typedef v8b vec;
    static __device__ __forceinline__ v4f mul(v8b a, v8b b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct operand<_Float16> {
    static constexpr int V = 8;
    typedef v8h vec;
    static __device__ __forceinline__ v4f mul(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct operand<float> {
    static constexpr int V = 4;
    typedef v4f vec;
    static __device__ __forceinline__ v4f mul(v4f a, v4f b, v4f c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// Values k .. k + V - 1 of a row of n values, zeros behind its end: 16 bytes (of E) at once (n and k multiples of V), or one by one.
template <class E, bool WIDE, class S>
__device__ __forceinline__ typename operand<E>::vec fetch(const S * row, int k, int n) {
    constexpr int V = operand<E>::V;
    typename operand<E>::vec v;
    if constexpr (WIDE) {
        typedef S svec __attribute__((ext_vector_type(V)));
        svec x = {};
        if (k < n) x = *reinterpret_cast<const svec *>(row + k);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (E) x[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = k + i < n ? (E) row[k + i] : (E) 0.0f;
    }
    return v;
}
// The V values of type S at p as an operand of type E, or zeros.
template <class E, class S>
__device__ __forceinline__ typename operand<E>::vec taken(const char * p, bool some) {
    constexpr int V = operand<E>::V;
    typedef S svec __attribute__((ext_vector_type(V)));
    const svec x = *reinterpret_cast<const svec *>(p);
    typename operand<E>::vec v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = some ? (E) x[i] : (E) 0.0f;
    return v;
}
// Before a wave reads what its other lanes left in LDS, and after: LDS takes a wave's instructions in their order, and so must the compiler.
__device__ __forceinline__ void in_order() { asm volatile("" ::: "memory"); }
// A barrier for LDS alone: loads from memory stay under way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Rows that are read once leave the caches to what is read again (the weights, s and g): with ordinary loads 32,000 rows of 1,024 to
// 1,024 take 65 us for 46 (bf16) and 114 for 87 (fp32), the gradients over 65,536 rows 70 for 50.
template <class T>
__device__ __forceinline__ T once(const void * p) { return __builtin_nontemporal_load(reinterpret_cast<const T *>(p)); }

// x as the sum of two bf16 values: itself rounded, and what is left.
__device__ __forceinline__ void split(const float (&x)[8], v8b & hi, v8b & lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) hi[i] = (__bf16) x[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = (__bf16) (x[i] - (float) hi[i]);
}
__device__ __forceinline__ void split(v8h x, v8b & hi, v8b & lo) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float) x[i];
    split(f, hi, lo);
}

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Row offsets as the caller gave them, kept inside the arrays whatever they hold.
__device__ __forceinline__ int offset(const int32_t * cu, int d, int T) { return min(max(cu[d], 0), T); }

struct adapter_p {
    const char * x, * base;
    char * y;                      // null: s alone
    const void * a, * b;           // down [n][r][K], up [n][N][r]
    float * s;                     // [T][r]
    int64_t x_s, base_s, y_s;      // strides in bytes
    const int32_t * cu, * ids;
    int32_t T, K, N, r, n, n_seqs;
    float pre, post;               // factors on s and on the second product
    bool gather;                   // documents of one row that share an adapter go together
    int32_t window;                // among so many of them
};

struct tile {
    int row, len, id;              // rows row .. row + len - 1 of adapter id
    int doc;
    bool whole;                    // the document
};

// The tile of size rows of a slot. Document d owns the slots from floor(cu[d] / size) + d, at least as many as it has tiles,
// so that T / size + n_seqs slots do and the lengths need no pass over them. 64 documents are tried at a time.
__device__ __forceinline__ tile find_tile(const adapter_p & p, int size, int slot) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = p.n_seqs;
    while (n > 1) {
        const int step = (n + 63) >> 6, d = lo + lane * step;
        const bool at = lane * step < n && offset(p.cu, d, p.T) / size + d <= slot;
        const int last = max((int) __popcll(__ballot(at)) - 1, 0);
        n = min(step, n - last * step);
        lo += last * step;
    }
    lo = uni(lo);
    const int r0 = uni(offset(p.cu, lo, p.T)), r1 = uni(offset(p.cu, lo + 1, p.T)), at = slot - (r0 / size + lo);
    tile t;
    t.row = r0 + at * size;
    t.len = at < 0 ? 0 : min(size, r1 - t.row);
    t.doc = lo;
    t.whole = t.len == r1 - r0;
    const int id = uni(p.ids[lo]);
    t.id = id >= 0 && id < p.n ? id : -1;
    return t;
}

// s beside rows of type E, 16 RT ranks of it: operands of 16 ranks each (fp32, and RT 1 with both parts of s side by side), else 32.
template <class E, int RT> struct ranks {
    static constexpr bool F32 = std::is_same<E, float>::value;
    static constexpr int Q = F32 ? RT : RT == 1 ? 1 : RT / 2, SV = F32 || RT == 1 ? 1 : 2;
    typedef typename std::conditional<F32, v4f, v8b>::type vec;

    // the first rank of a lane's values of operand q
    static __device__ __forceinline__ int first(int q, int g) { return F32 ? 16 * q + 4 * g : RT == 1 ? 8 * (g & 1) : 32 * q + 8 * g; }
    // from a token's row of s in LDS
    static __device__ __forceinline__ void operands(vec (&s)[Q][SV], const float * row, int g) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            if constexpr (F32) {
                s[q][0] = *reinterpret_cast<const v4f *>(row + first(q, g));
            } else {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = row[first(q, g) + i];
                v8b hi, lo;
                split(x, hi, lo);
                if constexpr (RT == 1) {
                    s[q][0] = g < 2 ? hi : lo;
                } else {
                    s[q][0] = hi;
                    s[q][1] = lo;
                }
            }
        }
    }
    // up += operand q of B times s
    static __device__ __forceinline__ void multiply(v4f & up, const typename operand<E>::vec & b, const vec (&s)[SV]) {
        if constexpr (F32) {
            up = operand<float>::mul(b, s[0], up);
        } else {
            v8b hi, lo;
            if constexpr (std::is_same<E, _Float16>::value) split(b, hi, lo);
            else hi = b;
#pragma unroll
            for (int k = 0; k < SV; ++k) up = operand<__bf16>::mul(hi, s[k], up);
            if constexpr (std::is_same<E, _Float16>::value) up = operand<__bf16>::mul(lo, s[0], up);
        }
    }
};

// Documents of one row that have an adapter in common, 16 at a time (197 of 64 adapters of rank 128, fp32: 36 us, one by one 45): the rows
// of the tile's document and of those that follow it, into `rows`, and their number; 0 where the document is among those of one
// before it. They are looked for in a window of documents, so that what a workgroup looks over does not grow with their number.
// By every wave of a workgroup; ends with a barrier.
__device__ __forceinline__ int gather_rows(const adapter_p & p, const tile & c, int * rows) {
    const int lane = threadIdx.x & 63, first = c.doc / p.window * p.window, end = min(first + p.window, p.n_seqs);
    auto alike = [&](int d, int end) { return d < end && p.ids[d] == c.id && offset(p.cu, d + 1, p.T) - offset(p.cu, d, p.T) == 1; };
    int before = 0, found = 1;
    for (int d = first; d < c.doc; d += 256) before += __syncthreads_count(alike(d + threadIdx.x, c.doc));
    if (before % 16) return 0;
    if (threadIdx.x == 0) rows[0] = c.row;
    for (int d = c.doc + 1; d < end && found < 16; d += 64) {
        const bool mine = alike(d + lane, end);
        const uint64_t all = __ballot(mine);
        const int at = found + __popcll(all & ((1ull << lane) - 1));
        if (mine && at < 16 && threadIdx.x < 64) rows[at] = offset(p.cu, d + lane, p.T);
        found += __popcll(all);
    }
    __syncthreads();
    return min(found, 16);
}

// The rows of a document without an adapter: base as it is, s = 0. By a workgroup, V values at a time.
template <class E, int V>
__device__ __forceinline__ void copy_rows(const adapter_p & p, const tile & c) {
    typedef E vec __attribute__((ext_vector_type(V)));
    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
    for (int i = threadIdx.x; i < c.len * p.r; i += 256) p.s[(int64_t) c.row * p.r + i] = 0.0f;
    if (!p.y || p.y == p.base) return;
    for (int t = wave; t < c.len; t += 4) {
        const E * from = reinterpret_cast<const E *>(p.base + (c.row + (int64_t) t) * p.base_s);
        E * to = reinterpret_cast<E *>(p.y + (c.row + (int64_t) t) * p.y_s);
#pragma unroll 4
        for (int k = lane * V; k < p.N; k += 64 * V) {
            vec x = {};
            if (p.base) x = *reinterpret_cast<const vec *>(from + k);
            *reinterpret_cast<vec *>(to + k) = x;
        }
    }
}

// A workgroup: 16 rows of one document. Its four waves share the contracted index of x A^T out, 128 bytes of every row a step, so
// that the weights are read once per workgroup; their sums are joined in LDS, in a fixed order. Then they share out the columns of
// s B^T, taken as (B s^T), 128 bytes of every row a block: of a result, a lane has V columns next to each other of one row.
//
// THROUGH_LDS: everything comes from memory 8 lanes to 128 bytes of a row, a step or block ahead, and goes to the operands' lanes (16 of
// them 16 rows) through LDS that a wave has to itself; results go the same way back. A wave's load of 16 bytes from each of 64 places
// takes the first cache four times as long as one of 16 runs of 64 bytes, and bound this kernel before (32,935 rows of fp32, rank 16:
// 181 us with 64 rows a workgroup, 110 with 16; 79 now). WIDE: operands straight from memory, 16 bytes a lane, for calls of few workgroups,
// which wait for their own chain of loads alone. BY_VALUE: rows off 16 bytes.
enum { THROUGH_LDS, WIDE, BY_VALUE };
template <class E, class W, int RT, int HOW>
__global__ __launch_bounds__(256) void adapter_rows_kernel(adapter_p p) {
    constexpr int V = operand<E>::V, RP = 16 * RT, LD = RP + 4;
    constexpr int WV = 16 / (int) sizeof(W), A_ROW = 8 * V * (int) sizeof(W);      // weights of 16 bytes; bytes of a rank's step
    constexpr int A_LOADS = RP * A_ROW / 1024;             // 16-byte loads of a step's, or a block's, weights: 64 lanes each
    constexpr int OUT = 8 * V * 4 + 16;                    // bytes of a row of results in LDS
    constexpr int X_BYTES = 16 * OUT, A_BYTES = RP * A_ROW + 8 * V * 16;
    constexpr int SUMS = 2 * 16 * LD * 4, LDS = HOW == THROUGH_LDS ? std::max(4 * (X_BYTES + A_BYTES), SUMS) : SUMS;
    typedef typename operand<E>::vec vec;
    __shared__ __align__(16) char lds[LDS];
    __shared__ int gathered[16];
    tile c = find_tile(p, 16, blockIdx.x);
    if (c.len <= 0) return;
    if (c.id < 0) {
        if (blockIdx.y == 0) copy_rows<E, HOW == BY_VALUE ? 1 : V>(p, c);
        return;
    }
    const bool many = p.gather && c.whole && c.len == 1;
    if (many) {
        c.len = gather_rows(p, c, gathered);
        if (c.len == 0) return;
    }
    auto row_of = [&](int t) { return many ? (int64_t) gathered[t] : c.row + (int64_t) t; };
    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    char * xs = lds + wave * (X_BYTES + A_BYTES), * as = xs + X_BYTES;     // the wave's own
    const int row8 = lane >> 3, at8 = lane & 7;                            // 8 lanes a row

    // s, ranks as rows and tokens as columns
    v4f acc[RT];
#pragma unroll
    for (int j = 0; j < RT; ++j) acc[j] = v4f{};
    const W * a = static_cast<const W *>(p.a) + (int64_t) c.id * p.r * p.K;
    constexpr int STEP = 32 * V;
    int k0 = wave * 8 * V;
    if constexpr (HOW == THROUGH_LDS) {
        // 16-byte chunk i of row r is at chunk i ^ (r / 2) % 8 of it (rows of 64 bytes: i ^ (r / 4) % 4): 16 rows' same chunk fill the banks
        struct step {
            v4i x[2], a[A_LOADS];
        };
        const char * x[2];
        int ar[A_LOADS];
#pragma unroll
        for (int i = 0; i < 2; ++i) x[i] = p.x + row_of(min(8 * i + row8, c.len - 1)) * p.x_s;
#pragma unroll
        for (int i = 0; i < A_LOADS; ++i) ar[i] = min(A_ROW == 128 ? 8 * i + row8 : 16 * i + (lane >> 2), p.r - 1) * p.K;
        auto load = [&](step & s, int k0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) s.x[i] = once<v4i>(x[i] + min(k0 + at8 * V, p.K - V) * (int) sizeof(E));
#pragma unroll
            for (int i = 0; i < A_LOADS; ++i) s.a[i] = *reinterpret_cast<const v4i *>(a + ar[i] + min(k0 + (A_ROW == 128 ? at8 : lane & 3) * WV, p.K - WV));
        };
        auto use = [&](const step & s, int k0) {
            in_order();
#pragma unroll
            for (int i = 0; i < 2; ++i) *reinterpret_cast<v4i *>(xs + (8 * i + row8) * 128 + ((at8 ^ ((4 * i + (lane >> 4)) & 7)) << 4)) = s.x[i];
#pragma unroll
            for (int i = 0; i < A_LOADS; ++i) {
                if constexpr (A_ROW == 128) *reinterpret_cast<v4i *>(as + (8 * i + row8) * 128 + ((at8 ^ ((4 * i + (lane >> 4)) & 7)) << 4)) = s.a[i];
                else *reinterpret_cast<v4i *>(as + (16 * i + (lane >> 2)) * 64 + (((lane & 3) ^ ((lane >> 4) & 3)) << 4)) = s.a[i];
            }
            in_order();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = k0 + (4 * h + g) * V, sw = (4 * h + g) ^ (col >> 1);
                const vec xf = taken<E, E>(xs + col * 128 + (sw << 4), true);
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    const char * from = A_ROW == 128 ? as + (16 * j + col) * 128 + (sw << 4)
                                                     : as + (16 * j + col) * 64 + (((2 * h + (g >> 1)) ^ (col >> 2)) << 4) + (g & 1) * 8;
                    acc[j] = operand<E>::mul(taken<E, W>(from, k < p.K && 16 * j + col < p.r), xf, acc[j]);
                }
            }
        };
        step s0, s1;
        load(s0, k0);
        for (; k0 < p.K; k0 += 2 * STEP) {
            load(s1, k0 + STEP);
            use(s0, k0);
            if (k0 + STEP >= p.K) break;
            load(s0, k0 + 2 * STEP);
            use(s1, k0 + STEP);
        }
    } else {
        const E * x = reinterpret_cast<const E *>(p.x + row_of(min(col, c.len - 1)) * p.x_s);
        constexpr int BATCH = HOW == WIDE ? 8 : 2;         // operands whose loads are under way together
        for (; k0 < p.K; k0 += BATCH / 2 * STEP) {
            vec xf[BATCH], af[BATCH][RT];
#pragma unroll
            for (int h = 0; h < BATCH; ++h) {
                const int k = k0 + h / 2 * STEP + (4 * (h % 2) + g) * V;
                xf[h] = fetch<E, HOW == WIDE>(x, k, p.K);
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    const int r = 16 * j + col;
                    af[h][j] = fetch<E, HOW == WIDE>(a + (int64_t) r * p.K, r < p.r ? k : p.K, p.K);
                }
            }
#pragma unroll
            for (int h = 0; h < BATCH; ++h)
#pragma unroll
                for (int j = 0; j < RT; ++j) acc[j] = operand<E>::mul(af[h][j], xf[h], acc[j]);
        }
    }
    // The waves' sums: 0 + 2 and 1 + 3, then both. The first columns' weights and base are under way meanwhile (start).
    typedef float row_sums[16][LD];
    row_sums * sums = reinterpret_cast<row_sums *>(lds);
    constexpr int Q = ranks<E, RT>::Q, M = V / 4;          // M results make up a lane's V columns
    typename ranks<E, RT>::vec s[Q][ranks<E, RT>::SV];
    auto join = [&]() {
        if (HOW == THROUGH_LDS) lds_barrier();
        for (int turn = 0; turn < 2; ++turn) {
            if ((wave >> 1) == turn) {
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    v4f * to = reinterpret_cast<v4f *>(&sums[wave & 1][col][16 * j + 4 * g]);
                    *to = turn ? *to + acc[j] : acc[j];
                }
            }
            lds_barrier();
        }
        for (int i = threadIdx.x; i < 16 * RP; i += 256) {
            const int t = i / RP, r = i % RP;
            const float x = (sums[0][t][r] + sums[1][t][r]) * p.pre;
            sums[0][t][r] = x;
            if (blockIdx.y == 0 && t < c.len && r < p.r) p.s[row_of(t) * p.r + r] = x;
        }
        lds_barrier();
        ranks<E, RT>::operands(s, sums[0][col], g);
        if (HOW == THROUGH_LDS) lds_barrier();
    };
    if (!p.y) {
        join();
        return;
    }

    const W * b = static_cast<const W *>(p.b) + (int64_t) c.id * p.N * p.r;
    // row of B for a lane of result i of columns 4 V h .. of a block; its first rank of operand q
    auto b_row = [&](int h, int i) { return 4 * V * h + V * (col >> 2) + 4 * i + (col & 3); };
    auto b_rank = [&](int q) { return ranks<E, RT>::first(q, g); };
    const int step = 32 * V * (int) gridDim.y;
    int n0 = (blockIdx.y * 4 + wave) * 8 * V;
    if constexpr (HOW == THROUGH_LDS) {
        struct block {
            v4i before[2], b[A_LOADS];
        };
        const int64_t row[2] = {row_of(min(row8, c.len - 1)), row_of(min(8 + row8, c.len - 1))};
        // B's rows of a block lie one after another; in LDS they are 16 bytes apart, where they are whole chunks
        const int row_bytes = p.r * (int) sizeof(W), chunks = 8 * V * row_bytes / 16;
        const bool whole = row_bytes % 16 == 0, aligned = p.r % V == 0;
        const int stride = row_bytes + (whole ? 16 : 0);
        int at[A_LOADS];                                   // the lane's chunks' places
#pragma unroll
        for (int i = 0; i < A_LOADS; ++i) {
            const int q = 64 * i + lane;
            at[i] = q >= chunks ? -1 : 16 * (whole ? q + q / (row_bytes / 16) : q);
        }
        auto load = [&](block & k, int n0) {
            n0 = min(n0, (p.N - 1) / (8 * V) * 8 * V);     // behind the last block: that one
            const char * from = reinterpret_cast<const char *>(b + (int64_t) n0 * p.r);
            const int last = min(chunks, (p.N - n0) * row_bytes / 16) - 1;
#pragma unroll
            for (int i = 0; i < A_LOADS; ++i) k.b[i] = *reinterpret_cast<const v4i *>(from + min(64 * i + lane, last) * 16);
            if (p.base) {
#pragma unroll
                for (int i = 0; i < 2; ++i) k.before[i] = once<v4i>(p.base + row[i] * p.base_s + min(n0 + at8 * V, p.N - V) * (int) sizeof(E));
            }
        };
        auto use = [&](const block & k, int n0) {
            in_order();
#pragma unroll
            for (int i = 0; i < A_LOADS; ++i)
                if (at[i] >= 0) *reinterpret_cast<v4i *>(as + at[i]) = k.b[i];
            in_order();
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < M; ++i) {
                    const char * from = as + b_row(h, i) * stride;
                    v4f up = {};
#pragma unroll
                    for (int q = 0; q < Q; ++q) {
                        vec bf;
                        if (aligned) bf = taken<E, W>(from + b_rank(q) * (int) sizeof(W), b_rank(q) < p.r);
                        else bf = fetch<E, false>(reinterpret_cast<const W *>(from), b_rank(q), p.r);
                        ranks<E, RT>::multiply(up, bf, s[q]);
                    }
                    *reinterpret_cast<v4f *>(xs + col * OUT + (4 * V * h + V * g + 4 * i) * 4) = up;
                }
            in_order();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int t = 8 * i + row8, n = n0 + at8 * V;
                const float * up = reinterpret_cast<const float *>(xs + t * OUT) + at8 * V;
                vec before, out;
                __builtin_memcpy(&before, &k.before[i], 16);
#pragma unroll
                for (int e = 0; e < V; ++e) out[e] = (E) __builtin_fmaf(up[e], p.post, p.base ? (float) before[e] : 0.0f);
                if (t < c.len && n < p.N) __builtin_nontemporal_store(out, reinterpret_cast<vec *>(p.y + row[i] * p.y_s + (int64_t) n * (int) sizeof(E)));
            }
        };
        block b0, b1;
        load(b0, n0);
        join();
        for (; n0 < p.N; n0 += 2 * step) {
            load(b1, n0 + step);
            use(b0, n0);
            if (n0 + step >= p.N) break;
            load(b0, n0 + 2 * step);
            use(b1, n0 + step);
        }
    } else {
        const bool whole = HOW == WIDE && p.r % V == 0;
        const int64_t row = row_of(min(col, c.len - 1));
        const E * from = reinterpret_cast<const E *>(p.base + row * p.base_s);
        E * to = reinterpret_cast<E *>(p.y + row * p.y_s);
        vec before[2], bf[2][M][Q];
        auto load = [&]() {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                before[h] = fetch<E, HOW == WIDE>(from, p.base && col < c.len ? n0 + 4 * V * h + V * g : p.N, p.N);
#pragma unroll
                for (int i = 0; i < M; ++i) {
                    const W * br = b + (int64_t) min(n0 + b_row(h, i), p.N - 1) * p.r;
#pragma unroll
                    for (int q = 0; q < Q; ++q) bf[h][i][q] = whole ? fetch<E, true>(br, b_rank(q), p.r) : fetch<E, false>(br, b_rank(q), p.r);
                }
            }
        };
        if (HOW == WIDE) load();
        join();
        for (; n0 < p.N; n0 += step) {
            if (HOW != WIDE || n0 >= step) load();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = n0 + 4 * V * h + V * g;
                vec out;
#pragma unroll
                for (int i = 0; i < M; ++i) {
                    v4f up = {};
#pragma unroll
                    for (int q = 0; q < Q; ++q) ranks<E, RT>::multiply(up, bf[h][i][q], s[q]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) out[4 * i + e] = (E) __builtin_fmaf(up[e], p.post, (float) before[h][4 * i + e]);
                }
                if (col >= c.len) continue;
                if constexpr (HOW == WIDE) {
                    if (n < p.N) *reinterpret_cast<vec *>(to + n) = out;
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (n + e < p.N) to[n + e] = out[e];
                }
            }
        }
    }
}

// The same for larger ranks and many rows: a workgroup takes 64 MT rows, a wave 16 MT of them for itself, and its four waves share
// the weights, which they bring to LDS together, a step or block at a time (two in turn, so that one barrier a step does). That reads
// the weights a fourth as often as above, and leaves a wave the registers of few loads. 65,536 bf16 rows of 1,024 to 2,304, rank 64:
// 158 us (4.7 TB/s).
template <class E, class W, int MT, int RT>
__global__ __launch_bounds__(256, 2) void adapter_rows_tall_kernel(adapter_p p) {
    constexpr int V = operand<E>::V, RP = 16 * RT, LD = RP + 4;
    constexpr int WV = 16 / (int) sizeof(W), A_ROW = 8 * V * (int) sizeof(W);
    constexpr int A_LOADS = RP * A_ROW / 4096;             // of a wave
    static_assert(RP * A_ROW % 4096 == 0, "the four waves' loads are all of a step's weights");
    constexpr int OUT = 8 * V * 4 + 16;
    constexpr int X_BYTES = std::max(std::max(16 * MT * 128, 16 * OUT), 16 * LD * 4), A_BYTES = RP * A_ROW + 8 * V * 16;
    typedef typename operand<E>::vec vec;
    __shared__ __align__(16) char lds[4 * X_BYTES + 2 * A_BYTES];
    const tile c = find_tile(p, 64 * MT, blockIdx.x);
    if (c.len <= 0) return;
    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int row8 = lane >> 3, at8 = lane & 7;
    char * xs = lds + wave * X_BYTES, * const as = lds + 4 * X_BYTES;
    const int t0 = 16 * MT * wave;                         // the wave's first row

    if (c.id < 0) return copy_rows<E, V>(p, c);

    v4f acc[MT][RT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[m][j] = v4f{};
    const W * a = static_cast<const W *>(p.a) + (int64_t) c.id * p.r * p.K;
    {
        struct step {
            v4i x[2 * MT], a[A_LOADS];
        };
        const char * x[2 * MT];
        int ar[A_LOADS], rank[A_LOADS];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) x[i] = p.x + (c.row + (int64_t) min(t0 + 8 * i + row8, c.len - 1)) * p.x_s;
#pragma unroll
        for (int i = 0; i < A_LOADS; ++i) {
            rank[i] = A_ROW == 128 ? 8 * (4 * i + wave) + row8 : 16 * (4 * i + wave) + (lane >> 2);
            ar[i] = min(rank[i], p.r - 1) * p.K;
        }
        auto load = [&](step & s, int k0) {
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) s.x[i] = once<v4i>(x[i] + min(k0 + at8 * V, p.K - V) * (int) sizeof(E));
#pragma unroll
            for (int i = 0; i < A_LOADS; ++i) s.a[i] = *reinterpret_cast<const v4i *>(a + ar[i] + min(k0 + (A_ROW == 128 ? at8 : lane & 3) * WV, p.K - WV));
        };
        auto use = [&](step & s, int k0, char * buf, bool more) {
            in_order();
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) *reinterpret_cast<v4i *>(xs + (8 * i + row8) * 128 + ((at8 ^ ((4 * i + (lane >> 4)) & 7)) << 4)) = s.x[i];
#pragma unroll
            for (int i = 0; i < A_LOADS; ++i) {
                if constexpr (A_ROW == 128) *reinterpret_cast<v4i *>(buf + rank[i] * 128 + ((at8 ^ ((rank[i] >> 1) & 7)) << 4)) = s.a[i];
                else *reinterpret_cast<v4i *>(buf + rank[i] * 64 + (((lane & 3) ^ ((rank[i] >> 2) & 3)) << 4)) = s.a[i];
            }
            if (more) load(s, k0 + 16 * V);
            lds_barrier();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = k0 + (4 * h + g) * V, sw = (4 * h + g) ^ (col >> 1);
                vec xf[MT];
#pragma unroll
                for (int m = 0; m < MT; ++m) xf[m] = taken<E, E>(xs + (16 * m + col) * 128 + (sw << 4), true);
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    const char * from = A_ROW == 128 ? buf + (16 * j + col) * 128 + (sw << 4)
                                                     : buf + (16 * j + col) * 64 + (((2 * h + (g >> 1)) ^ (col >> 2)) << 4) + (g & 1) * 8;
                    const vec af = taken<E, W>(from, k < p.K && 16 * j + col < p.r);
#pragma unroll
                    for (int m = 0; m < MT; ++m) acc[m][j] = operand<E>::mul(af, xf[m], acc[m][j]);
                }
            }
        };
        step s0, s1;
        load(s0, 0);
        if (8 * V < p.K) load(s1, 8 * V);
        for (int k0 = 0; k0 < p.K; k0 += 16 * V) {
            use(s0, k0, as, k0 + 16 * V < p.K);
            if (k0 + 8 * V < p.K) use(s1, k0 + 8 * V, as + A_BYTES, k0 + 24 * V < p.K);
        }
    }
    // s of 16 rows at a time through LDS: its rows to memory, and the next product's operands
    constexpr int Q = ranks<E, RT>::Q;
    typename ranks<E, RT>::vec s[MT][Q][ranks<E, RT>::SV];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        float * rows = reinterpret_cast<float *>(xs);
        in_order();
#pragma unroll
        for (int j = 0; j < RT; ++j) *reinterpret_cast<v4f *>(rows + col * LD + 16 * j + 4 * g) = acc[m][j] * p.pre;
        in_order();
#pragma unroll
        for (int i = 0; i < RP / 4; ++i) {
            const int t = (64 * i + lane) / RP, r = (64 * i + lane) % RP;
            if (t0 + 16 * m + t < c.len && r < p.r) p.s[(c.row + (int64_t) t0 + 16 * m + t) * p.r + r] = rows[t * LD + r];
        }
        ranks<E, RT>::operands(s[m], rows + col * LD, g);
    }
    if (!p.y) return;
    lds_barrier();

    constexpr int M = V / 4;
    const W * b = static_cast<const W *>(p.b) + (int64_t) c.id * p.N * p.r;
    struct block {
        v4i before[2 * MT], b[A_LOADS];
    };
    const int row_bytes = p.r * (int) sizeof(W), chunks = 8 * V * row_bytes / 16;
    const bool whole = row_bytes % 16 == 0, aligned = p.r % V == 0;
    const int stride = row_bytes + (whole ? 16 : 0);
    int at[A_LOADS], from_q[A_LOADS];
#pragma unroll
    for (int i = 0; i < A_LOADS; ++i) {
        const int q = 64 * (4 * i + wave) + lane;
        from_q[i] = q;
        at[i] = q >= chunks ? -1 : 16 * (whole ? q + q / (row_bytes / 16) : q);
    }
    auto load = [&](block & k, int n0) {
        const char * from = reinterpret_cast<const char *>(b + (int64_t) n0 * p.r);
        const int last = min(chunks, (p.N - n0) * row_bytes / 16) - 1;
#pragma unroll
        for (int i = 0; i < A_LOADS; ++i) k.b[i] = *reinterpret_cast<const v4i *>(from + min(from_q[i], last) * 16);
        if (p.base) {
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) {
                const char * row = p.base + (c.row + (int64_t) min(t0 + 8 * i + row8, c.len - 1)) * p.base_s;
                k.before[i] = once<v4i>(row + min(n0 + at8 * V, p.N - V) * (int) sizeof(E));
            }
        }
    };
    auto use = [&](block & k, int n0, char * buf, bool more) {
        in_order();
#pragma unroll
        for (int i = 0; i < A_LOADS; ++i)
            if (at[i] >= 0) *reinterpret_cast<v4i *>(buf + at[i]) = k.b[i];
        v4i before[2 * MT];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) before[i] = k.before[i];
        if (more) load(k, n0 + 16 * V);
        lds_barrier();
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            in_order();
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < M; ++i) {
                    const int n = 4 * V * h + V * (col >> 2) + 4 * i + (col & 3);
                    v4f up = {};
#pragma unroll
                    for (int q = 0; q < Q; ++q) {
                        const int r = ranks<E, RT>::first(q, g);
                        vec bf;
                        if (aligned) bf = taken<E, W>(buf + n * stride + r * (int) sizeof(W), r < p.r);
                        else bf = fetch<E, false>(reinterpret_cast<const W *>(buf + n * stride), r, p.r);
                        ranks<E, RT>::multiply(up, bf, s[m][q]);
                    }
                    *reinterpret_cast<v4f *>(xs + col * OUT + (4 * V * h + V * g + 4 * i) * 4) = up;
                }
            in_order();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int t = t0 + 16 * m + 8 * i + row8, n = n0 + at8 * V;
                const float * up = reinterpret_cast<const float *>(xs + (8 * i + row8) * OUT) + at8 * V;
                vec old, out;
                __builtin_memcpy(&old, &before[2 * m + i], 16);
#pragma unroll
                for (int e = 0; e < V; ++e) out[e] = (E) __builtin_fmaf(up[e], p.post, p.base ? (float) old[e] : 0.0f);
                if (t < c.len && n < p.N) *reinterpret_cast<vec *>(p.y + (c.row + (int64_t) t) * p.y_s + (int64_t) n * (int) sizeof(E)) = out;
            }
        }
    };
    block b0, b1;
    load(b0, 0);
    if (8 * V < p.N) load(b1, 8 * V);
    for (int n0 = 0; n0 < p.N; n0 += 16 * V) {
        use(b0, n0, as, n0 + 16 * V < p.N);
        if (n0 + 8 * V < p.N) use(b1, n0 + 8 * V, as + A_BYTES, n0 + 24 * V < p.N);
    }
}

// ---------------------------------------------------------------------------
// gradients of the adapters
// ---------------------------------------------------------------------------

// Rows in the order of their adapters, an adapter's in the order of its documents; an adapter's rows are taken in chunks, by a
// workgroup for every slab of columns.
struct chunk {
    int id, from, count, part;     // id -1: none;  part: the place of its sums, or -1 where the adapter has no other chunk
};
struct adapter_rows_of {
    int row, rows, doc, docs, slot, part, chunks, unused;
};

struct grads_p {
    const int32_t * cu, * ids;
    int32_t T, K, N, r, n, n_seqs, size, n_slots, slabs_a, slabs_b;
    const void * a, * b;           // [n][r][K], [n][N][r]
    void * at, * bt;               // [n][K][r], [n][r][N]
    int32_t * order, * pos;        // the documents by adapter, and their first rows' places in that order
    int32_t * counts, runs;        // [runs][n], for the plan: runs of documents, a wave's each
    chunk * slots;
    adapter_rows_of * of;
    const char * x, * dy;
    int64_t x_s, dy_s;
    const float * g, * s;
    float * part_a, * part_b;      // [parts][r][K], [parts][r][N]
    void * da, * db;
    float scale;
    int32_t w_type, n_out_blocks;
    bool whole;                    // da and db are 16-byte aligned
};

// The sum of x over a wave's lanes up to this one: within rows of 16, then the last of a row to the next, of two to the others.
__device__ __forceinline__ int scan64(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}

// The sums of N values over the threads of `waves` waves before this one, and over all of them; a wave's own sum counts as `most` at most.
template <int N>
__device__ __forceinline__ void scan_all(int (&x)[N], int (&total)[N], int most, int (*sums)[16], int waves) {
    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int upto[N];
#pragma unroll
    for (int i = 0; i < N; ++i) upto[i] = scan64(x[i]);
    __syncthreads();
    if (lane == 63) {
#pragma unroll
        for (int i = 0; i < N; ++i) sums[i][wave] = min(upto[i], most);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = upto[i] - x[i];
        total[i] = 0;
        for (int w = 0; w < waves; ++w) {
            const int sum = sums[i][w];
            x[i] += w < wave ? sum : 0;
            total[i] += sum;
        }
    }
}

// Who has which rows, by one workgroup: the documents sorted by adapter, an adapter's in their own order, by counting. Every wave counts
// a run of documents for itself, then, from where its run's first of each adapter goes, places them; so the work goes by the
// documents and the adapters, and not by their product. Sums are kept at most T, so that offsets that do not rise make no place
// past the arrays. `room`: of lds, for the counts and then the documents' lengths where they fit.
__device__ __forceinline__ void plan_rows(const grads_p & p, int * lds, int room, int (*sums)[16]) {
    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
    // few documents and adapters: one wave, whose barriers wait for no other
    const int waves = p.n_seqs <= 64 && p.n <= 64 ? 1 : 16, threads = 64 * waves;
    if (wave >= waves) return;
    const int64_t n_counts = p.runs * (int64_t) p.n;
    const bool inside = n_counts + p.n_seqs <= room;
    int * counts = inside ? lds : p.counts;                // [runs][n]
    int * lens = inside ? lds + n_counts : p.pos;          // of the documents in their order
    int * mine = counts + (int64_t) wave * p.n;
    // the wave's documents, none of them behind the last run
    const int run = (p.n_seqs + 64 * p.runs - 1) / (64 * p.runs) * 64;
    const int first = wave < p.runs ? min(wave * run, p.n_seqs) : p.n_seqs, end = wave < p.runs ? min(first + run, p.n_seqs) : p.n_seqs;
    const int bits = p.n > 1 ? 32 - __clz(p.n - 1) : 0;
    // a lane's document: its adapter (-1: none), its rows, and the lanes with the same adapter
    int id, len;
    uint64_t same;
    auto take = [&](int d) {
        id = d < end ? p.ids[d] : -1;
        len = d < end ? max(offset(p.cu, d + 1, p.T) - offset(p.cu, d, p.T), 0) : 0;
        if (id < 0 || id >= p.n) id = -1;
        same = __ballot(id >= 0);
        for (int b = 0; b < bits; ++b) {
            const uint64_t ones = __ballot(id >> b & 1);
            same &= id >> b & 1 ? ones : ~ones;
        }
    };
    for (int64_t i = threadIdx.x; i < n_counts; i += threads) counts[i] = 0;
    __syncthreads();
    for (int d = first; d < end; d += 64) {
        take(d + lane);
        if (id >= 0 && (same & ((1ull << lane) - 1)) == 0) mine[id] += __popcll(same);
        __threadfence_block();             // the next step's lanes are others
    }
    __syncthreads();
    int docs_all = 0, doc = 0, docs = 0;   // of every adapter, and of a thread's: the first, and their number
    for (int i0 = 0; i0 < p.n; i0 += threads) {
        const int i = i0 + threadIdx.x;
        docs = 0;
        for (int w = 0; w < p.runs && i < p.n; ++w) docs += counts[(int64_t) w * p.n + i];
        int before[1] = {docs}, total[1];
        scan_all(before, total, INT32_MAX, sums, waves);
        doc = docs_all + before[0];
        docs_all += total[0];
        if (i >= p.n) continue;
        p.of[i].doc = doc;
        p.of[i].docs = docs;
        int k = doc;
        for (int w = 0; w < p.runs; ++w) {
            int & c = counts[(int64_t) w * p.n + i];
            const int here = c;
            c = k;
            k += here;
        }
    }
    __syncthreads();
    for (int d = first; d < end; d += 64) {
        if (run > 64) take(d + lane);      // else they are those of before
        const int before = __popcll(same & ((1ull << lane) - 1)), k = id >= 0 ? mine[id] : 0;
        __threadfence_block();
        if (id >= 0 && before == 0) mine[id] = k + __popcll(same);
        if (id >= 0) {
            p.order[k + before] = d + lane;
            lens[k + before] = len;
        }
        __threadfence_block();
    }
    __syncthreads();
    int rows_all = 0;
    for (int k0 = 0; k0 < docs_all; k0 += threads) {
        const int k = k0 + threadIdx.x;
        int before[1] = {k < docs_all ? lens[k] : 0}, total[1];
        scan_all(before, total, p.T, sums, waves);
        if (k < docs_all) p.pos[k] = lens[k] = min(rows_all + before[0], p.T);
        rows_all = min(rows_all + total[0], p.T);
    }
    __syncthreads();
    int slots = 0, parts = 0;
    for (int i0 = 0; i0 < p.n; i0 += threads) {
        const int i = i0 + threadIdx.x;
        adapter_rows_of o = {};
        if (i < p.n) {
            o.doc = p.n > threads ? p.of[i].doc : doc;
            o.docs = p.n > threads ? p.of[i].docs : docs;
            o.row = o.doc < docs_all ? lens[o.doc] : rows_all;
            o.rows = (o.doc + o.docs < docs_all ? lens[o.doc + o.docs] : rows_all) - o.row;
            o.chunks = max((o.rows + p.size - 1) / p.size, 1);
        }
        int before[2] = {o.chunks, o.chunks > 1 ? o.chunks : 0}, total[2];
        scan_all(before, total, INT32_MAX, sums, waves);
        o.slot = slots + before[0];
        o.part = parts + before[1];
        slots += total[0];
        parts += total[1];
        if (i < p.n) p.of[i] = o;
        // Every chunks-th step of 32 rows: all workgroups go over the rows side by side. Adapters of one chunk a lane, others a wave.
        if (i < p.n && o.chunks == 1 && o.slot < p.n_slots) p.slots[o.slot] = chunk{i, o.row, o.rows, -1};
        for (uint64_t left = __ballot(o.chunks > 1); left; left &= left - 1) {
            const int l = __ffsll((unsigned long long) left) - 1;
            const int chunks = __shfl(o.chunks, l), rows = __shfl(o.rows, l), row = __shfl(o.row, l), slot = __shfl(o.slot, l),
                      part = __shfl(o.part, l), steps = (rows + 31) / 32;
            for (int k = lane; k < chunks && slot + k < p.n_slots; k += 64) {
                const int own = (steps - k + chunks - 1) / chunks;
                const int count = max(32 * own - (own > 0 && (own - 1) * chunks + k == steps - 1 ? 32 * steps - rows : 0), 0);
                p.slots[slot + k] = chunk{i - lane + l, row + 32 * k, count, part + k};
            }
        }
    }
    for (int k = slots + (int) threadIdx.x; k < p.n_slots; k += threads) p.slots[k].id = -1;
}

// The first workgroup: plan_rows. Each other one: 64 columns of one adapter's down weights, or 64 rows of its up weights, turned round.
// Those go over the documents to see whether their adapter has rows; where documents times adapters are more than FEW_PAIRS they are a
// launch of their own behind the plan, which says so (gradients of 4,096 documents with 64 adapters of rank 16 117 us in one launch and
// 128 in two, of 1,000 with 1,000 363 and 334, of 4,096 with 1,000 458 and 392).
// 4 adapters of rank 16, 32 documents: 4.3 us, the plan's chain of loads.
constexpr int64_t FEW_PAIRS = 1 << 19;
enum { PLAN = 1, TURN = 2 };
template <class W>
__global__ __launch_bounds__(1024) void adapter_prepare_kernel(grads_p p, int what) {
    __shared__ __align__(16) W lds[MAX_RANK][66];
    __shared__ int sums[2][16];
    if ((what & PLAN) && blockIdx.x == 0) {
        plan_rows(p, reinterpret_cast<int *>(lds), sizeof(lds) / sizeof(int), sums);
        return;
    }
    const int strips_k = (p.K + 63) / 64, strips = strips_k + (p.N + 63) / 64, job = blockIdx.x - (what & PLAN ? 1 : 0);
    const int id = job / strips, strip = job % strips;
    if (what & PLAN) {
        bool some = false;         // has the adapter rows?
        for (int d = threadIdx.x; d < p.n_seqs; d += 1024) some |= p.ids[d] == id && offset(p.cu, d + 1, p.T) > offset(p.cu, d, p.T);
        if (!__syncthreads_or(some)) return;
    } else if (p.of[id].rows == 0) {
        return;
    }
    const bool down = strip < strips_k;
    const int c0 = (down ? strip : strip - strips_k) * 64, C = down ? p.K : p.N, cols = min(64, C - c0);
    const int64_t first = (int64_t) id * p.r * C;
    const W * from = static_cast<const W *>(down ? p.a : p.b) + first;
    W * to = static_cast<W *>(down ? p.at : p.bt) + first;
    for (int i = threadIdx.x; i < p.r * 64; i += 1024) {
        const int r = down ? i / 64 : i % p.r, k = down ? i % 64 : i / p.r;
        if (k < cols) lds[r][k] = down ? from[(int64_t) r * C + c0 + k] : from[(int64_t) (c0 + k) * p.r + r];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.r * 64; i += 1024) {
        const int r = down ? i % p.r : i / 64, k = down ? i / p.r : i % 64;
        if (k < cols) to[down ? (int64_t) (c0 + k) * p.r + r : (int64_t) r * C + c0 + k] = lds[r][k];
    }
}

__device__ __forceinline__ void put(void * to, int64_t i, float x, int32_t type) {
    if (type == NXG_TYPE_F32) static_cast<float *>(to)[i] = x;
    else if (type == NXG_TYPE_F16) static_cast<_Float16 *>(to)[i] = (_Float16) x;
    else static_cast<__bf16 *>(to)[i] = (__bf16) x;
}

template <int N>
__device__ __forceinline__ void put(void * to, int64_t i, const float (&x)[N], int32_t type) {
    typedef float fvec __attribute__((ext_vector_type(4)));
    typedef _Float16 hvec __attribute__((ext_vector_type(N)));
    typedef __bf16 bvec __attribute__((ext_vector_type(N)));
    if (type == NXG_TYPE_F32) {
#pragma unroll
        for (int k = 0; k < N; k += 4) *reinterpret_cast<fvec *>(static_cast<float *>(to) + i + k) = fvec{x[k], x[k + 1], x[k + 2], x[k + 3]};
    } else if (type == NXG_TYPE_F16) {
        hvec v;
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = (_Float16) x[k];
        *reinterpret_cast<hvec *>(static_cast<_Float16 *>(to) + i) = v;
    } else {
        bvec v;
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = (__bf16) x[k];
        *reinterpret_cast<bvec *>(static_cast<__bf16 *>(to) + i) = v;
    }
}

// The sum over a chunk's rows of u^T z, r x 64 V columns: u = g, z = x (dA), or u = s, z = dy (dB), 32 rows a step. A wave has 16 V columns:
// a lane loads 16 bytes of 8 rows, whose values of one column, next to each other after a permutation of bytes, are the
// operand as it is (its 16 lanes' columns are V apart). u is brought to LDS once for the four waves, turned round and as operands
// (two steps' in turn). The next step's loads are under way beside a step's products.
// 65,536 rows of bf16, 1,024 and 1,024 columns, rank 16: 50 us, 5.4 TB/s; rank 64, 1,024 and 2,304 columns: 102 to 117.
constexpr int CHUNK = 2048;        // rows of a chunk, at most
template <class E, int RT, int V, bool WIDE>
__global__ __launch_bounds__(256) void adapter_grads_kernel(grads_p p) {
    constexpr bool F32 = std::is_same<E, float>::value, F16 = std::is_same<E, _Float16>::value;
    constexpr int DEPTH = 2;                                   // steps whose loads are under way (4: 17.9 us for 16.2)
    constexpr int RP = 16 * RT, CW = 64 * V, TP = RP / 8;      // TP: tokens of u of a thread
    constexpr int U_ROW = F32 ? 32 * 4 + 16 : 32 * 2 + 16;     // bytes of a rank's 32 rows (of one part)
    constexpr int PARTS = F32 ? 1 : 2, U_BYTES = RP * U_ROW;
    typedef E evec __attribute__((ext_vector_type(V)));
    typedef typename std::conditional<F32, float, __bf16>::type U;
    typedef U uvec __attribute__((ext_vector_type(TP)));
    __shared__ __align__(16) int rows[CHUNK];
    __shared__ __align__(16) char us[2][PARTS][U_BYTES];
    const int slabs = p.slabs_a + p.slabs_b, slab = blockIdx.x % slabs;
    const chunk c = p.slots[blockIdx.x / slabs];
    if (c.id < 0) return;
    const bool down = slab < p.slabs_a;
    const int C = down ? p.K : p.N;
    const int64_t z_s = down ? p.x_s : p.dy_s;
    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int c0 = (down ? slab : slab - p.slabs_a) * CW + wave * 16 * V;      // the wave's first column
    const char * z = (down ? p.x : p.dy) + (int64_t) min(c0 + V * col, WIDE ? C - V : C - 1) * (int) sizeof(E);
    const int rank = threadIdx.x % RP, tok = threadIdx.x / RP * TP;            // of u
    const float * u = (down ? p.g : p.s) + min(rank, p.r - 1);

    const int doc = p.of[c.id].doc, docs = p.of[c.id].docs, chunks = p.of[c.id].chunks;
    for (int i = threadIdx.x; i < c.count; i += 256) {
        const int at = c.from + i / 32 * 32 * chunks + i % 32;
        int lo = doc, hi = doc + docs - 1;             // the last document that starts there or before
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (p.pos[mid] <= at) lo = mid;
            else hi = mid - 1;
        }
        rows[i] = min(max(offset(p.cu, p.order[lo], p.T) + at - p.pos[lo], 0), p.T - 1);
    }
    __syncthreads();

    v4f acc[V][RT];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[v][j] = v4f{};
    struct step {
        evec z[8];
        float u[TP];
    };
    // Loads go on without a branch, behind the chunk's end as its last row, and into the registers that a step has just done with: where
    // the compiler has to move a load's registers, it waits for the load first.
    auto load = [&](step & s, int t0) {
#pragma unroll
        for (int k = 0; k < TP; ++k) s.u[k] = u[(int64_t) rows[min(t0 + tok + k, c.count - 1)] * p.r];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const char * from = z + rows[min(t0 + 8 * g + k, c.count - 1)] * z_s;
            if constexpr (WIDE) {
                s.z[k] = once<evec>(from);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) s.z[k][v] = c0 + V * col + v < C ? reinterpret_cast<const E *>(from)[v] : (E) 0.0f;
            }
        }
    };
    auto use = [&](step & s, int t0, int buf) {
        // rows behind the chunk's end, and ranks behind the last, are zeros, in both operands
        uvec hi;
#pragma unroll
        for (int k = 0; k < TP; ++k) hi[k] = (U) (s.u[k] = t0 + tok + k < c.count && rank < p.r ? s.u[k] : 0.0f);
        *reinterpret_cast<uvec *>(us[buf][0] + rank * U_ROW + tok * (int) sizeof(U)) = hi;
        if constexpr (!F32) {
            uvec lo;
#pragma unroll
            for (int k = 0; k < TP; ++k) lo[k] = (U) (s.u[k] - (float) hi[k]);
            *reinterpret_cast<uvec *>(us[buf][1] + rank * U_ROW + tok * (int) sizeof(U)) = lo;
        }
        if (t0 + 32 > c.count) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (t0 + 8 * g + k >= c.count) s.z[k] = evec{};
        }
        lds_barrier();
        if constexpr (F32) {
            v4f uv[RT][2];
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) uv[j][i] = *reinterpret_cast<const v4f *>(us[buf][0] + (16 * j + col) * U_ROW + 32 * g + 16 * i);
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int j = 0; j < RT; ++j) acc[v][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(uv[j][k / 4][k % 4], s.z[k][v], acc[v][j], 0, 0, 0);
        } else {
            v8b uh[RT], ul[RT];
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                uh[j] = *reinterpret_cast<const v8b *>(us[buf][0] + (16 * j + col) * U_ROW + 16 * g);
                ul[j] = *reinterpret_cast<const v8b *>(us[buf][1] + (16 * j + col) * U_ROW + 16 * g);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                typename operand<E>::vec zc;
#pragma unroll
                for (int k = 0; k < 8; ++k) zc[k] = s.z[k][v];
                v8b zh, zl;
                if constexpr (F16) split(zc, zh, zl);
                else zh = zc;
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    acc[v][j] = operand<__bf16>::mul(uh[j], zh, acc[v][j]);
                    acc[v][j] = operand<__bf16>::mul(ul[j], zh, acc[v][j]);
                    if constexpr (F16) acc[v][j] = operand<__bf16>::mul(uh[j], zl, acc[v][j]);
                }
            }
        }
    };
    if (c.count > 0) {
        step ahead[DEPTH];
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) load(ahead[i], 32 * i);
        for (int t0 = 0; t0 < c.count; t0 += 32 * DEPTH) {
#pragma unroll
            for (int i = 0; i < DEPTH; ++i) {
                use(ahead[i], t0 + 32 * i, i % 2);
                load(ahead[i], t0 + 32 * (i + DEPTH));
            }
        }
    }
    const float f = down ? 1.0f : p.scale;
    float * part = c.part < 0 ? nullptr : (down ? p.part_a : p.part_b) + (int64_t) c.part * p.r * C;
    const int n = c0 + V * col;
    if (n >= C) return;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
        const int r0 = 16 * j + 4 * g;
        if (!part && !down && p.r % 4 == 0 && p.whole) {       // four ranks of a row of db
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float x[4] = {acc[v][j][0] * f, acc[v][j][1] * f, acc[v][j][2] * f, acc[v][j][3] * f};
                if (r0 < p.r && n + v < C) put<4>(p.db, ((int64_t) c.id * C + n + v) * p.r + r0, x, p.w_type);
            }
            continue;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + i;
            if (r >= p.r) continue;
            float x[V];
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = acc[v][j][i] * f;
            if (WIDE && part) {
                put<V>(part, (int64_t) r * C + n, x, NXG_TYPE_F32);
            } else if (WIDE && down && p.whole) {
                put<V>(p.da, ((int64_t) c.id * p.r + r) * C + n, x, p.w_type);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (n + v >= C) continue;
                    if (part) part[(int64_t) r * C + n + v] = x[v];
                    else if (down) put(p.da, ((int64_t) c.id * p.r + r) * C + n + v, x[v], p.w_type);
                    else put(p.db, ((int64_t) c.id * C + n + v) * p.r + r, x[v], p.w_type);
                }
            }
        }
    }
}

// The chunks' sums of the adapters that have several, in order: a value a lane, its four waves every fourth chunk (rank 64, 36
// chunks of 3,328 columns: 8 us, 31 MB).
__global__ __launch_bounds__(256) void adapter_join_kernel(grads_p p) {
    __shared__ float lds[4][64];
    const int id = blockIdx.x / p.n_out_blocks, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const adapter_rows_of o = p.of[id];
    if (o.chunks < 2) return;
    const int64_t n_a = p.slabs_a ? (int64_t) p.r * p.K : 0, n_b = p.slabs_b ? (int64_t) p.r * p.N : 0;
    int64_t e = (int64_t) (blockIdx.x % p.n_out_blocks) * 64 + lane;
    const bool some = e < n_a + n_b, down = e < n_a;
    if (!down) e -= n_a;
    const int64_t n = down ? n_a : n_b;
    float x = 0.0f;
    if (some) {
        const float * from = (down ? p.part_a : p.part_b) + o.part * n + e;
#pragma unroll 8
        for (int k = wave; k < o.chunks; k += 4) x += from[k * n];
    }
    lds[wave][lane] = x;
    __syncthreads();
    if (wave || !some) return;
    x = lds[0][lane] + lds[1][lane] + lds[2][lane] + lds[3][lane];
    if (down) put(p.da, id * n + e, x, p.w_type);
    else put(p.db, id * n + e % p.N * p.r + e / p.N, x, p.w_type);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

#define NXG_TRY(call) do { const int32_t rc_ = (call); if (rc_) return rc_; } while (0)

constexpr int64_t MAX_GRID = (1 << 24) - 1;    // workgroups of a launch: less than 2^32 threads
constexpr int MAX_WINDOW = 4096;               // of documents among which single rows are gathered

int size_of(int32_t type) { return type == NXG_TYPE_F32 ? 4 : type == NXG_TYPE_F16 || type == NXG_TYPE_BF16 ? 2 : 0; }

template <int N> using num = std::integral_constant<int, N>;

template <class F>
void by_type(int32_t type, F f) {
    if (type == NXG_TYPE_F32) f(float());
    else if (type == NXG_TYPE_F16) f((_Float16) 0.0f);
    else f((__bf16) 0.0f);
}
template <class F>
void by_types(int32_t type, int32_t w_type, F f) {
    if (type == NXG_TYPE_F32) by_type(w_type, [&](auto w) { f(float(), w); });
    else by_type(type, [&](auto e) { if constexpr (sizeof(e) == 2) f(e, e); });
}
template <class F>
void by_rank(int32_t r, F f) {
    if (r <= 16) f(num<1>());
    else if (r <= 32) f(num<2>());
    else if (r <= 64) f(num<4>());
    else f(num<8>());
}

int32_t check_params(const char * what, const nxg_adapter_rows_params * p) {
    if (!p) return nxg_fail(NXG_EINVAL, "%s: null params", what);
    if (!size_of(p->type)) return nxg_fail(NXG_EINVAL, "%s: type %d (F32, F16 or BF16)", what, p->type);
    if (!size_of(p->w_type) || (p->w_type != p->type && p->type != NXG_TYPE_F32)) {
        return nxg_fail(NXG_EINVAL, "%s: weight type %d (the rows'; any beside F32 rows)", what, p->w_type);
    }
    if (p->T < 0 || p->T >= 1 << 24 || p->n_seqs < 0 || p->n_seqs >= 1 << 22) return nxg_fail(NXG_EINVAL, "%s: T=%d n_seqs=%d", what, p->T, p->n_seqs);
    if (p->n_in < 1 || p->n_out < 1 || p->n_in > 1 << 20 || p->n_out > 1 << 20) return nxg_fail(NXG_EINVAL, "%s: n_in=%d n_out=%d", what, p->n_in, p->n_out);
    if (p->rank < 1 || p->rank > MAX_RANK) return nxg_fail(NXG_EINVAL, "%s: rank=%d (1 to %d)", what, p->rank, MAX_RANK);
    if (p->n_adapters < 1 || (int64_t) p->n_adapters * p->rank * std::max(p->n_in, p->n_out) > INT32_MAX ||
        p->n_adapters * (int64_t) ((p->rank * ((int64_t) p->n_in + p->n_out) + 63) / 64) > MAX_GRID) {
        return nxg_fail(NXG_EINVAL, "%s: n_adapters=%d of rank %d is none, or too large", what, p->n_adapters, p->rank);
    }
    if (!std::isfinite(p->scale)) return nxg_fail(NXG_EINVAL, "%s: scale=%g", what, p->scale);
    return NXG_OK;
}

int32_t check_arrays(const char * what, const nxg_adapter_rows_params * p) {
    if ((p->n_seqs && (!p->cu || !p->ids)) || !p->a || !p->b) return nxg_fail(NXG_EINVAL, "%s: null cu, ids, a or b", what);
    if (((uintptr_t) p->a | (uintptr_t) p->b) & 15) return nxg_fail(NXG_EINVAL, "%s: a and b must be 16-byte aligned", what);
    return NXG_OK;
}

int32_t check_rows(const char * what, const char * name, const void * p, int64_t stride, int32_t T, int32_t C, int es, bool written) {
    if (!p || ((uintptr_t) p & (es - 1))) return nxg_fail(NXG_EINVAL, "%s: %s is null or not aligned to its type", what, name);
    if (T > 1 && (stride < (written ? C : 0) || stride > INT64_MAX / 16 / T)) {
        return nxg_fail(NXG_EINVAL, "%s: stride %lld of %s for rows of %d", what, (long long) stride, name, C);
    }
    return NXG_OK;
}

// 16 bytes at a time where every row allows it.
bool wide(const void * p, int64_t stride_bytes) { return (((uintptr_t) p | (uintptr_t) stride_bytes) & 15) == 0; }

// The kernel of both directions: K values of x down to s, up to N values of y.
int32_t launch_rows(const char * what, adapter_p & p, int32_t type, int32_t w_type, void * stream) {
    const int V = 16 / size_of(type), cus = nxg_device_cus();
    const bool w = wide(p.x, p.x_s) && (!p.base || wide(p.base, p.base_s)) && wide(p.y, p.y ? p.y_s : 0) && p.K % V == 0 && p.N % V == 0 &&
                   p.K * (int64_t) size_of(w_type) % 16 == 0 && p.N * (int64_t) p.r * size_of(w_type) % 16 == 0;
    // Which kernel, and rows of a workgroup: the larger ones read the weights less often, where that leaves work for every CU. 1,024 to
    // 1,024, caches cold, one document and 32, with 64 rows and with 16 (320, 2,304 and 4,096 columns give the same answers):
    //   bf16 rank 32   24,000 rows 38, 39 and 39, 42 us   32,768 42, 49 and 51, 52   65,536 73, 85 and 98, 98
    //   bf16 rank 64   16,000 43, 47 and 38, 40           32,768 53, 63 and 77, 78   65,536 86, 88 and 152, 159
    //   bf16 rank 128  8,192 62, 62 and 51, 72            16,000 64, 74 and 97, 99   32,768 80, 126 and 191, 193
    //   fp32 rank 64   24,000 110, 111 and 99, 101        32,768 116, 150 and 132, 134   40,000 152, 152 and 162, 164
    //   fp32 rank 128  24,000 192, 193 and 236, 240       32,768 197, 275 and 314, 319   65,536 381, 387 and 614, 628
    // With 128 rows and with 64, bf16 rank 128: 65,536 rows 122, 189 and 149, 149; 100,000 219, 221 and 251, 253. fp32 has none of them: 65,536
    // rows 356, 525 and 381, 387; 80,000 545, 623 and 449, 450; 130,000 683, 684 and 700, 700. The steps are those of 512 workgroups at a time.
    // Straight from memory: one row of bf16 rank 16 6.4 us, through LDS 8.3; 64 requests of one row 8.7 and 10.0; 2,000 rows 12.5 both;
    // 3,500 rows 13.4 and 12.8, of rank 32 15.2 and 13.6; 8,000 rows 24.6 and 17.8. fp32 rows go through LDS always: one row of rank 16 6.4 us,
    // straight 7.1; 64 requests 7.9 and 9.4; 500 rows 7.2 and 9.4; 1,900 rows 12.7 and 15.1, of rank 32 14.3 and 19.3.
    const bool f32 = type == NXG_TYPE_F32;
    int rows = 16;
    // A tile's rows are of one document, so that the documents have to be long enough on the average, too (8 adapters, with 64 rows and
    // with 16: 65,536 rows of bf16 rank 64 in documents of 48 rows 114 and 200 us, of 32 143 and 164, of 16 226 and 281, of 8 406 and 285,
    // of 1 2,928 and 583; 32,768 of fp32 rank 128 of 48 rows 279 and 435, of 32 468 and 356, of 1 10,051 and 852).
    const int mean = p.T / p.n_seqs;
    if (w && p.r > (f32 ? 32 : 16) && mean >= (f32 ? 48 : 32)) {
        if (p.r > 64 && !f32 && p.T / 128 >= 2 * cus && mean >= 128) rows = 128;
        else if (p.T / 64 >= (p.r > 64 && !f32 ? 1 : 2) * cus) rows = 64;
    }
    const int64_t slots = p.T / rows + (int64_t) p.n_seqs;         // below 2^20 + 2^22
    const bool direct = !f32 && p.r <= 32 && slots < cus / 2;
    // Single rows, two an adapter on the average: those that share one go together (fp32, ids by chance, together and one by one: 65 rows of
    // 64 adapters of rank 16 11.0 and 10.3 us, of rank 128 both 35; 1,000 rows of 512 30 and 28, 131 and 161; 4,096 rows of 64 45 and 73,
    // 167 and 678). The window: so that 16 rows of an adapter are in it, but no larger than keeps its search short (16,384 rows of 512
    // adapters of rank 16 200, 162 and 200 us with 1,024, 4,096 and 8,192 documents, of rank 128 1,609, 926 and 1,062).
    p.gather = rows == 16 && p.T <= p.n_seqs && p.n_seqs / 2 >= p.n;
    p.window = 1024;
    while (p.window < MAX_WINDOW && p.window < 16 * (int64_t) p.n) p.window *= 2;
    const int64_t tiles = p.gather ? std::min<int64_t>(slots, (p.n_seqs + p.window - 1) / p.window * (int64_t) p.n + p.n_seqs / 16) : slots;
    // few tiles: several workgroups share out a tile's columns, each with the down product of its own
    int parts = 1;
    while (p.y && rows == 16 && tiles * parts * 2 <= cus && p.N > 32 * V * parts) parts *= 2;
    const dim3 grid((unsigned) slots, (unsigned) parts);
    hipStream_t s = (hipStream_t) stream;
    by_types(type, w_type, [&](auto e, auto we) {
        typedef decltype(e) E;
        typedef decltype(we) W;
        by_rank(p.r, [&](auto rt) {
            constexpr bool F32 = std::is_same<E, float>::value;
            if (!w) return adapter_rows_kernel<E, W, rt(), BY_VALUE><<<grid, 256, 0, s>>>(p);
            if constexpr (!F32 && rt() <= 2) {
                if (direct) return adapter_rows_kernel<E, W, rt(), WIDE><<<grid, 256, 0, s>>>(p);
            }
            if constexpr (!F32 && rt() == 8) {
                if (rows == 128) return adapter_rows_tall_kernel<E, W, 2, rt()><<<grid, 256, 0, s>>>(p);
            }
            if constexpr (rt() > (F32 ? 2 : 1)) {
                if (rows == 64) return adapter_rows_tall_kernel<E, W, 1, rt()><<<grid, 256, 0, s>>>(p);
            }
            adapter_rows_kernel<E, W, rt(), THROUGH_LDS><<<grid, 256, 0, s>>>(p);
        });
    });
    return nxg_launch_check(what);
}

// What the backward pass keeps in its workspace.
struct layout {
    int size, cw;                  // rows of a chunk, columns of a slab
    int64_t n_slots, n_parts;
    int64_t order, pos, counts, slots, of, at, bt, g, part_a, part_b, bytes;
    int runs;                      // of documents, in the plan
};
layout plan_backward(const nxg_adapter_rows_params & p) {
    layout l;
    const int es = size_of(p.type), ws = size_of(p.w_type);
    l.cw = es == 4 || p.rank > 64 ? 256 : 512;
    const int64_t slabs = (p.n_in + l.cw - 1) / l.cw + (p.n_out + l.cw - 1) / l.cw;
    // rows of a chunk: so that the workgroups, one more chunk an adapter counted in, are one a CU (32 documents of 4 adapters 30 us; a
    // few more than that many take 42); at most twice as many with many adapters
    const int64_t cus = nxg_device_cus(), room = std::max(cus - p.n_adapters * slabs, cus / 2);
    l.size = (int) std::min<int64_t>(CHUNK, std::max<int64_t>(64, (p.T * slabs / room + 32) / 32 * 32));
    l.n_slots = p.T / l.size + (int64_t) p.n_adapters;
    l.n_parts = 2 * (int64_t) p.T / l.size;            // adapters of more rows than a chunk have less than twice as many chunks as whole ones
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    l.order = take(4 * (int64_t) p.n_seqs);
    l.pos = take(4 * (int64_t) p.n_seqs);
    l.runs = std::min(16, std::max(1, (p.n_seqs + 63) / 64));
    l.counts = take(4 * (int64_t) l.runs * p.n_adapters);
    l.slots = take((int64_t) sizeof(chunk) * l.n_slots);
    l.of = take((int64_t) sizeof(adapter_rows_of) * p.n_adapters);
    l.at = take((int64_t) p.n_adapters * p.rank * p.n_in * ws);
    l.bt = take((int64_t) p.n_adapters * p.rank * p.n_out * ws);
    l.g = take((int64_t) p.T * p.rank * 4);
    l.part_a = take(l.n_parts * p.rank * p.n_in * 4);
    l.part_b = take(l.n_parts * p.rank * p.n_out * 4);
    l.bytes = at;
    return l;
}

} // namespace

extern "C" {

int32_t nxg_adapter_rows(const nxg_adapter_rows_params * params, const void * x, int64_t x_stride, const void * base,
                         int64_t base_stride, void * y, int64_t y_stride, float * s, void * stream) {
    const char * what = "adapter_rows";
    NXG_TRY(check_params(what, params));
    const nxg_adapter_rows_params & a = *params;
    if (a.T == 0 || a.n_seqs == 0) return NXG_OK;
    NXG_TRY(check_arrays(what, params));
    const int es = size_of(a.type);
    NXG_TRY(check_rows(what, "x", x, x_stride, a.T, a.n_in, es, false));
    if (base) NXG_TRY(check_rows(what, "base", base, base_stride, a.T, a.n_out, es, false));
    NXG_TRY(check_rows(what, "y", y, y_stride, a.T, a.n_out, es, true));
    if (!s || ((uintptr_t) s & 3)) return nxg_fail(NXG_EINVAL, "%s: s is null or not aligned to its type", what);
    if (y == base && a.T > 1 && y_stride != base_stride) return nxg_fail(NXG_EINVAL, "%s: y is base with another stride", what);
    if (y == x || y == (void *) s || x == (void *) s || base == (void *) s) return nxg_fail(NXG_EINVAL, "%s: y or s is another tensor of the call", what);
    NXG_TRY(nxg_check_device());
    adapter_p p = {};
    p.x = static_cast<const char *>(x);
    p.base = static_cast<const char *>(base);
    p.y = static_cast<char *>(y);
    p.a = a.a;
    p.b = a.b;
    p.s = s;
    p.x_s = a.T > 1 ? x_stride * es : 0;
    p.base_s = a.T > 1 ? base_stride * es : 0;
    p.y_s = a.T > 1 ? y_stride * es : 0;
    p.cu = a.cu;
    p.ids = a.ids;
    p.T = a.T;
    p.K = a.n_in;
    p.N = a.n_out;
    p.r = a.rank;
    p.n = a.n_adapters;
    p.n_seqs = a.n_seqs;
    p.pre = 1.0f;
    p.post = a.scale;
    return launch_rows(what, p, a.type, a.w_type, stream);
}

int64_t nxg_adapter_rows_backward_workspace_bytes(const nxg_adapter_rows_params * params) {
    const int32_t rc = check_params("adapter_rows_backward_workspace_bytes", params);
    return rc ? -rc : plan_backward(*params).bytes;
}

int32_t nxg_adapter_rows_backward(const nxg_adapter_rows_params * params, const void * dy, int64_t dy_stride, const void * x,
                                  int64_t x_stride, const float * s, const void * base, int64_t base_stride, void * dx,
                                  int64_t dx_stride, void * da, void * db, void * workspace, int64_t workspace_bytes, void * stream) {
    const char * what = "adapter_rows_backward";
    NXG_TRY(check_params(what, params));
    const nxg_adapter_rows_params & a = *params;
    if (!dx && !da && !db) return NXG_OK;
    NXG_TRY(check_arrays(what, params));
    const int es = size_of(a.type), ws = size_of(a.w_type);
    const bool some = a.T > 0 && a.n_seqs > 0;
    if (some) {
        NXG_TRY(check_rows(what, "dy", dy, dy_stride, a.T, a.n_out, es, false));
        if (da || db || x) NXG_TRY(check_rows(what, "x", x, x_stride, a.T, a.n_in, es, false));
        if (base) NXG_TRY(check_rows(what, "base", base, base_stride, a.T, a.n_in, es, false));
        if (dx) NXG_TRY(check_rows(what, "dx", dx, dx_stride, a.T, a.n_in, es, true));
        if (!s || ((uintptr_t) s & 3)) return nxg_fail(NXG_EINVAL, "%s: s is null or not aligned to its type", what);
        if (dx && dx == base && a.T > 1 && dx_stride != base_stride) return nxg_fail(NXG_EINVAL, "%s: dx is base with another stride", what);
        if (dx && (dx == dy || dx == x || dx == (const void *) s)) return nxg_fail(NXG_EINVAL, "%s: dx is another tensor of the call", what);
    }
    for (const void * o : {(const void *) da, (const void *) db}) {
        if (!o) continue;
        if ((uintptr_t) o & (ws - 1)) return nxg_fail(NXG_EINVAL, "%s: da or db is not aligned to its type", what);
        if (o == dy || o == x || o == (const void *) s || o == base || o == dx || o == a.a || o == a.b || da == db) {
            return nxg_fail(NXG_EINVAL, "%s: da or db is another tensor of the call", what);
        }
    }
    const layout l = plan_backward(a);
    if (!workspace || ((uintptr_t) workspace & 15) || workspace_bytes < l.bytes) {
        return nxg_fail(NXG_EINVAL, "%s: workspace must be 16-byte aligned memory of %lld bytes", what, (long long) l.bytes);
    }
    char * w = static_cast<char *>(workspace);
    grads_p p = {};
    p.cu = a.cu;
    p.ids = a.ids;
    p.T = a.T;
    p.K = a.n_in;
    p.N = a.n_out;
    p.r = a.rank;
    p.n = a.n_adapters;
    p.n_seqs = some ? a.n_seqs : 0;
    p.size = l.size;
    p.n_slots = (int32_t) l.n_slots;
    p.slabs_a = da ? (a.n_in + l.cw - 1) / l.cw : 0;
    p.slabs_b = db ? (a.n_out + l.cw - 1) / l.cw : 0;
    p.a = a.a;
    p.b = a.b;
    p.at = w + l.at;
    p.bt = w + l.bt;
    p.order = reinterpret_cast<int32_t *>(w + l.order);
    p.pos = reinterpret_cast<int32_t *>(w + l.pos);
    p.counts = reinterpret_cast<int32_t *>(w + l.counts);
    p.runs = l.runs;
    p.slots = reinterpret_cast<chunk *>(w + l.slots);
    p.of = reinterpret_cast<adapter_rows_of *>(w + l.of);
    p.x = static_cast<const char *>(x);
    p.dy = static_cast<const char *>(dy);
    p.x_s = a.T > 1 ? x_stride * es : 0;
    p.dy_s = a.T > 1 ? dy_stride * es : 0;
    p.g = reinterpret_cast<const float *>(w + l.g);
    p.s = s;
    p.part_a = reinterpret_cast<float *>(w + l.part_a);
    p.part_b = reinterpret_cast<float *>(w + l.part_b);
    p.da = da;
    p.db = db;
    p.whole = (((uintptr_t) da | (uintptr_t) db) & 15) == 0;
    p.scale = a.scale;
    p.w_type = a.w_type;
    const int64_t turned = (int64_t) a.n_adapters * ((a.n_in + 63) / 64 + (a.n_out + 63) / 64);
    const int64_t jobs = l.n_slots * (p.slabs_a + p.slabs_b);
    // the strips' workgroups have 1,024 threads, four times the others'
    if (turned >= MAX_GRID / 4 || jobs > MAX_GRID) return nxg_fail(NXG_EINVAL, "%s: T=%d n_adapters=%d is too large", what, a.T, a.n_adapters);
    NXG_TRY(nxg_check_device());
    hipStream_t st = (hipStream_t) stream;
    auto prepare = [&](int64_t grid, int parts) {
        by_type(a.w_type, [&](auto we) { adapter_prepare_kernel<decltype(we)><<<(unsigned) grid, 1024, 0, st>>>(p, parts); });
        return nxg_launch_check(what);
    };
    if (some && p.n_seqs * (int64_t) p.n <= FEW_PAIRS) {
        NXG_TRY(prepare(1 + turned, PLAN | TURN));
    } else {
        NXG_TRY(prepare(1, PLAN));
        if (some) NXG_TRY(prepare(turned, TURN));
    }
    if (some && (dx || da)) {
        adapter_p f = {};
        f.x = p.dy;
        f.base = static_cast<const char *>(base);
        f.y = static_cast<char *>(dx);
        f.a = p.bt;
        f.b = p.at;
        f.s = reinterpret_cast<float *>(w + l.g);
        f.x_s = p.dy_s;
        f.base_s = a.T > 1 ? base_stride * es : 0;
        f.y_s = a.T > 1 ? dx_stride * es : 0;
        f.cu = a.cu;
        f.ids = a.ids;
        f.T = a.T;
        f.K = a.n_out;
        f.N = a.n_in;
        f.r = a.rank;
        f.n = a.n_adapters;
        f.n_seqs = a.n_seqs;
        f.pre = a.scale;
        f.post = 1.0f;
        NXG_TRY(launch_rows(what, f, a.type, a.w_type, stream));
    }
    if (jobs == 0) return NXG_OK;
    // V columns at a time, in what is read and in what is written: without rows their number alone decides
    const int V = 16 / es;
    const bool wd = (!da || (a.n_in % V == 0 && (!some || wide(x, p.x_s)))) && (!db || (a.n_out % V == 0 && (!some || wide(dy, p.dy_s))));
    by_type(a.type, [&](auto e) {
        typedef decltype(e) E;
        by_rank(a.rank, [&](auto rt) {
            constexpr int VC = sizeof(E) == 4 || rt() == 8 ? 4 : 8;
            if (wd) adapter_grads_kernel<E, rt(), VC, true><<<(unsigned) jobs, 256, 0, st>>>(p);
            else adapter_grads_kernel<E, rt(), VC, false><<<(unsigned) jobs, 256, 0, st>>>(p);
        });
    });
    NXG_TRY(nxg_launch_check(what));
    if (l.n_parts == 0) return NXG_OK;
    p.n_out_blocks = (int32_t) (((da ? (int64_t) a.rank * a.n_in : 0) + (db ? (int64_t) a.rank * a.n_out : 0) + 63) / 64);
    adapter_join_kernel<<<(unsigned) (p.n_out_blocks * (int64_t) a.n_adapters), 256, 0, st>>>(p);
    return nxg_launch_check(what);
}

} // extern "C"
