// nxg_adapter_rows.hip -- gfx950 low-rank adapters over packed rows, forward and backward, and their C ABI
// (include/nxg_rows.h).
//
// A document's rows go through two thin products, down to `rank` values and up again. The forward pass and dx are the same
// kernel: s = x A^T, y = base + s B^T, and g = dy B, dx = base + g A with the weights turned round beforehand. What is left are sums
// over rows, g^T x and s^T dy, for each adapter. All of it is bound by HBM for ranks up to 64: the matrix instructions are
// 16x16 ones (32 values of the contracted index in 16 bits, 4 in fp32), whose operands come from memory straight into registers.
//
// s and g stay fp32. Beside 16-bit rows they enter the next product as the sum of two bf16 values, which is off by at most
// 2^-16 of a value, beside a result's own rounding by 2^-8 (bf16) or 2^-11 (fp16). fp16 rows and weights are the sum of two bf16
// values exactly, and of the four products only that of both second parts is left out (2^-16 again); so no value leaves
// a type's range on the way. Beside fp32 rows every product is fp32.

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

// Values k .. k + V - 1 of a row of n values, zeros behind its end. WIDE: 16 bytes of the row at once (n and k multiples of V).
template <class E, class S, bool WIDE>
__device__ __forceinline__ typename operand<E>::vec fetch(const S * row, int k, int n) {
    constexpr int V = operand<E>::V;
    typename operand<E>::vec v;
    if constexpr (WIDE) {
        typedef S svec __attribute__((ext_vector_type(V)));
        svec x;
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (S) 0.0f;
        if (k < n) x = *reinterpret_cast<const svec *>(row + k);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (E) x[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = k + i < n ? (E) row[k + i] : (E) 0.0f;
    }
    return v;
}

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
};

struct tile {
    int row, len, id;              // rows row .. row + len - 1 of adapter id
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
    const int id = uni(p.ids[lo]);
    t.id = id >= 0 && id < p.n ? id : -1;
    return t;
}

// A workgroup: 16 MT rows of one document. Its four waves share the contracted index of x A^T out, a line of 128 bytes of every
// row at a time, so that the weights are read once per workgroup; their sums are joined in LDS, in a fixed order. Then they
// share out the columns of s B^T, taken as (B s^T): a lane has V columns next to each other of one row, 16 bytes, from
// V / 4 results whose rows of B are picked for that.
template <class E, class W, int MT, int RT, bool WIDE>
__global__ __launch_bounds__(256) void adapter_rows_kernel(adapter_p p) {
    constexpr bool F32 = std::is_same<E, float>::value, F16 = std::is_same<E, _Float16>::value;
    constexpr int V = operand<E>::V, BM = 16 * MT, RP = 16 * RT, LD = RP + 4;
    typedef typename operand<E>::vec vec;
    __shared__ __align__(16) float lds[2][BM][LD];
    const tile c = find_tile(p, BM, blockIdx.x);
    if (c.len <= 0) return;
    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;

    if (c.id < 0) {                // no adapter: base as it is, s = 0
        if (blockIdx.y) return;
        for (int i = threadIdx.x; i < c.len * p.r; i += 256) p.s[(int64_t) c.row * p.r + i] = 0.0f;
        if (!p.y || p.y == p.base) return;
        for (int t = wave; t < c.len; t += 4) {
            const E * from = reinterpret_cast<const E *>(p.base + (c.row + (int64_t) t) * p.base_s);
            E * to = reinterpret_cast<E *>(p.y + (c.row + (int64_t) t) * p.y_s);
            for (int k = lane; k < p.N; k += 64) to[k] = p.base ? from[k] : (E) 0.0f;
        }
        return;
    }

    // s, ranks as rows and tokens as columns
    v4f acc[MT][RT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[m][j] = v4f{};
    {
        const E * x[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) x[m] = reinterpret_cast<const E *>(p.x + (c.row + (int64_t) min(16 * m + col, c.len - 1)) * p.x_s);
        const W * a = static_cast<const W *>(p.a) + (int64_t) c.id * p.r * p.K;
#pragma unroll 1
        for (int k0 = wave * 8 * V; k0 < p.K; k0 += 32 * V) {
            vec xf[2][MT], af[2][RT];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = k0 + (2 * g + h) * V;
#pragma unroll
                for (int m = 0; m < MT; ++m) xf[h][m] = fetch<E, E, WIDE>(x[m], k, p.K);
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    const int r = 16 * j + col;
                    af[h][j] = fetch<E, W, WIDE>(a + (int64_t) r * p.K, r < p.r ? k : p.K, p.K);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int j = 0; j < RT; ++j) acc[m][j] = operand<E>::mul(af[h][j], xf[h][m], acc[m][j]);
        }
    }
    // the waves' sums: 0 + 2 and 1 + 3, then both
    for (int turn = 0; turn < 2; ++turn) {
        if ((wave >> 1) == turn) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    v4f * to = reinterpret_cast<v4f *>(&lds[wave & 1][16 * m + col][16 * j + 4 * g]);
                    *to = turn ? *to + acc[m][j] : acc[m][j];
                }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < BM * RP; i += 256) {
        const int t = i / RP, r = i % RP;
        const float x = (lds[0][t][r] + lds[1][t][r]) * p.pre;
        lds[0][t][r] = x;
        if (blockIdx.y == 0 && t < c.len && r < p.r) p.s[(c.row + (int64_t) t) * p.r + r] = x;
    }
    if (!p.y) return;
    __syncthreads();

    // s as operands
    constexpr int Q = F32 ? RT : RT == 1 ? 1 : RT / 2;      // ranks of one: 16 (fp32, and RT 1 with both parts side by side), else 32
    constexpr int SV = F32 || RT == 1 ? 1 : 2;              // operands for them
    typedef typename std::conditional<F32, v4f, v8b>::type svec;
    svec s[MT][Q][SV];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const float * row = lds[0][16 * m + col];
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            if constexpr (F32) {
                s[m][q][0] = *reinterpret_cast<const v4f *>(row + 16 * q + 4 * g);
            } else {
                const float * f = row + (RT == 1 ? 8 * (g & 1) : 32 * q + 8 * g);
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = f[i];
                v8b hi, lo;
                split(x, hi, lo);
                if constexpr (RT == 1) {
                    s[m][q][0] = g < 2 ? hi : lo;
                } else {
                    s[m][q][0] = hi;
                    s[m][q][1] = lo;
                }
            }
        }
    }

    constexpr int M = V / 4;       // results that make up a lane's 16 bytes
    const W * b = static_cast<const W *>(p.b) + (int64_t) c.id * p.N * p.r;
    const bool whole = p.r % V == 0;
    for (int n0 = (blockIdx.y * 4 + wave) * 8 * V; n0 < p.N; n0 += 32 * V * (int) gridDim.y) {
        // two groups of 4 V columns: 128 bytes of a row
        vec before[2][MT];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int n = n0 + 4 * V * h + V * g, t = 16 * m + col;
                const E * from = reinterpret_cast<const E *>(p.base + (c.row + (int64_t) t) * p.base_s);
                before[h][m] = fetch<E, E, WIDE>(from, p.base && t < c.len ? n : p.N, p.N);
            }
        vec bf[2][M][Q];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < M; ++i) {
                const W * row = b + (int64_t) min(n0 + 4 * V * h + V * (col >> 2) + 4 * i + (col & 3), p.N - 1) * p.r;
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    const int r = F32 ? 16 * q + 4 * g : RT == 1 ? 8 * (g & 1) : 32 * q + 8 * g;
                    if (whole) bf[h][i][q] = fetch<E, W, true>(row, r, p.r);
                    else bf[h][i][q] = fetch<E, W, false>(row, r, p.r);
                }
            }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v4f up[M][MT];
#pragma unroll
            for (int i = 0; i < M; ++i) {
#pragma unroll
                for (int m = 0; m < MT; ++m) up[i][m] = v4f{};
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    if constexpr (F32) {
#pragma unroll
                        for (int m = 0; m < MT; ++m) up[i][m] = operand<float>::mul(bf[h][i][q], s[m][q][0], up[i][m]);
                    } else {
                        v8b hi, lo;
                        if constexpr (F16) split(bf[h][i][q], hi, lo);
                        else hi = bf[h][i][q];
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
#pragma unroll
                            for (int k = 0; k < SV; ++k) up[i][m] = operand<__bf16>::mul(hi, s[m][q][k], up[i][m]);
                            if constexpr (F16) up[i][m] = operand<__bf16>::mul(lo, s[m][q][0], up[i][m]);
                        }
                    }
                }
            }
            const int n = n0 + 4 * V * h + V * g;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int t = 16 * m + col;
                vec out;
#pragma unroll
                for (int i = 0; i < V; ++i) out[i] = (E) __builtin_fmaf(up[i / 4][m][i % 4], p.post, (float) before[h][m][i]);
                if (t >= c.len) continue;
                E * to = reinterpret_cast<E *>(p.y + (c.row + (int64_t) t) * p.y_s);
                if constexpr (WIDE) {
                    if (n < p.N) *reinterpret_cast<vec *>(to + n) = out;
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (n + i < p.N) to[n + i] = out[i];
                }
            }
        }
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
    chunk * slots;
    adapter_rows_of * of;
    const char * x, * dy;
    int64_t x_s, dy_s;
    const float * g, * s;
    float * part_a, * part_b;      // [parts][r][K], [parts][r][N]
    void * da, * db;
    float scale;
    int32_t w_type, n_out_blocks;
};

__device__ __forceinline__ int scan64(int x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 1; k < 64; k *= 2) {
        const int y = __shfl_up(x, k);
        x += lane >= k ? y : 0;
    }
    return x;
}

// Who has which rows: by one workgroup, a wave an adapter. Sums are kept at most T, so that offsets that do not rise
// make no place past the arrays.
__device__ void plan_rows(const grads_p & p) {
    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
    auto length = [&](int d, int id) {
        return d < p.n_seqs && p.ids[d] == id ? max(offset(p.cu, d + 1, p.T) - offset(p.cu, d, p.T), 0) : -1;
    };
    for (int id = wave; id < p.n; id += 16) {
        int rows = 0, docs = 0;
        for (int d0 = 0; d0 < p.n_seqs; d0 += 64) {
            const int len = length(d0 + lane, id);
            docs += __popcll(__ballot(len >= 0));
            rows = min(rows + uni(__shfl(scan64(max(len, 0)), 63)), p.T);
        }
        if (lane == 0) {
            p.of[id].rows = rows;
            p.of[id].docs = docs;
        }
    }
    __syncthreads();
    if (wave == 0) {
        int row = 0, doc = 0, slot = 0, part = 0;
        for (int i0 = 0; i0 < p.n; i0 += 64) {
            const int id = i0 + lane;
            const int rows = id < p.n ? p.of[id].rows : 0, docs = id < p.n ? p.of[id].docs : 0;
            // 64 times T is below 2^31
            const int upto = min(row + scan64(rows), p.T), here = min(row + scan64(rows) - rows, p.T);
            const int chunks = id < p.n ? max((upto - here + p.size - 1) / p.size, 1) : 0, parts = chunks > 1 ? chunks : 0;
            const int d = doc + scan64(docs), c = slot + scan64(chunks), q = part + scan64(parts);
            if (id < p.n) {
                adapter_rows_of o;
                o.row = here;
                o.rows = upto - here;
                o.doc = d - docs;
                o.docs = docs;
                o.slot = c - chunks;
                o.part = q - parts;
                o.chunks = chunks;
                o.unused = 0;
                p.of[id] = o;
            }
            row = uni(__shfl(upto, 63));
            doc = uni(__shfl(d, 63));
            slot = uni(__shfl(c, 63));
            part = uni(__shfl(q, 63));
        }
        for (int k = slot + lane; k < p.n_slots; k += 64) p.slots[k].id = -1;
    }
    __syncthreads();
    for (int id = wave; id < p.n; id += 16) {
        const adapter_rows_of o = p.of[id];
        for (int k = lane; k < o.chunks && o.slot + k < p.n_slots; k += 64) {
            chunk c;
            c.id = id;
            c.from = o.row + k * p.size;
            c.count = min(p.size, o.rows - k * p.size);
            c.part = o.chunks > 1 ? o.part + k : -1;
            p.slots[o.slot + k] = c;
        }
        int rows = 0, docs = 0;
        for (int d0 = 0; d0 < p.n_seqs; d0 += 64) {
            const int len = length(d0 + lane, id);
            const uint64_t mine = __ballot(len >= 0);
            const int upto = scan64(max(len, 0));
            if (len >= 0) {
                const int k = o.doc + docs + __popcll(mine & ((1ull << lane) - 1));
                p.order[k] = d0 + lane;
                p.pos[k] = o.row + min(rows + upto - len, o.rows);
            }
            docs += __popcll(mine);
            rows = min(rows + uni(__shfl(upto, 63)), p.T);
        }
    }
}

// The first workgroup: plan_rows. Each other one: 64 columns of one adapter's down weights, or 64 rows of its up weights, turned round.
template <class W>
__global__ __launch_bounds__(1024) void adapter_prepare_kernel(grads_p p) {
    if (blockIdx.x == 0) {
        plan_rows(p);
        return;
    }
    __shared__ W lds[MAX_RANK][66];
    const int strips_k = (p.K + 63) / 64, strips = strips_k + (p.N + 63) / 64;
    const int id = (blockIdx.x - 1) / strips, strip = (blockIdx.x - 1) % strips;
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

// The sum over a chunk's rows of u^T z, r x 16 V columns: u = g, z = x (dA), or u = s, z = dy (dB). A wave takes every
// fourth 32 rows: a lane loads 16 bytes of 8 rows, whose values of one column, next to each other after a
// permutation of bytes, are the operand as it is (its 16 lanes' columns are V apart). The waves' sums are joined in LDS, in order.
constexpr int CHUNK = 1024;        // rows of a chunk, at most
template <class E, int RT, int V, bool WIDE>
__global__ __launch_bounds__(256) void adapter_grads_kernel(grads_p p) {
    constexpr bool F32 = std::is_same<E, float>::value, F16 = std::is_same<E, _Float16>::value;
    constexpr int RP = 16 * RT, CW = 16 * V;
    typedef E evec __attribute__((ext_vector_type(V)));
    __shared__ __align__(16) int rows[CHUNK];
    __shared__ __align__(16) float sum[RP][CW + 4];
    const int slabs = p.slabs_a + p.slabs_b, slab = blockIdx.x % slabs;
    const chunk c = p.slots[blockIdx.x / slabs];
    if (c.id < 0) return;
    const bool down = slab < p.slabs_a;
    const int C = down ? p.K : p.N, c0 = (down ? slab : slab - p.slabs_a) * CW;
    const char * z = down ? p.x : p.dy;
    const int64_t z_s = down ? p.x_s : p.dy_s;
    const float * u = down ? p.g : p.s;
    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;

    const int doc = p.of[c.id].doc, docs = p.of[c.id].docs;
    for (int i = threadIdx.x; i < c.count; i += 256) {
        int lo = doc, hi = doc + docs - 1;             // the last document that starts there or before
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (p.pos[mid] <= c.from + i) lo = mid;
            else hi = mid - 1;
        }
        rows[i] = min(max(offset(p.cu, p.order[lo], p.T) + c.from + i - p.pos[lo], 0), p.T - 1);
    }
    __syncthreads();

    v4f acc[V][RT];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[v][j] = v4f{};
    for (int t0 = wave * 32; t0 < c.count; t0 += 128) {
        evec zv[8];
        float uv[RT][8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int t = t0 + 8 * g + k;
            const bool some = t < c.count;
            const int64_t row = some ? rows[t] : 0;
            const E * from = reinterpret_cast<const E *>(z + row * z_s) + c0 + V * col;
#pragma unroll
            for (int v = 0; v < V; ++v) zv[k][v] = (E) 0.0f;
            if constexpr (WIDE) {
                if (some && c0 + V * col < C) zv[k] = *reinterpret_cast<const evec *>(from);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (some && c0 + V * col + v < C) zv[k][v] = from[v];
            }
#pragma unroll
            for (int j = 0; j < RT; ++j) uv[j][k] = some && 16 * j + col < p.r ? u[row * p.r + 16 * j + col] : 0.0f;
        }
        if constexpr (F32) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int j = 0; j < RT; ++j) acc[v][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(uv[j][k], zv[k][v], acc[v][j], 0, 0, 0);
        } else {
            v8b hi[RT], lo[RT];
#pragma unroll
            for (int j = 0; j < RT; ++j) split(uv[j], hi[j], lo[j]);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                typename operand<E>::vec zc;
#pragma unroll
                for (int k = 0; k < 8; ++k) zc[k] = zv[k][v];
                v8b zh, zl;
                if constexpr (F16) split(zc, zh, zl);
                else zh = zc;
#pragma unroll
                for (int j = 0; j < RT; ++j) {
                    acc[v][j] = operand<__bf16>::mul(hi[j], zh, acc[v][j]);
                    acc[v][j] = operand<__bf16>::mul(lo[j], zh, acc[v][j]);
                    if constexpr (F16) acc[v][j] = operand<__bf16>::mul(hi[j], zl, acc[v][j]);
                }
            }
        }
    }
    for (int turn = 0; turn < 4; ++turn) {
        if (wave == turn) {
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int v = 0; v < V; v += 4) {
                        v4f * to = reinterpret_cast<v4f *>(&sum[16 * j + 4 * g + i][V * col + v]);
                        const v4f x = {acc[v][j][i], acc[v + 1][j][i], acc[v + 2][j][i], acc[v + 3][j][i]};
                        *to = turn ? *to + x : x;
                    }
        }
        __syncthreads();
    }
    const int cols = min(CW, C - c0);
    const float f = down ? 1.0f : p.scale;
    if (c.part >= 0) {
        float * to = (down ? p.part_a : p.part_b) + (int64_t) c.part * p.r * C + c0;
        for (int i = threadIdx.x; i < p.r * CW; i += 256)
            if (i % CW < cols) to[(int64_t) (i / CW) * C + i % CW] = sum[i / CW][i % CW] * f;
    } else if (down) {
        for (int i = threadIdx.x; i < p.r * CW; i += 256)
            if (i % CW < cols) put(p.da, ((int64_t) c.id * p.r + i / CW) * C + c0 + i % CW, sum[i / CW][i % CW], p.w_type);
    } else {
        for (int i = threadIdx.x; i < p.r * cols; i += 256) put(p.db, ((int64_t) c.id * C + c0) * p.r + i, sum[i % p.r][i / p.r] * f, p.w_type);
    }
}

// The chunks' sums of the adapters that have several, in order: a value a lane, its four waves every fourth chunk.
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
    const bool w = wide(p.x, p.x_s) && (!p.base || wide(p.base, p.base_s)) && wide(p.y, p.y ? p.y_s : 0) && p.K % V == 0 && p.N % V == 0;
    // 64 rows a workgroup read the weights a quarter as often as 16, where that leaves work for every CU
    const bool tall = w && p.T / 64 >= 2 * cus;
    const int64_t slots = p.T / (tall ? 64 : 16) + (int64_t) p.n_seqs;
    if (slots > MAX_GRID) return nxg_fail(NXG_EINVAL, "%s: T=%d n_seqs=%d is too large", what, p.T, p.n_seqs);
    // few rows: several workgroups share out the columns, each with the down product of its own
    int parts = 1;
    while (p.y && !tall && slots * parts * 2 <= cus && p.N > 32 * V * parts) parts *= 2;
    const dim3 grid((unsigned) slots, (unsigned) parts);
    hipStream_t s = (hipStream_t) stream;
    by_types(type, w_type, [&](auto e, auto we) {
        typedef decltype(e) E;
        typedef decltype(we) W;
        by_rank(p.r, [&](auto rt) {
            if (tall) adapter_rows_kernel<E, W, 4, rt(), true><<<grid, 256, 0, s>>>(p);
            else if (w) adapter_rows_kernel<E, W, 1, rt(), true><<<grid, 256, 0, s>>>(p);
            else adapter_rows_kernel<E, W, 1, rt(), false><<<grid, 256, 0, s>>>(p);
        });
    });
    return nxg_launch_check(what);
}

// What the backward pass keeps in its workspace.
struct layout {
    int size, cw;                  // rows of a chunk, columns of a slab
    int64_t n_slots, n_parts;
    int64_t order, pos, slots, of, at, bt, g, part_a, part_b, bytes;
};
layout plan_backward(const nxg_adapter_rows_params & p) {
    layout l;
    const int es = size_of(p.type), ws = size_of(p.w_type);
    l.cw = es == 4 || p.rank > 64 ? 64 : 128;
    const int64_t slabs = (p.n_in + l.cw - 1) / l.cw + (p.n_out + l.cw - 1) / l.cw;
    // rows of a chunk: as many as leave about four workgroups a CU
    l.size = CHUNK;
    while (l.size > 128 && p.T / l.size * slabs < 4 * nxg_device_cus()) l.size /= 2;
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
    p.scale = a.scale;
    p.w_type = a.w_type;
    const int64_t turned = (int64_t) a.n_adapters * ((a.n_in + 63) / 64 + (a.n_out + 63) / 64);
    const int64_t jobs = l.n_slots * (p.slabs_a + p.slabs_b);
    if (turned >= MAX_GRID || jobs > MAX_GRID) return nxg_fail(NXG_EINVAL, "%s: T=%d n_adapters=%d is too large", what, a.T, a.n_adapters);
    NXG_TRY(nxg_check_device());
    hipStream_t st = (hipStream_t) stream;
    by_type(a.w_type, [&](auto we) { adapter_prepare_kernel<decltype(we)><<<(unsigned) (some ? 1 + turned : 1), 1024, 0, st>>>(p); });
    NXG_TRY(nxg_launch_check(what));
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
    const int V = 16 / es;
    const bool wd = (!da || !some || (wide(x, p.x_s) && a.n_in % V == 0)) && (!db || !some || (wide(dy, p.dy_s) && a.n_out % V == 0));
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
