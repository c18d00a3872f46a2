// nxg_rows.hip -- gfx950 kernels over packed floating-point rows: rotary positions, layer norm, head norms with rotary positions (both
// with their gradients) and dropout, and their C ABI (include/nxg_rows.h). All of them are bound by HBM: rows are read and written
// 16 bytes per lane, once.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "nxg_rows.h"
#include "nxg_internal.h"

namespace {

// V values at p (16 bytes, or one value), and back.
template <class E, int V>
__device__ __forceinline__ void load(float (&x)[V], const E * p) {
    typedef E vec __attribute__((ext_vector_type(V == 1 ? 2 : V)));
    if constexpr (V == 1) {
        x[0] = (float) *p;
    } else {
        const vec v = *reinterpret_cast<const vec *>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (float) v[i];
    }
}
// The same for rows that are read and written once, by the caches' own hint (dropout of 65,536 rows 99 us for 110).
template <class E, int V>
__device__ __forceinline__ void load_once(float (&x)[V], const E * p) {
    typedef E vec __attribute__((ext_vector_type(V == 1 ? 2 : V)));
    if constexpr (V == 1) {
        x[0] = (float) *p;
    } else {
        const vec v = __builtin_nontemporal_load(reinterpret_cast<const vec *>(p));
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (float) v[i];
    }
}
template <class E, int V>
__device__ __forceinline__ void store(E * p, const float (&x)[V]) {
    typedef E vec __attribute__((ext_vector_type(V == 1 ? 2 : V)));
    if constexpr (V == 1) {
        *p = (E) x[0];
    } else {
        vec v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (E) x[i];
        *reinterpret_cast<vec *>(p) = v;
    }
}
template <class E, int V>
__device__ __forceinline__ void store_once(E * p, const float (&x)[V]) {
    typedef E vec __attribute__((ext_vector_type(V == 1 ? 2 : V)));
    if constexpr (V == 1) {
        *p = (E) x[0];
    } else {
        vec v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (E) x[i];
        __builtin_nontemporal_store(v, reinterpret_cast<vec *>(p));
    }
}

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------

struct rope_p {
    const void * x;
    void * out;
    int64_t x_ts, x_hs, o_ts, o_hs;        // strides in values
    const double * freq;
    const int32_t * positions, * cu;
    int32_t T, H, D, n, n_seqs, tb, hb;    // tokens of a workgroup, heads of one (grid.y)
    uint32_t by_token, by_head, by_token_last;   // 2^32 / pieces of a token's heads, of a head, of a token in the last grid.y, rounded up
    float mscale, sign;
    bool copy;                             // out is not x: values behind n are written too
};

// The largest d with cu[d] <= t (0 if none), t's document: for all lanes of a wave, 64 documents at a time.
__device__ __forceinline__ int doc_of_rows(const int32_t * cu, int n_seqs, int t) {
    int lo = 0, n = n_seqs;
    while (n > 1) {
        const int step = (n + 63) >> 6, k = (threadIdx.x & 63) * step;
        const int last = max((int) __popcll(__ballot(k < n && cu[lo + k] <= t)) - 1, 0);
        n = min(step, n - last * step);
        lo += last * step;
    }
    return lo;
}

// The turns of `tokens` rows from t0, [tokens][half], as (cos, sin) times the factor on the result, by the 256 threads of a workgroup.
template <class P>
__device__ __forceinline__ void find_turns(float2 * turn, const P & p, int t0, int tokens, int half) {
    const int first = p.positions ? 0 : doc_of_rows(p.cu, p.n_seqs, t0);
    for (int k = threadIdx.x; k < tokens * half; k += 256) {
        const int t = t0 + k / half, i = k % half;
        const double f = p.freq[i];
        int pos;
        if (p.positions) {
            pos = p.positions[t];
        } else {
            // steps of 1, 2, 4, .. documents on, then halves: one load where the row is in the first, 2 log2(n) behind n empty ones
            uint32_t d = first, step = 1;
            const uint32_t n = p.n_seqs;
            for (; d + step < n && p.cu[d + step] <= t; step *= 2) d += step;
            while (step /= 2)
                if (d + step < n && p.cu[d + step] <= t) d += step;
            pos = t - p.cu[d];
        }
        const double turns = (double) pos * f * 0.15915494309189533577;   // 1 / (2 pi)
        float s, c;
        sincospif(2.0f * (float) (turns - rint(turns)), &s, &c);
        turn[k] = make_float2(c * p.mscale, s * p.mscale * p.sign);
    }
}

// A workgroup: tb tokens of hb heads. Their angles once, into LDS: position * frequency in 64 bits, as
// turns less whole turns, then fp32 (error 2^-25 of a turn). Then the heads' rows as one run of
// pieces, neighbouring lanes on neighbouring pieces: V values of a head from i and V from i + n / 2
// (HALF), V values in a row (else; a pair of single values where V is 1), or V values behind n to copy.
// Bound by HBM: 65,536 tokens of 24 heads of 64 in a fused projection's rows, fp32, 805 MB in 153 us, 5.3 TB/s (a large copy
// reaches 5.1 to 5.5); loads and stores past the caches take 246 to 261. Divisions are multiplications by a 32-bit
// reciprocal, exact for the numbers of a workgroup.
template <class E, int V, bool HALF>
__global__ __launch_bounds__(256) void rope_rows_kernel(rope_p p) {
    extern __shared__ float2 turn[];       // [tb][n / 2]
    const int half = p.n / 2;
    const int64_t t0 = (int64_t) blockIdx.x * p.tb;
    const int tokens = (int) min((int64_t) p.tb, p.T - t0);
    find_turns(turn, p, (int) t0, tokens, half);
    __syncthreads();
    const int h0 = blockIdx.y * p.hb, heads = min(p.hb, p.H - h0);
    const int pieces = HALF || V == 1 ? half / V : p.n / V, per_head = pieces + (p.copy ? (p.D - p.n) / V : 0), per_token = per_head * heads;
    const E * x0 = (const E *) p.x;
    E * o0 = (E *) p.out;
    const uint32_t by_token = heads == p.hb ? p.by_token : p.by_token_last;
    for (int k = threadIdx.x; k < tokens * per_token; k += 256) {
        // k / per_token and r / per_head: exact while k * per_token < 2^32
        const int t = by_token ? __umulhi(k, by_token) : k, r = k - t * per_token;
        const int h = p.by_head ? __umulhi(r, p.by_head) : r, piece = r - h * per_head;
        const E * x = x0 + (t0 + t) * p.x_ts + (h0 + h) * p.x_hs;
        E * o = o0 + (t0 + t) * p.o_ts + (h0 + h) * p.o_hs;
        if (piece >= pieces) {
            const int d = p.n + (piece - pieces) * V;
            float a[V];
            load<E, V>(a, x + d);
            store<E, V>(o + d, a);
            continue;
        }
        if constexpr (HALF || V == 1) {
            const float2 * w = turn + t * half + piece * V;
            const int da = HALF ? piece * V : 2 * piece, db = HALF ? half + piece * V : 2 * piece + 1;
            float a[V], b[V], y[V], z[V];
            load<E, V>(a, x + da);
            load<E, V>(b, x + db);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float c = w[i].x, s = w[i].y;
                y[i] = a[i] * c - b[i] * s;
                z[i] = a[i] * s + b[i] * c;
            }
            store<E, V>(o + da, y);
            store<E, V>(o + db, z);
        } else {
            const float2 * w = turn + t * half + piece * (V / 2);
            float a[V], y[V];
            load<E, V>(a, x + piece * V);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float c = w[i].x, s = w[i].y;
                y[2 * i] = a[2 * i] * c - a[2 * i + 1] * s;
                y[2 * i + 1] = a[2 * i] * s + a[2 * i + 1] * c;
            }
            store<E, V>(o + piece * V, y);
        }
    }
}

// ---------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------

template <int TPR>
__device__ __forceinline__ float row_sum(float x, float * lds) {
#pragma unroll
    for (int k = 32; k; k >>= 1) x += __shfl_xor(x, k);
    if constexpr (TPR == 64) return x;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

struct norm_p {
    const void * x, * dy, * w, * b;
    void * y, * dx, * dw, * db;
    float * mean, * rstd, * part;          // part: [workgroups][2][C]
    int64_t x_s, dy_s, y_s, dx_s;
    int32_t T, C, n_part;
    float eps;
};

// A row by TPR threads (a wave, or the workgroup), held in registers as NC pieces of V values a thread: one
// read, the mean, then the squares of what is left. Bound by HBM: 65,536 rows of 1,024 bf16 values, 269 MB in 41 to 43 us,
// 6.3 TB/s (part of the output stays in the last cache); 8,192 rows of 8,192 in 45 us.
template <class E, class W, int V, int NC, int TPR>
__global__ __launch_bounds__(256) void layer_norm_rows_kernel(norm_p p) {
    __shared__ float lds[4];
    const int64_t row = (int64_t) blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const int t = threadIdx.x % TPR;
    if (row >= p.T) return;                // whole waves, or whole workgroups
    const E * x = (const E *) p.x + row * p.x_s;
    E * y = (E *) p.y + row * p.y_s;
    float v[NC][V], s = 0.0f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        const int c = (k * TPR + t) * V;
        if (c < p.C) {
            load<E, V>(v[k], x + c);
#pragma unroll
            for (int i = 0; i < V; ++i) s += v[k][i];
        }
    }
    const float mean = row_sum<TPR>(s, lds) / (float) p.C;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        if ((k * TPR + t) * V < p.C) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[k][i] -= mean;
                s += v[k][i] * v[k][i];
            }
        }
    }
    const float rstd = 1.0f / sqrtf(row_sum<TPR>(s, lds) / (float) p.C + p.eps);
    if (t == 0) {
        if (p.mean) p.mean[row] = mean;
        if (p.rstd) p.rstd[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        const int c = (k * TPR + t) * V;
        if (c < p.C) {
            float w[V], b[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                w[i] = 1.0f;
                b[i] = 0.0f;
            }
            if (p.w) load<W, V>(w, (const W *) p.w + c);
            if (p.b) load<W, V>(b, (const W *) p.b + c);
#pragma unroll
            for (int i = 0; i < V; ++i) v[k][i] = v[k][i] * rstd * w[i] + b[i];
            store<E, V>(y + c, v[k]);
        }
    }
}

// Rows too long for registers: read three times by a workgroup, from HBM once, a value a lane in the order that rows off 16 bytes
// need too, so that both give the same bits. 8,192 rows of 9,000 bf16 values 162 us, 1.8 TB/s of HBM: bound by the loads'
// number.
template <class E, class W>
__global__ __launch_bounds__(256) void layer_norm_long_kernel(norm_p p) {
    __shared__ float lds[4];
    const int64_t row = blockIdx.x;
    const E * x = (const E *) p.x + row * p.x_s;
    E * y = (E *) p.y + row * p.y_s;
    float s = 0.0f;
    for (int c = threadIdx.x; c < p.C; c += 256) s += (float) x[c];
    const float mean = row_sum<256>(s, lds) / (float) p.C;
    s = 0.0f;
    for (int c = threadIdx.x; c < p.C; c += 256) {
        const float d = (float) x[c] - mean;
        s += d * d;
    }
    const float rstd = 1.0f / sqrtf(row_sum<256>(s, lds) / (float) p.C + p.eps);
    if (threadIdx.x == 0) {
        if (p.mean) p.mean[row] = mean;
        if (p.rstd) p.rstd[row] = rstd;
    }
    for (int c = threadIdx.x; c < p.C; c += 256) {
        const float w = p.w ? (float) ((const W *) p.w)[c] : 1.0f, b = p.b ? (float) ((const W *) p.b)[c] : 0.0f;
        y[c] = (E) (((float) x[c] - mean) * rstd * w + b);
    }
}

// Gradients: the rows of a workgroup (every gridDim.x'th group of 256 / TPR) one after another, dw and db of
// its rows in registers, left at the end as one row of `part` each; norm_reduce_kernel sums those. Bound by HBM: 32,900 rows
// of 1,024 bf16 values, 203 MB in 38.5 us, 5.3 TB/s, with 4.2 us of norm_reduce_kernel.
template <class E, class W, int V, int NC, int TPR>
__global__ __launch_bounds__(256) void layer_norm_back_kernel(norm_p p) {
    __shared__ float lds[4];
    const int t = threadIdx.x % TPR;
    float w[NC][V], dw[NC][V], db[NC][V];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        const int c = (k * TPR + t) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            w[k][i] = 1.0f;
            dw[k][i] = db[k][i] = 0.0f;
        }
        if (p.w && c < p.C) load<W, V>(w[k], (const W *) p.w + c);
    }
    const float inv = 1.0f / (float) p.C;
    for (int64_t row = (int64_t) blockIdx.x * (256 / TPR) + threadIdx.x / TPR; row < p.T; row += (int64_t) gridDim.x * (256 / TPR)) {
        const E * x = (const E *) p.x + row * p.x_s, * dy = (const E *) p.dy + row * p.dy_s;
        const float mean = p.mean[row], rstd = p.rstd[row];
        float h[NC][V], g[NC][V], sg = 0.0f, sgh = 0.0f;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            const int c = (k * TPR + t) * V;
            if (c < p.C) {
                load<E, V>(h[k], x + c);
                load<E, V>(g[k], dy + c);
            }
        }
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            if ((k * TPR + t) * V < p.C) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    h[k][i] = (h[k][i] - mean) * rstd;
                    dw[k][i] += g[k][i] * h[k][i];
                    db[k][i] += g[k][i];
                    g[k][i] *= w[k][i];
                    sg += g[k][i];
                    sgh += g[k][i] * h[k][i];
                }
            }
        }
        if (!p.dx) continue;
        sg = row_sum<TPR>(sg, lds) * inv;
        sgh = row_sum<TPR>(sgh, lds) * inv;
        E * dx = (E *) p.dx + row * p.dx_s;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            const int c = (k * TPR + t) * V;
            if (c < p.C) {
#pragma unroll
                for (int i = 0; i < V; ++i) g[k][i] = rstd * (g[k][i] - sg - h[k][i] * sgh);
                store<E, V>(dx + c, g[k]);
            }
        }
    }
    if (!p.part) return;
    extern __shared__ float sums[];        // TPR 64: [2][C], the waves' sums one wave after another
    float * part = p.part + (int64_t) blockIdx.x * 2 * p.C;
    if constexpr (TPR == 256) {
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            const int c = (k * TPR + t) * V;
            if (c < p.C) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    part[c + i] = dw[k][i];
                    part[p.C + c + i] = db[k][i];
                }
            }
        }
    } else {
        for (int turn = 0; turn < 4; ++turn) {
            if ((int) (threadIdx.x >> 6) == turn) {
#pragma unroll
                for (int k = 0; k < NC; ++k) {
                    const int c = (k * TPR + t) * V;
                    if (c < p.C) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            sums[c + i] = turn ? sums[c + i] + dw[k][i] : dw[k][i];
                            sums[p.C + c + i] = turn ? sums[p.C + c + i] + db[k][i] : db[k][i];
                        }
                    }
                }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < 2 * p.C; c += 256) part[c] = sums[c];
    }
}

// Rows too long for registers: dx by a workgroup a row (8,192 rows of 9,000 bf16 values 170 us), and the rows' sums by columns,
// which read the rows once more (88 us, 3.4 TB/s).
template <class E, class W>
__global__ __launch_bounds__(256) void layer_norm_back_long_kernel(norm_p p) {
    __shared__ float lds[4];
    const int64_t row = blockIdx.x;
    const E * x = (const E *) p.x + row * p.x_s, * dy = (const E *) p.dy + row * p.dy_s;
    E * dx = (E *) p.dx + row * p.dx_s;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float sg = 0.0f, sgh = 0.0f;
    for (int c = threadIdx.x; c < p.C; c += 256) {
        const float g = (float) dy[c] * (p.w ? (float) ((const W *) p.w)[c] : 1.0f);
        sg += g;
        sgh += g * (((float) x[c] - mean) * rstd);
    }
    sg = row_sum<256>(sg, lds) / (float) p.C;
    sgh = row_sum<256>(sgh, lds) / (float) p.C;
    for (int c = threadIdx.x; c < p.C; c += 256) {
        const float g = (float) dy[c] * (p.w ? (float) ((const W *) p.w)[c] : 1.0f);
        const float h = ((float) x[c] - mean) * rstd;
        dx[c] = (E) (rstd * (g - sg - h * sgh));
    }
}
template <class E>
__global__ __launch_bounds__(256) void layer_norm_back_columns_kernel(norm_p p) {
    const int c = blockIdx.y * 256 + threadIdx.x;
    if (c >= p.C) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = blockIdx.x; row < p.T; row += gridDim.x) {
        const float g = (float) ((const E *) p.dy)[row * p.dy_s + c];
        dw += g * (((float) ((const E *) p.x)[row * p.x_s + c] - p.mean[row]) * p.rstd[row]);
        db += g;
    }
    float * part = p.part + (int64_t) blockIdx.x * 2 * p.C;
    part[c] = dw;
    part[p.C + c] = db;
}

// The columns' sums of the n_part rows of `part`: 16 columns of dw or db a workgroup, 64 threads each, every 64th row
// a thread (8 loads under way at a time), then the 64 in order.
template <class W>
__global__ __launch_bounds__(1024) void norm_reduce_kernel(norm_p p) {
    __shared__ float lds[64][17];
    const int64_t col = (int64_t) blockIdx.x * 16 + threadIdx.x % 16, n = 2 * (int64_t) p.C;
    const int sub = threadIdx.x / 16;
    float s = 0.0f;
    if (col < n) {
#pragma unroll 8
        for (int r = sub; r < p.n_part; r += 64) s += p.part[r * n + col];
    }
    lds[sub][threadIdx.x % 16] = s;
    __syncthreads();
    if (sub || col >= n) return;
    s = 0.0f;
#pragma unroll 16
    for (int k = 0; k < 64; ++k) s += lds[k][threadIdx.x];
    if (col < p.C) {
        if (p.dw) ((W *) p.dw)[col] = (W) s;
    } else if (p.db) {
        ((W *) p.db)[col - p.C] = (W) s;
    }
}

// ---------------------------------------------------------------------------
// norms of queries and keys, and their rotation
// ---------------------------------------------------------------------------

struct qk_rows {
    const void * x, * dy;
    void * out;                            // y, or dx
    const void * w;
    int64_t x_ts, x_hs, dy_ts, dy_hs, o_ts, o_hs;
    int32_t H;
};
struct qk_p {
    qk_rows of[2];                         // queries, keys
    const double * freq;
    const int32_t * positions, * cu;
    float * part;                          // [workgroups][D], the queries' first
    int32_t T, D, n, n_seqs, tb, lanes;    // tokens of a workgroup at a time, lanes of a head (a power of two)
    int32_t n_q;                           // workgroups of the queries (gradients)
    float mscale, sign, eps;
    int32_t w_type;
    void * dw[2];
};

// Where a head's values lie in its lanes: slot j (lane j % lanes, its j / lanes'th) has V values from d[0] and V from d[1]. A pair that is
// turned is within a slot: values i of both pieces (HALF, and single values), or neighbours in one piece. A piece behind the head's
// end has d = -1; turn: the first angle of the slot, or of the piece, or -1 where nothing is turned.
struct qk_slot {
    int d[2], turn[2];
};
template <int V, bool HALF>
__device__ __forceinline__ qk_slot qk_slot_of(int j, int n, int D) {
    qk_slot s;
    const int half = n / 2;
    if (HALF && j < half / V) {
        s.d[0] = j * V;
        s.d[1] = half + j * V;
        s.turn[0] = s.turn[1] = j * V;
        return s;
    }
    s.d[0] = HALF ? n + 2 * V * (j - half / V) : 2 * V * j;
    s.d[1] = s.d[0] + V;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        s.turn[k] = !HALF && s.d[k] < n ? s.d[k] / 2 : -1;
        if (s.d[k] >= D) s.d[k] = -1;
    }
    return s;
}

// A slot's values turned by the token's turns w.
template <int V, bool HALF>
__device__ __forceinline__ void qk_turn(float (&x)[2][V], const qk_slot & s, const float2 * w) {
    if constexpr (HALF || V == 1) {
        if (s.turn[0] < 0) return;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float c = w[s.turn[0] + i].x, z = w[s.turn[0] + i].y, a = x[0][i], b = x[1][i];
            x[0][i] = a * c - b * z;
            x[1][i] = a * z + b * c;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (s.turn[k] < 0) continue;
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float c = w[s.turn[k] + i].x, z = w[s.turn[k] + i].y, a = x[k][2 * i], b = x[k][2 * i + 1];
                x[k][2 * i] = a * c - b * z;
                x[k][2 * i + 1] = a * z + b * c;
            }
        }
    }
}

// A slot's values as they are in memory, and as fp32.
template <class E, int V> using qk_piece = E __attribute__((ext_vector_type(V == 1 ? 2 : V)));
template <class E, int V>
__device__ __forceinline__ void qk_load(qk_piece<E, V> (&x)[2], const E * row, const qk_slot & s) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        x[k] = qk_piece<E, V>{};
        if (s.d[k] >= 0) {
            if constexpr (V == 1) x[k][0] = row[s.d[k]];
            else x[k] = *reinterpret_cast<const qk_piece<E, V> *>(row + s.d[k]);
        }
    }
}
template <class E, int V>
__device__ __forceinline__ void qk_take(float (&x)[2][V], const qk_piece<E, V> (&from)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) x[k][i] = (float) from[k][i];
}
template <class E, int V>
__device__ __forceinline__ void qk_store(E * row, const float (&x)[2][V], const qk_slot & s) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (s.d[k] >= 0) store<E, V>(row + s.d[k], x[k]);
}

// Sum over the lanes of a head, the same bits in each: neighbours, pairs, fours and eights mirrored, then rows of 16.
__device__ __forceinline__ float head_sum(float x, int lanes) {
    auto add = [](float x, auto ctrl) {
        return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), ctrl(), 0xf, 0xf, false));
    };
    if (lanes > 1) x = add(x, std::integral_constant<int, 0xb1>());
    if (lanes > 2) x = add(x, std::integral_constant<int, 0x4e>());
    if (lanes > 4) x = add(x, std::integral_constant<int, 0x141>());
    if (lanes > 8) x = add(x, std::integral_constant<int, 0x140>());
    if (lanes > 16) x += __shfl_xor(x, 16);
    if (lanes > 32) x += __shfl_xor(x, 32);
    return x;
}

__device__ __forceinline__ float qk_weight(const void * w, int i, int32_t type) {
    if (type == NXG_TYPE_F32) return static_cast<const float *>(w)[i];
    return type == NXG_TYPE_F16 ? (float) static_cast<const _Float16 *>(w)[i] : (float) static_cast<const __bf16 *>(w)[i];
}
// Both weights as fp32 in LDS.
__device__ __forceinline__ void qk_weights(float * w, const qk_p & p) {
    for (int k = threadIdx.x; k < 2 * p.D; k += 256) {
        const void * from = p.of[k / p.D].w;
        w[k] = from ? qk_weight(from, k % p.D, p.w_type) : 0.0f;
    }
}

// The heads of a run of tokens, one after another, `step` apart.
struct qk_walk {
    int t, h, step_t, step_h, heads;
    __device__ __forceinline__ qk_walk(int first, int step, int heads_)
        : t(first / heads_), h(first % heads_), step_t(step / heads_), step_h(step % heads_), heads(heads_) {}
    __device__ __forceinline__ void next() {
        t += step_t;
        h += step_h;
        if (h >= heads) {
            h -= heads;
            ++t;
        }
    }
};

// A workgroup: tb tokens, their turns and the weights once in LDS, then their heads, `lanes` lanes a head, P slots a lane: one
// read, one write. The first heads' rows are under way while the turns are made, each next while one is turned. Bound by HBM: 32
// documents of 32,935 tokens, 24 heads of 64 in bf16, 42 us (4.8 TB/s); 65,536 tokens of 24 heads of 128 in fp16 156 us (5.1 TB/s).
// Loads past the caches are slower here (168 for 158 us), as a head's two halves share lines.
template <class E, int V, bool HALF, int P>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(qk_p p) {
    extern __shared__ float lds[];
    const int half = p.n / 2;
    float * w = lds;                                       // [2][D]
    float2 * turn = reinterpret_cast<float2 *>(lds + 2 * p.D);
    const int64_t t0 = (int64_t) blockIdx.x * p.tb;
    const int tokens = (int) min((int64_t) p.tb, p.T - t0);
    const int lane = threadIdx.x % p.lanes, first = threadIdx.x / p.lanes, step = 256 / p.lanes, heads = p.of[0].H + p.of[1].H;
    qk_slot at[P];
#pragma unroll
    for (int s = 0; s < P; ++s) at[s] = qk_slot_of<V, HALF>(lane + s * p.lanes, p.n, p.D);
    qk_walk u(first, step, heads);
    qk_piece<E, V> raw[P][2];
    auto load = [&](const qk_walk & u) {
        const int key = u.h >= p.of[0].H;
        const qk_rows & r = p.of[key];
        const E * x = static_cast<const E *>(r.x) + (t0 + u.t) * r.x_ts + (u.h - (key ? p.of[0].H : 0)) * r.x_hs;
#pragma unroll
        for (int s = 0; s < P; ++s) qk_load<E, V>(raw[s], x, at[s]);
    };
    if (u.t < tokens) load(u);
    qk_weights(w, p);
    find_turns(turn, p, (int) t0, tokens, half);
    __syncthreads();
    const float inv = 1.0f / (float) p.D;
    while (u.t < tokens) {
        const int t = u.t, key = u.h >= p.of[0].H, h = u.h - (key ? p.of[0].H : 0);
        const qk_rows & r = p.of[key];
        E * o = static_cast<E *>(r.out) + (t0 + t) * r.o_ts + h * r.o_hs;
        float v[P][2][V], ss = 0.0f;
#pragma unroll
        for (int s = 0; s < P; ++s) {
            qk_take<E, V>(v[s], raw[s]);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) ss += v[s][k][i] * v[s][k][i];
        }
        u.next();
        if (u.t < tokens) load(u);
        const float rstd = 1.0f / sqrtf(head_sum(ss, p.lanes) * inv + p.eps);
#pragma unroll
        for (int s = 0; s < P; ++s) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float * wk = w + key * p.D + max(at[s].d[k], 0);
#pragma unroll
                for (int i = 0; i < V; ++i) v[s][k][i] *= rstd * wk[i];
            }
            qk_turn<V, HALF>(v[s], at[s], turn + t * half);
            qk_store<E, V>(o, v[s], at[s]);
        }
    }
}

// Gradients: a workgroup has queries or keys alone, a run of tokens in groups of tb one after another, the weights' sums of
// its heads in registers, left at the end as a row of `part`. The next group's turns are made into the other half of the LDS, so that
// a barrier a group does; the next heads' rows are under way while one head's are worked on. Bound by HBM and the turns' 64-bit
// angles: 32 documents 73 us (4.2 TB/s); queries and keys in one workgroup, with twice the registers, took 147.
template <class E, int V, bool HALF, int P>
__global__ __launch_bounds__(256) void qk_norm_rope_back_kernel(qk_p p) {
    extern __shared__ float lds[];                         // weights [D], turns [2][tb][n / 2]; then sums [256 / lanes][D]
    const int half = p.n / 2, key = (int) blockIdx.x >= p.n_q;
    const int lane = threadIdx.x % p.lanes, first = threadIdx.x / p.lanes, step = 256 / p.lanes;
    const int64_t parts = key ? (int) gridDim.x - p.n_q : p.n_q, part = (int) blockIdx.x - (key ? p.n_q : 0);
    const int64_t end = p.T * (part + 1) / parts;          // of the workgroup's tokens
    int64_t t0 = p.T * part / parts;
    const qk_rows & r = p.of[key];
    qk_slot at[P];
    float dw[P][2][V];
#pragma unroll
    for (int s = 0; s < P; ++s) {
        at[s] = qk_slot_of<V, HALF>(lane + s * p.lanes, p.n, p.D);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) dw[s][k][i] = 0.0f;
    }
    const float inv = 1.0f / (float) p.D;
    auto tokens_of = [&](int64_t t0) { return (int) min((int64_t) p.tb, end - t0); };
    qk_piece<E, V> rx[P][2], rg[P][2];
    auto load = [&](int64_t t0, const qk_walk & u) {
        const E * x = static_cast<const E *>(r.x) + (t0 + u.t) * r.x_ts + u.h * r.x_hs;
        const E * dy = static_cast<const E *>(r.dy) + (t0 + u.t) * r.dy_ts + u.h * r.dy_hs;
#pragma unroll
        for (int s = 0; s < P; ++s) {
            qk_load<E, V>(rx[s], x, at[s]);
            qk_load<E, V>(rg[s], dy, at[s]);
        }
    };
    const qk_walk begin(first, step, r.H);
    float2 * turn = reinterpret_cast<float2 *>(lds + (p.D + 3) / 4 * 4), * other = turn + p.tb * half;
    if (begin.t < tokens_of(t0)) load(t0, begin);
    for (int k = threadIdx.x; k < p.D; k += 256) lds[k] = qk_weight(r.w, k, p.w_type);
    find_turns(turn, p, (int) t0, tokens_of(t0), half);
    for (; t0 < end; t0 += p.tb) {
        const int tokens = tokens_of(t0);
        __syncthreads();
        const bool more = t0 + p.tb < end;
        qk_walk u = begin;
        while (u.t < tokens) {
            E * o = static_cast<E *>(r.out) + (t0 + u.t) * r.o_ts + u.h * r.o_hs;
            const float2 * turns = turn + u.t * half;
            float v[P][2][V], g[P][2][V], ss = 0.0f, gx = 0.0f;
#pragma unroll
            for (int s = 0; s < P; ++s) {
                qk_take<E, V>(v[s], rx[s]);
                qk_take<E, V>(g[s], rg[s]);
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) ss += v[s][k][i] * v[s][k][i];
            }
            u.next();
            if (u.t < tokens) load(t0, u);
            else if (more && begin.t < tokens_of(t0 + p.tb)) load(t0 + p.tb, begin);
            const float rstd = 1.0f / sqrtf(head_sum(ss, p.lanes) * inv + p.eps);
#pragma unroll
            for (int s = 0; s < P; ++s) {
                qk_turn<V, HALF>(g[s], at[s], turns);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float * w = lds + max(at[s].d[k], 0);        // values behind a head's end are zeros
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        v[s][k][i] *= rstd;
                        dw[s][k][i] += g[s][k][i] * v[s][k][i];
                        g[s][k][i] *= w[i];
                        gx += g[s][k][i] * v[s][k][i];
                    }
                }
            }
            gx = head_sum(gx, p.lanes) * inv;
#pragma unroll
            for (int s = 0; s < P; ++s) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) g[s][k][i] = rstd * (g[s][k][i] - v[s][k][i] * gx);
                qk_store<E, V>(o, g[s], at[s]);
            }
        }
        if (more) find_turns(other, p, (int) (t0 + p.tb), tokens_of(t0 + p.tb), half);
        float2 * const swap = turn;
        turn = other;
        other = swap;
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < P; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (at[s].d[k] >= 0) lds[first * p.D + at[s].d[k] + i] = dw[s][k][i];
    __syncthreads();
    for (int c = threadIdx.x; c < p.D; c += 256) {
        float x = 0.0f;
        for (int k = 0; k < step; ++k) x += lds[k * p.D + c];
        p.part[(int64_t) blockIdx.x * p.D + c] = x;
    }
}

// The workgroups' rows of `part` summed up in order: 16 columns of dwq or dwk a workgroup, 64 threads each, every 64th row a thread (8
// loads under way at a time), then the 64 in order.
template <class W>
__global__ __launch_bounds__(1024) void qk_reduce_kernel(qk_p p, int n_all) {
    __shared__ float lds[64][17];
    const int blocks = (p.D + 15) / 16, key = (int) blockIdx.x >= blocks;
    const int col = ((int) blockIdx.x - (key ? blocks : 0)) * 16 + threadIdx.x % 16, sub = threadIdx.x / 16;
    const int r0 = key ? p.n_q : 0, r1 = key ? n_all : p.n_q;
    float s = 0.0f;
    if (col < p.D) {
#pragma unroll 8
        for (int r = r0 + sub; r < r1; r += 64) s += p.part[(int64_t) r * p.D + col];
    }
    lds[sub][threadIdx.x % 16] = s;
    __syncthreads();
    if (sub || col >= p.D) return;
    s = 0.0f;
#pragma unroll 16
    for (int k = 0; k < 64; ++k) s += lds[k][threadIdx.x];
    static_cast<W *>(p.dw[key])[col] = (W) s;
}

// ---------------------------------------------------------------------------
// dropout
// ---------------------------------------------------------------------------

struct dropout_p {
    const void * x, * residual;
    void * out;
    int64_t x_s, r_s, o_s;
    const int64_t * step;
    uint64_t seed, offset;
    int32_t T, C, groups;                  // groups of 8 values of a row
    uint32_t by_groups;                    // 2^32 / groups, rounded up; 0 for 1
    uint32_t least;                        // the least 16 bits that keep a value
    float scale;
};

// Philox 4x32-10: ten rounds of two 32 x 32-bit products on the counter, with a key that goes on by two constants.
__device__ __forceinline__ void philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t a = (uint64_t) c[0] * 0xD2511F53u, b = (uint64_t) c[2] * 0xCD9E8D57u;
        c[0] = (uint32_t) (b >> 32) ^ c[1] ^ k0;
        c[1] = (uint32_t) b;
        c[2] = (uint32_t) (a >> 32) ^ c[3] ^ k1;
        c[3] = (uint32_t) a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

constexpr int DROP_GROUPS = 4;             // of a thread, whose loads are under way together

// A thread: DROP_GROUPS groups of 8 values of a row, 256 apart, of the rows' groups one after another. The mask's bits are made while
// the loads are under way.
// Bound by HBM: 65,536 rows of 2,304 bf16 values 98 us (6.2 TB/s), 32,935 of 1,024 with a residual 34 (5.9 TB/s).
template <class E, bool WIDE>
__global__ __launch_bounds__(256) void dropout_rows_kernel(dropout_p p) {
    constexpr int V = WIDE ? 16 / (int) sizeof(E) : 1, N = 8 / V;
    const uint64_t first = (uint64_t) blockIdx.x * 256 * DROP_GROUPS;
    const uint32_t row0 = (uint32_t) (first / (uint32_t) p.groups), group0 = (uint32_t) (first % (uint32_t) p.groups);
    const uint64_t offset = p.offset + (p.step ? (uint64_t) *p.step : 0);
    const E * x = static_cast<const E *>(p.x), * residual = static_cast<const E *>(p.residual);
    E * out = static_cast<E *>(p.out);
    float v[DROP_GROUPS][N][V], r[DROP_GROUPS][N][V];
    uint32_t row[DROP_GROUPS], group[DROP_GROUPS];
#pragma unroll
    for (int k = 0; k < DROP_GROUPS; ++k) {
        // groups behind the first of row0: below 2^11 past a row's, or past one row at most
        const uint32_t at = group0 + threadIdx.x + 256 * k, groups = p.groups;
        const uint32_t rows = groups >= 256 * DROP_GROUPS ? at >= groups : p.by_groups ? __umulhi(at, p.by_groups) : at;
        row[k] = row0 + rows;
        group[k] = at - rows * groups;
        const bool some = row[k] < (uint32_t) p.T;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int c = 8 * (int) group[k] + j * V;
#pragma unroll
            for (int i = 0; i < V; ++i) v[k][j][i] = r[k][j][i] = 0.0f;
            if (some && c < p.C) {
                load_once<E, V>(v[k][j], x + (int64_t) row[k] * p.x_s + c);
                if (residual) load_once<E, V>(r[k][j], residual + (int64_t) row[k] * p.r_s + c);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < DROP_GROUPS; ++k) {
        uint32_t bits[4] = {group[k], row[k], (uint32_t) offset, (uint32_t) (offset >> 32)};
        philox(bits, (uint32_t) p.seed, (uint32_t) (p.seed >> 32));
        if (row[k] >= (uint32_t) p.T) continue;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int c = 8 * (int) group[k] + j * V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int e = j * V + i;
                const uint32_t u = bits[e / 2] >> (16 * (e % 2)) & 0xffffu;
                v[k][j][i] = (u >= p.least ? v[k][j][i] * p.scale : 0.0f) + r[k][j][i];
            }
            if (c < p.C) store_once<E, V>(out + (int64_t) row[k] * p.o_s + c, v[k][j]);
        }
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

#define NXG_TRY(call) do { const int32_t rc_ = (call); if (rc_) return rc_; } while (0)

int size_of(int32_t type) { return type == NXG_TYPE_F32 ? 4 : type == NXG_TYPE_F16 || type == NXG_TYPE_BF16 ? 2 : 0; }

template <class F>
void by_type(int32_t type, F f) {
    if (type == NXG_TYPE_F32) f(float());
    else if (type == NXG_TYPE_F16) f((_Float16) 0.0f);
    else f((__bf16) 0.0f);
}
template <class F>
void by_types(int32_t type, int32_t w_type, F f) {
    by_type(type, [&](auto e) {
        if (w_type == NXG_TYPE_F32) f(e, float());
        else f(e, e);
    });
}

constexpr int NORM_PARTS = 512;        // workgroups of the gradients' kernels: two a CU

// 16 bytes at a time where every row allows it.
bool wide(const void * p, int64_t stride, int es) { return ((uintptr_t) p & 15) == 0 && stride * es % 16 == 0; }
bool aligned(const void * p, int es) { return ((uintptr_t) p & (es - 1)) == 0; }

constexpr int MAX_GRID = (1 << 24) - 1;        // workgroups of a launch: less than 2^32 threads
constexpr int MAX_C = 1 << 23;
int32_t check_norm(const char * what, int32_t type, int32_t w_type, int32_t T, int32_t C) {
    if (!size_of(type)) return nxg_fail(NXG_EINVAL, "%s: type %d (F32, F16 or BF16)", what, type);
    if (w_type != type && w_type != NXG_TYPE_F32) return nxg_fail(NXG_EINVAL, "%s: weight type %d (the rows' or F32)", what, w_type);
    if (T < 0 || C < 1) return nxg_fail(NXG_EINVAL, "%s: T=%d C=%d", what, T, C);
    if (C > MAX_C || T > (C <= 1024 ? 4 : 1) * MAX_GRID) return nxg_fail(NXG_EINVAL, "%s: T=%d C=%d is too large", what, T, C);
    return NXG_OK;
}
int32_t check_norm_rows(const char * what, const char * name, const void * p, int64_t stride, int32_t T, int32_t C, int es, bool written) {
    if (!p || !aligned(p, es)) return nxg_fail(NXG_EINVAL, "%s: %s is null or not aligned to its type", what, name);
    if (T > 1 && (stride < (written ? C : 0) || stride > INT64_MAX / 16 / T)) {
        return nxg_fail(NXG_EINVAL, "%s: stride %lld of %s for rows of %d", what, (long long) stride, name, C);
    }
    return NXG_OK;
}

template <int N> using num = std::integral_constant<int, N>;

// The instance for rows of C values: f(V, NC, TPR) as compile-time numbers; false where a row does not fit
// registers. A wave a row where its lanes hold it (32 values a lane), else the workgroup.
template <class F>
bool by_row(int C, int es, bool wide, F f) {
    if (wide) {
        const int V = 16 / es;
        if (es == 2) {
            if (C <= 64 * V) f(num<8>(), num<1>(), num<64>());
            else if (C <= 64 * V * 2) f(num<8>(), num<2>(), num<64>());
            else if (C <= 64 * V * 4) f(num<8>(), num<4>(), num<64>());
            else if (C <= 256 * V * 2) f(num<8>(), num<2>(), num<256>());
            else if (C <= 256 * V * 4) f(num<8>(), num<4>(), num<256>());
            else return false;
        } else {
            if (C <= 64 * V * 2) f(num<4>(), num<2>(), num<64>());
            else if (C <= 64 * V * 4) f(num<4>(), num<4>(), num<64>());
            else if (C <= 64 * V * 8) f(num<4>(), num<8>(), num<64>());
            else if (C <= 256 * V * 4) f(num<4>(), num<4>(), num<256>());
            else if (C <= 256 * V * 8) f(num<4>(), num<8>(), num<256>());
            else return false;
        }
        return true;
    }
    if (C <= 64 * 4) f(num<1>(), num<4>(), num<64>());
    else if (C <= 64 * 16) f(num<1>(), num<16>(), num<64>());
    else if (C <= 256 * 16) f(num<1>(), num<16>(), num<256>());
    else if (C <= 256 * 32) f(num<1>(), num<32>(), num<256>());
    else return false;
    return true;
}

int norm_parts(int32_t T, int32_t C) {
    const int rows = C <= 1024 ? 4 : 1;          // of a workgroup at a time, at least
    return (int) std::max<int64_t>(1, std::min<int64_t>(NORM_PARTS, ((int64_t) T + rows - 1) / rows));
}

// Strides of rows of n_head heads that one call may read; of an output's, that no two of its rows overlap.
int32_t check_heads(const char * what, const char * name, const nxg_rows * r, int32_t T, int32_t n_head, int32_t D, int es, bool written) {
    if (!r || !r->data) return nxg_fail(NXG_EINVAL, "%s: %s is null", what, name);
    const int64_t most = INT64_MAX / 16, ts = T > 1 ? r->token_stride : 0, hs = n_head > 1 ? r->head_stride : 0;
    if (!aligned(r->data, es) || ts < 0 || hs < 0 || ts > most / T || hs > most / n_head) {
        return nxg_fail(NXG_EINVAL, "%s: %s is not aligned to its type, or has strides %lld, %lld", what, name, (long long) ts, (long long) hs);
    }
    if (written) {
        const bool heads_in = hs <= ts || T == 1;
        const int64_t in_n = heads_in ? n_head : T, in_s = heads_in ? hs : ts, out_n = heads_in ? T : n_head, out_s = heads_in ? ts : hs;
        if ((in_n > 1 && in_s < D) || (out_n > 1 && out_s < (in_n - 1) * in_s + D)) {
            return nxg_fail(NXG_EINVAL, "%s: rows of %s overlap (strides %lld, %lld)", what, name, (long long) ts, (long long) hs);
        }
    }
    return NXG_OK;
}

int32_t check_qk(const char * what, const nxg_qk_norm_rope_params * p) {
    if (!p) return nxg_fail(NXG_EINVAL, "%s: null params", what);
    if (!size_of(p->type)) return nxg_fail(NXG_EINVAL, "%s: type %d (F32, F16 or BF16)", what, p->type);
    if (p->w_type != p->type && p->w_type != NXG_TYPE_F32) return nxg_fail(NXG_EINVAL, "%s: weight type %d (the rows' or F32)", what, p->w_type);
    if (p->T < 0 || p->n_head < 1 || p->n_kv_head < 0 || p->head_dim < 2 || p->head_dim > 1024 || p->n_head > 65536 || p->n_kv_head > 65536) {
        return nxg_fail(NXG_EINVAL, "%s: T=%d n_head=%d n_kv_head=%d head_dim=%d", what, p->T, p->n_head, p->n_kv_head, p->head_dim);
    }
    if (!(p->eps >= 0.0f) || !std::isfinite(p->eps)) return nxg_fail(NXG_EINVAL, "%s: eps=%g", what, p->eps);
    if (p->n_rot < 2 || p->n_rot % 2 || p->n_rot > p->head_dim) return nxg_fail(NXG_EINVAL, "%s: n_rot=%d of head_dim=%d", what, p->n_rot, p->head_dim);
    if (p->layout != NXG_ROPE_HALF && p->layout != NXG_ROPE_INTERLEAVED) return nxg_fail(NXG_EINVAL, "%s: layout %d", what, p->layout);
    return NXG_OK;
}

// The rows of one operand pair (queries, or keys) into p, checked. out: y, or dx.
int32_t take_qk(const char * what, const nxg_qk_norm_rope_params & a, qk_rows & r, bool keys, const nxg_rows * x, const nxg_rows * dy,
                const nxg_rows * out, bool back) {
    const int es = size_of(a.type);
    const char * x_name = keys ? "k" : "q", * dy_name = keys ? "dk_out" : "dq_out", * out_name = back ? (keys ? "dk" : "dq") : keys ? "k_out" : "q_out";
    r.H = keys ? a.n_kv_head : a.n_head;
    r.w = keys ? a.wk : a.wq;
    if (!r.w || !aligned(r.w, size_of(a.w_type))) return nxg_fail(NXG_EINVAL, "%s: %s is null or not aligned to its type", what, keys ? "wk" : "wq");
    NXG_TRY(check_heads(what, x_name, x, a.T, r.H, a.head_dim, es, false));
    if (back) NXG_TRY(check_heads(what, dy_name, dy, a.T, r.H, a.head_dim, es, false));
    NXG_TRY(check_heads(what, out_name, out, a.T, r.H, a.head_dim, es, true));
    auto ts = [&](const nxg_rows * v) { return a.T > 1 ? v->token_stride : 0; };
    auto hs = [&](const nxg_rows * v) { return r.H > 1 ? v->head_stride : 0; };
    for (const nxg_rows * v : {x, back ? dy : x}) {
        if (v->data == out->data && (ts(v) != ts(out) || hs(v) != hs(out))) {
            return nxg_fail(NXG_EINVAL, "%s: %s is an input with other strides", what, out_name);
        }
    }
    r.x = x->data;
    r.x_ts = ts(x);
    r.x_hs = hs(x);
    r.dy = back ? dy->data : nullptr;
    r.dy_ts = back ? ts(dy) : 0;
    r.dy_hs = back ? hs(dy) : 0;
    r.out = out->data;
    r.o_ts = ts(out);
    r.o_hs = hs(out);
    return NXG_OK;
}

constexpr int QK_PARTS = 768;          // workgroups of the gradients' kernel: three a CU, as many as its registers leave at once (1,024: 88 us for 73)

// Both directions' plan: tokens of a workgroup, lanes of a head, and the instance f(V, HALF, P).
struct qk_plan {
    bool wide;
    int slots, per_lane;
    size_t lds;
};
qk_plan plan_qk(const nxg_qk_norm_rope_params & a, qk_p & p, bool back) {
    qk_plan l;
    const int es = size_of(a.type), V = 16 / es;
    l.wide = a.n_rot % (a.layout == NXG_ROPE_HALF ? 2 * V : V) == 0 && a.head_dim % V == 0;
    for (const qk_rows & r : p.of) {
        if (r.H == 0) continue;
        l.wide = l.wide && wide(r.x, r.x_ts, es) && wide(r.x, r.x_hs, es) && wide(r.out, r.o_ts, es) && wide(r.out, r.o_hs, es) &&
                 wide(r.dy, r.dy_ts, es) && wide(r.dy, r.dy_hs, es);
    }
    const int v = l.wide ? V : 1;
    l.slots = a.layout == NXG_ROPE_HALF ? a.n_rot / 2 / v + (a.head_dim - a.n_rot + 2 * v - 1) / (2 * v) : (a.head_dim + 2 * v - 1) / (2 * v);
    p.lanes = 1;
    while (p.lanes < 64 && p.lanes < l.slots) p.lanes *= 2;
    l.per_lane = (l.slots + p.lanes - 1) / p.lanes;
    // tokens: about 24 KiB of rows and an angle a thread, so that the heads fill a few whole rounds of the workgroup (16 and 8 heads of 64
    // bf16 values: 3); gradients, whose workgroups stay, two angles a thread. Fewer where that would leave CUs without work
    const int64_t row = (int64_t) (a.n_head + a.n_kv_head) * a.head_dim * es;
    p.tb = std::max<int>(1, back ? std::min<int64_t>(1024 / a.n_rot, 65536 / row) : std::min<int64_t>(512 / a.n_rot, 24576 / row));
    while (p.tb > 1 && ((int64_t) a.T + p.tb - 1) / p.tb < (back ? QK_PARTS : 2 * nxg_device_cus())) p.tb /= 2;
    const size_t turns = (size_t) p.tb * (a.n_rot / 2) * sizeof(float2);
    l.lds = back ? std::max<size_t>((a.head_dim + 3) / 4 * 4 * sizeof(float) + 2 * turns, (size_t) (256 / p.lanes) * a.head_dim * sizeof(float)) : 2 * a.head_dim * sizeof(float) + turns;
    p.freq = a.freq;
    p.positions = a.positions;
    p.cu = a.cu;
    p.n_seqs = a.n_seqs;
    p.T = a.T;
    p.D = a.head_dim;
    p.n = a.n_rot;
    p.eps = a.eps;
    p.mscale = a.mscale;
    p.w_type = a.w_type;
    return l;
}
// A lane has one slot of 16-byte pieces, or two of fp32 heads over 512 values; up to 8 of single values.
template <class F>
void by_qk(const nxg_qk_norm_rope_params & a, const qk_plan & l, F f) {
    by_type(a.type, [&](auto e) {
        constexpr int V = 16 / (int) sizeof(e);
        auto by_lane = [&](auto half) {
            if (l.wide) {
                if constexpr (V == 4) {
                    if (l.per_lane > 1) return f(e, num<V>(), half, num<2>());
                }
                f(e, num<V>(), half, num<1>());
            } else if (l.per_lane <= 1) {
                f(e, num<1>(), half, num<1>());
            } else {
                f(e, num<1>(), half, num<8>());
            }
        };
        if (a.layout == NXG_ROPE_HALF) by_lane(std::true_type());
        else by_lane(std::false_type());
    });
}

int32_t check_positions(const char * what, const nxg_qk_norm_rope_params & a) {
    if (!a.freq || (!a.positions && !a.cu)) return nxg_fail(NXG_EINVAL, "%s: null freq, or neither positions nor cu", what);
    if (!a.positions && a.n_seqs < 1) return nxg_fail(NXG_EINVAL, "%s: n_seqs=%d", what, a.n_seqs);
    return NXG_OK;
}

} // namespace

extern "C" {

int32_t nxg_rope_frequencies(int32_t n_rot, double base, int32_t scaling, double factor, int32_t train_len, double * freq,
                             float * mscale) {
    const char * what = "rope_frequencies";
    if (n_rot < 2 || n_rot % 2 || !(base > 0.0) || !std::isfinite(base)) return nxg_fail(NXG_EINVAL, "%s: n_rot=%d base=%g", what, n_rot, base);
    if (scaling < NXG_ROPE_NONE || scaling > NXG_ROPE_BY_PARTS) return nxg_fail(NXG_EINVAL, "%s: scaling %d", what, scaling);
    if (scaling != NXG_ROPE_NONE && (!(factor >= 1.0) || !std::isfinite(factor))) return nxg_fail(NXG_EINVAL, "%s: factor=%g (at least 1)", what, factor);
    if (scaling == NXG_ROPE_NTK && n_rot <= 2) return nxg_fail(NXG_EINVAL, "%s: n_rot=%d (more than 2 for NTK)", what, n_rot);
    if (scaling == NXG_ROPE_BY_PARTS && train_len < 1) return nxg_fail(NXG_EINVAL, "%s: train_len=%d", what, train_len);
    if (!freq || !mscale) return nxg_fail(NXG_EINVAL, "%s: null output", what);
    const double pi2 = 6.283185307179586476925;
    if (scaling == NXG_ROPE_NTK) base *= std::pow(factor, n_rot / (n_rot - 2.0));
    *mscale = scaling == NXG_ROPE_BY_PARTS ? (float) (0.1 * std::log(factor) + 1.0) : 1.0f;
    for (int i = 0; i < n_rot / 2; ++i) {
        double f = std::pow(base, -2.0 * i / n_rot);
        if (scaling == NXG_ROPE_LINEAR) f /= factor;
        if (scaling == NXG_ROPE_BY_PARTS) {
            const double turns = train_len * f / pi2, keep = std::min(std::max((turns - 1.0) / 31.0, 0.0), 1.0);
            f = (1.0 - keep) * f / factor + keep * f;
        }
        freq[i] = f;
    }
    return NXG_OK;
}

int32_t nxg_rope_rows(int32_t type, const nxg_rows * x, int32_t T, int32_t n_head, int32_t head_dim, const double * freq,
                      int32_t n_rot, int32_t layout, float mscale, int32_t inverse, const int32_t * positions,
                      const int32_t * cu, int32_t n_seqs, const nxg_rows * out, void * stream) {
    const char * what = "rope_rows";
    const int es = size_of(type);
    if (!es) return nxg_fail(NXG_EINVAL, "%s: type %d (F32, F16 or BF16)", what, type);
    if (T < 0 || n_head < 1 || head_dim < 2 || head_dim > 1024) return nxg_fail(NXG_EINVAL, "%s: T=%d n_head=%d head_dim=%d", what, T, n_head, head_dim);
    if (n_rot < 2 || n_rot % 2 || n_rot > head_dim) return nxg_fail(NXG_EINVAL, "%s: n_rot=%d of head_dim=%d", what, n_rot, head_dim);
    if (layout != NXG_ROPE_HALF && layout != NXG_ROPE_INTERLEAVED) return nxg_fail(NXG_EINVAL, "%s: layout %d", what, layout);
    if (T == 0) return NXG_OK;
    if (!x || !x->data || !out || !out->data || !freq || (!positions && !cu)) return nxg_fail(NXG_EINVAL, "%s: null buffer", what);
    if (!positions && n_seqs < 1) return nxg_fail(NXG_EINVAL, "%s: n_seqs=%d", what, n_seqs);
    const int64_t most = INT64_MAX / 16;
    for (const nxg_rows * r : {x, out}) {
        const int64_t ts = T > 1 ? r->token_stride : 0, hs = n_head > 1 ? r->head_stride : 0;
        if (!aligned(r->data, es) || ts < 0 || hs < 0 || ts > most / T || hs > most / n_head) {
            return nxg_fail(NXG_EINVAL, "%s: rows not aligned to their type, or strides %lld, %lld", what, (long long) ts, (long long) hs);
        }
        if (r == out) {                  // no two rows of the output overlap
            const bool heads_in = hs <= ts || T == 1;
            const int64_t in_n = heads_in ? n_head : T, in_s = heads_in ? hs : ts, out_n = heads_in ? T : n_head, out_s = heads_in ? ts : hs;
            if ((in_n > 1 && in_s < head_dim) || (out_n > 1 && out_s < (in_n - 1) * in_s + head_dim)) {
                return nxg_fail(NXG_EINVAL, "%s: rows of out overlap (strides %lld, %lld)", what, (long long) ts, (long long) hs);
            }
        }
    }
    rope_p p;
    p.x = x->data;
    p.out = out->data;
    p.x_ts = T > 1 ? x->token_stride : 0;
    p.x_hs = n_head > 1 ? x->head_stride : 0;
    p.o_ts = T > 1 ? out->token_stride : 0;
    p.o_hs = n_head > 1 ? out->head_stride : 0;
    if (p.x == p.out && (p.x_ts != p.o_ts || p.x_hs != p.o_hs)) return nxg_fail(NXG_EINVAL, "%s: out is x with other strides", what);
    p.copy = p.x != p.out;
    p.freq = freq;
    p.positions = positions;
    p.cu = cu;
    p.T = T;
    p.H = n_head;
    p.D = head_dim;
    p.n = n_rot;
    p.n_seqs = n_seqs;
    p.mscale = mscale;
    p.sign = inverse ? -1.0f : 1.0f;
    const int V = 16 / es;
    const bool w = wide(p.x, p.x_ts, es) && wide(p.x, p.x_hs, es) && wide(p.out, p.o_ts, es) && wide(p.out, p.o_hs, es) &&
                   n_rot % (layout == NXG_ROPE_HALF ? 2 * V : V) == 0 && head_dim % V == 0;
    // tokens of a workgroup: at most an angle a thread, and about 12 KiB of rows (65,536 x 24 heads of 64: fp32 152 us
    // with 12 KiB, 160 with 98; bf16 75 with 12, 80 with 24, 82 with 3), fewer where that would leave CUs without
    // work; heads in pieces too for the shortest
    const int cus = nxg_device_cus();
    p.tb = std::max<int>(1, std::min<int64_t>(512 / n_rot, 12288 / ((int64_t) n_head * head_dim * es)));
    while (p.tb > 1 && ((int64_t) T + p.tb - 1) / p.tb < 2 * cus) p.tb /= 2;
    p.hb = n_head;
    while (p.hb > 1 && ((int64_t) T + p.tb - 1) / p.tb * ((n_head + p.hb - 1) / p.hb) < cus && p.hb * head_dim > 256 * (w ? V : 1)) p.hb = (p.hb + 1) / 2;
    const int v = w ? V : 1, per_head = (layout == NXG_ROPE_HALF || v == 1 ? n_rot / 2 / v : n_rot / v) + (p.copy ? (head_dim - n_rot) / v : 0);
    if (per_head == 0) return NXG_OK;
    p.hb = std::min(p.hb, 65535 / per_head);
    while (p.tb > 1 && (int64_t) p.tb * p.hb * per_head * p.hb * per_head > INT32_MAX) p.tb /= 2;
    auto magic = [](int d) { return (uint32_t) (((1ull << 32) + d - 1) / d); };       // 0 for 1
    p.by_head = magic(per_head);
    p.by_token = magic(per_head * p.hb);
    p.by_token_last = magic(per_head * ((n_head - 1) % p.hb + 1));
    const dim3 grid((unsigned) (((int64_t) T + p.tb - 1) / p.tb), (unsigned) (((int64_t) n_head + p.hb - 1) / p.hb));
    if (grid.y > 65535 || (int64_t) grid.x * grid.y > MAX_GRID) {
        return nxg_fail(NXG_EINVAL, "%s: T=%d n_head=%d is too large", what, T, n_head);
    }
    NXG_TRY(nxg_check_device());
    const size_t lds = (size_t) p.tb * (n_rot / 2) * sizeof(float2);
    hipStream_t s = (hipStream_t) stream;
    by_type(type, [&](auto e) {
        typedef decltype(e) E;
        constexpr int VE = 16 / (int) sizeof(E);
        if (layout == NXG_ROPE_HALF) {
            if (w) rope_rows_kernel<E, VE, true><<<grid, 256, lds, s>>>(p);
            else rope_rows_kernel<E, 1, true><<<grid, 256, lds, s>>>(p);
        } else {
            if (w) rope_rows_kernel<E, VE, false><<<grid, 256, lds, s>>>(p);
            else rope_rows_kernel<E, 1, false><<<grid, 256, lds, s>>>(p);
        }
    });
    return nxg_launch_check(what);
}

int32_t nxg_layer_norm_rows(int32_t type, const void * x, int64_t x_stride, const void * w, const void * b, int32_t w_type,
                            float eps, int32_t T, int32_t C, void * y, int64_t y_stride, float * mean, float * rstd, void * stream) {
    const char * what = "layer_norm_rows";
    NXG_TRY(check_norm(what, type, w_type, T, C));
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return nxg_fail(NXG_EINVAL, "%s: eps=%g", what, eps);
    if (T == 0) return NXG_OK;
    const int es = size_of(type), ws = size_of(w_type);
    NXG_TRY(check_norm_rows(what, "x", x, x_stride, T, C, es, false));
    NXG_TRY(check_norm_rows(what, "y", y, y_stride, T, C, es, true));
    if ((w && !aligned(w, ws)) || (b && !aligned(b, ws))) return nxg_fail(NXG_EINVAL, "%s: w or b is not aligned to its type", what);
    if (x == y && T > 1 && x_stride != y_stride) return nxg_fail(NXG_EINVAL, "%s: y is x with another stride", what);
    NXG_TRY(nxg_check_device());
    norm_p p = {};
    p.x = x;
    p.w = w;
    p.b = b;
    p.y = y;
    p.mean = mean;
    p.rstd = rstd;
    p.x_s = T > 1 ? x_stride : 0;
    p.y_s = T > 1 ? y_stride : 0;
    p.T = T;
    p.C = C;
    p.eps = eps;
    const bool v = wide(x, p.x_s, es) && wide(y, p.y_s, es) && (!w || wide(w, 0, ws)) && (!b || wide(b, 0, ws)) && C % (16 / es) == 0;
    hipStream_t s = (hipStream_t) stream;
    by_types(type, w_type, [&](auto e, auto we) {
        typedef decltype(e) E;
        typedef decltype(we) W;
        const bool done = by_row(C, es, v, [&](auto V, auto NC, auto TPR) {
            if constexpr (V() == 1 || V() == 16 / (int) sizeof(E)) {
                const unsigned grid = (unsigned) (((int64_t) T + 256 / TPR() - 1) / (256 / TPR()));
                layer_norm_rows_kernel<E, W, V(), NC(), TPR()><<<grid, 256, 0, s>>>(p);
            }
        });
        if (!done) layer_norm_long_kernel<E, W><<<(unsigned) T, 256, 0, s>>>(p);
    });
    return nxg_launch_check(what);
}

int64_t nxg_layer_norm_rows_workspace_bytes(int32_t T, int32_t C) {
    const int32_t rc = check_norm("layer_norm_rows_workspace_bytes", NXG_TYPE_F32, NXG_TYPE_F32, T, C);
    if (rc) return -rc;
    return (int64_t) norm_parts(T, C) * 2 * C * 4;
}

int32_t nxg_layer_norm_rows_backward(int32_t type, const void * dy, int64_t dy_stride, const void * x, int64_t x_stride,
                                     const float * mean, const float * rstd, const void * w, int32_t w_type, int32_t T,
                                     int32_t C, void * dx, int64_t dx_stride, void * dw, void * db, void * workspace,
                                     int64_t workspace_bytes, void * stream) {
    const char * what = "layer_norm_rows_backward";
    NXG_TRY(check_norm(what, type, w_type, T, C));
    const int es = size_of(type), ws = size_of(w_type);
    if ((w && !aligned(w, ws)) || (dw && !aligned(dw, ws)) || (db && !aligned(db, ws))) {
        return nxg_fail(NXG_EINVAL, "%s: w, dw or db is not aligned to its type", what);
    }
    if (!dx && !dw && !db) return NXG_OK;
    if (T > 0) {
        NXG_TRY(check_norm_rows(what, "dy", dy, dy_stride, T, C, es, false));
        NXG_TRY(check_norm_rows(what, "x", x, x_stride, T, C, es, false));
        if (dx) NXG_TRY(check_norm_rows(what, "dx", dx, dx_stride, T, C, es, true));
        if (!mean || !rstd) return nxg_fail(NXG_EINVAL, "%s: null mean or rstd", what);
        if (dx && T > 1 && ((dx == dy && dx_stride != dy_stride) || (dx == x && dx_stride != x_stride))) {
            return nxg_fail(NXG_EINVAL, "%s: dx is dy or x with another stride", what);
        }
    }
    norm_p p = {};
    p.n_part = T > 0 ? norm_parts(T, C) : 0;
    if (dw || db) {
        if (!workspace || ((uintptr_t) workspace & 15) || workspace_bytes < (int64_t) p.n_part * 2 * C * 4) {
            return nxg_fail(NXG_EINVAL, "%s: workspace must be 16-byte aligned memory of %lld bytes", what,
                            (long long) nxg_layer_norm_rows_workspace_bytes(T, C));
        }
        p.part = (float *) workspace;
    } else if (T == 0) {
        return NXG_OK;
    }
    NXG_TRY(nxg_check_device());
    p.x = x;
    p.dy = dy;
    p.w = w;
    p.dx = dx;
    p.dw = dw;
    p.db = db;
    p.mean = (float *) mean;
    p.rstd = (float *) rstd;
    p.x_s = T > 1 ? x_stride : 0;
    p.dy_s = T > 1 ? dy_stride : 0;
    p.dx_s = T > 1 ? dx_stride : 0;
    p.T = T;
    p.C = C;
    hipStream_t s = (hipStream_t) stream;
    if (T > 0) {
        const bool v = wide(x, p.x_s, es) && wide(dy, p.dy_s, es) && (!dx || wide(dx, p.dx_s, es)) && (!w || wide(w, 0, ws)) && C % (16 / es) == 0;
        by_types(type, w_type, [&](auto e, auto we) {
            typedef decltype(e) E;
            typedef decltype(we) W;
            const bool done = by_row(C, es, v, [&](auto V, auto NC, auto TPR) {
                if constexpr (V() == 1 || V() == 16 / (int) sizeof(E)) {
                    const size_t lds = TPR() == 64 && p.part ? (size_t) 2 * C * sizeof(float) : 0;
                    layer_norm_back_kernel<E, W, V(), NC(), TPR()><<<(unsigned) p.n_part, 256, lds, s>>>(p);
                }
            });
            if (done) return;
            // the columns first: dx may be dy or x
            if (p.part) {
                layer_norm_back_columns_kernel<E><<<dim3((unsigned) p.n_part, (unsigned) ((C + 255) / 256)), 256, 0, s>>>(p);
            }
            if (dx) layer_norm_back_long_kernel<E, W><<<(unsigned) T, 256, 0, s>>>(p);
        });
        NXG_TRY(nxg_launch_check(what));
    }
    if (!p.part) return NXG_OK;
    const unsigned grid = (unsigned) ((2 * (int64_t) C + 15) / 16);
    by_types(type, w_type, [&](auto, auto we) { norm_reduce_kernel<decltype(we)><<<grid, 1024, 0, s>>>(p); });
    return nxg_launch_check(what);
}

int32_t nxg_qk_norm_rope_rows(const nxg_qk_norm_rope_params * params, const nxg_rows * q, const nxg_rows * k, const nxg_rows * q_out,
                              const nxg_rows * k_out, void * stream) {
    const char * what = "qk_norm_rope_rows";
    NXG_TRY(check_qk(what, params));
    const nxg_qk_norm_rope_params & a = *params;
    if (a.T == 0) return NXG_OK;
    NXG_TRY(check_positions(what, a));
    qk_p p = {};
    NXG_TRY(take_qk(what, a, p.of[0], false, q, nullptr, q_out, false));
    if (a.n_kv_head) {
        NXG_TRY(take_qk(what, a, p.of[1], true, k, nullptr, k_out, false));
        if (q_out->data == k_out->data || q_out->data == k->data || k_out->data == q->data) {
            return nxg_fail(NXG_EINVAL, "%s: an output is another tensor of the call", what);
        }
    }
    const qk_plan l = plan_qk(a, p, false);
    p.sign = 1.0f;
    const int64_t grid = ((int64_t) a.T + p.tb - 1) / p.tb;
    if (grid > MAX_GRID) return nxg_fail(NXG_EINVAL, "%s: T=%d is too large", what, a.T);
    NXG_TRY(nxg_check_device());
    by_qk(a, l, [&](auto e, auto V, auto half, auto P) {
        qk_norm_rope_kernel<decltype(e), V(), half(), P()><<<(unsigned) grid, 256, l.lds, (hipStream_t) stream>>>(p);
    });
    return nxg_launch_check(what);
}

int64_t nxg_qk_norm_rope_rows_workspace_bytes(const nxg_qk_norm_rope_params * params) {
    const int32_t rc = check_qk("qk_norm_rope_rows_workspace_bytes", params);
    return rc ? -rc : (int64_t) QK_PARTS * params->head_dim * 4;
}

int32_t nxg_qk_norm_rope_rows_backward(const nxg_qk_norm_rope_params * params, const nxg_rows * dq_out, const nxg_rows * dk_out,
                                       const nxg_rows * q, const nxg_rows * k, const nxg_rows * dq, const nxg_rows * dk, void * dwq,
                                       void * dwk, void * workspace, int64_t workspace_bytes, void * stream) {
    const char * what = "qk_norm_rope_rows_backward";
    NXG_TRY(check_qk(what, params));
    const nxg_qk_norm_rope_params & a = *params;
    const int ws = size_of(a.w_type);
    if (!dwq || !aligned(dwq, ws) || (a.n_kv_head && (!dwk || !aligned(dwk, ws)))) {
        return nxg_fail(NXG_EINVAL, "%s: dwq or dwk is null or not aligned to its type", what);
    }
    if (!workspace || ((uintptr_t) workspace & 15) || workspace_bytes < (int64_t) QK_PARTS * a.head_dim * 4) {
        return nxg_fail(NXG_EINVAL, "%s: workspace must be 16-byte aligned memory of %lld bytes", what,
                        (long long) nxg_qk_norm_rope_rows_workspace_bytes(params));
    }
    qk_p p = {};
    int64_t grid = 0;
    hipStream_t s = (hipStream_t) stream;
    if (a.T > 0) {
        NXG_TRY(check_positions(what, a));
        NXG_TRY(take_qk(what, a, p.of[0], false, q, dq_out, dq, true));
        if (a.n_kv_head) {
            NXG_TRY(take_qk(what, a, p.of[1], true, k, dk_out, dk, true));
            for (const nxg_rows * o : {dq, dk}) {
                const nxg_rows * other[] = {o == dq ? k : q, o == dq ? dk_out : dq_out, o == dq ? dk : dq};
                for (const nxg_rows * r : other)
                    if (o->data == r->data) return nxg_fail(NXG_EINVAL, "%s: an output is another tensor of the call", what);
            }
        }
        const qk_plan l = plan_qk(a, p, true);
        p.sign = -1.0f;
        p.part = static_cast<float *>(workspace);
        // workgroups shared out by the heads
        const int64_t groups = ((int64_t) a.T + p.tb - 1) / p.tb;
        p.n_q = (int32_t) std::min<int64_t>(groups, std::max<int64_t>(1, (int64_t) QK_PARTS * a.n_head / (a.n_head + a.n_kv_head)));
        if (a.n_kv_head) p.n_q = std::min(p.n_q, QK_PARTS - 1);
        grid = p.n_q + (a.n_kv_head ? std::min<int64_t>(groups, QK_PARTS - p.n_q) : 0);
        NXG_TRY(nxg_check_device());
        by_qk(a, l, [&](auto e, auto V, auto half, auto P) {
            qk_norm_rope_back_kernel<decltype(e), V(), half(), P()><<<(unsigned) grid, 256, l.lds, s>>>(p);
        });
        NXG_TRY(nxg_launch_check(what));
    } else {
        NXG_TRY(nxg_check_device());
    }
    p.part = static_cast<float *>(workspace);
    p.D = a.head_dim;
    p.dw[0] = dwq;
    p.dw[1] = dwk;
    const unsigned blocks = (unsigned) ((a.head_dim + 15) / 16 * (a.n_kv_head ? 2 : 1));
    by_types(a.type, a.w_type, [&](auto, auto we) { qk_reduce_kernel<decltype(we)><<<blocks, 1024, 0, s>>>(p, (int) grid); });
    return nxg_launch_check(what);
}

int32_t nxg_dropout_rows(int32_t type, const void * x, int64_t x_stride, const void * residual, int64_t residual_stride, int32_t T,
                         int32_t C, double drop, uint64_t seed, uint64_t offset, const int64_t * step, void * out,
                         int64_t out_stride, void * stream) {
    const char * what = "dropout_rows";
    const int es = size_of(type);
    if (!es) return nxg_fail(NXG_EINVAL, "%s: type %d (F32, F16 or BF16)", what, type);
    if (T < 0 || C < 1 || C > 1 << 30) return nxg_fail(NXG_EINVAL, "%s: T=%d C=%d", what, T, C);
    if (!(drop >= 0.0) || !(drop < 1.0) || std::nearbyint(drop * 65536.0) > 65535.0) return nxg_fail(NXG_EINVAL, "%s: p=%g (0 to 65535 / 65536)", what, drop);
    if (T == 0) return NXG_OK;
    NXG_TRY(check_norm_rows(what, "x", x, x_stride, T, C, es, false));
    if (residual) NXG_TRY(check_norm_rows(what, "residual", residual, residual_stride, T, C, es, false));
    NXG_TRY(check_norm_rows(what, "out", out, out_stride, T, C, es, true));
    if (step && !aligned(step, 8)) return nxg_fail(NXG_EINVAL, "%s: step is not aligned to its type", what);
    if (T > 1 && ((out == x && out_stride != x_stride) || (out == residual && out_stride != residual_stride))) {
        return nxg_fail(NXG_EINVAL, "%s: out is x or residual with another stride", what);
    }
    dropout_p p = {};
    p.x = x;
    p.residual = residual;
    p.out = out;
    p.x_s = T > 1 ? x_stride : 0;
    p.r_s = T > 1 ? residual_stride : 0;
    p.o_s = T > 1 ? out_stride : 0;
    p.step = step;
    p.seed = seed;
    p.offset = offset;
    p.T = T;
    p.C = C;
    p.groups = (C + 7) / 8;
    p.by_groups = (uint32_t) (((1ull << 32) + p.groups - 1) / p.groups);
    p.least = (uint32_t) std::nearbyint(drop * 65536.0);
    p.scale = 65536.0f / (float) (65536 - p.least);
    const int64_t grid = ((int64_t) T * p.groups + 256 * DROP_GROUPS - 1) / (256 * DROP_GROUPS);
    if (grid > MAX_GRID) return nxg_fail(NXG_EINVAL, "%s: T=%d C=%d is too large", what, T, C);
    NXG_TRY(nxg_check_device());
    const bool w = wide(x, p.x_s, es) && (!residual || wide(residual, p.r_s, es)) && wide(out, p.o_s, es) && C % (16 / es) == 0;
    by_type(type, [&](auto e) {
        if (w) dropout_rows_kernel<decltype(e), true><<<(unsigned) grid, 256, 0, (hipStream_t) stream>>>(p);
        else dropout_rows_kernel<decltype(e), false><<<(unsigned) grid, 256, 0, (hipStream_t) stream>>>(p);
    });
    return nxg_launch_check(what);
}

} // extern "C"
