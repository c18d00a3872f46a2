// nxg_rows.hip -- gfx950 kernels over packed floating-point rows: rotary positions and layer norm with its
// gradients, and their C ABI (include/nxg_rows.h). All of them are bound by HBM: rows are read and written
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

// The largest d with cu[d] <= t (0 if none): the row's document.
__device__ __forceinline__ int doc_of_row(const int32_t * cu, int n_seqs, int t) {
    int lo = 0, hi = n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
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
    for (int k = threadIdx.x; k < tokens * half; k += 256) {
        const int t = (int) t0 + k / half, i = k % half;
        int pos;
        if (p.positions) pos = p.positions[t];
        else pos = t - p.cu[doc_of_row(p.cu, p.n_seqs, t)];
        const double turns = (double) pos * p.freq[i] * 0.15915494309189533577;   // 1 / (2 pi)
        float s, c;
        sincospif(2.0f * (float) (turns - rint(turns)), &s, &c);
        turn[k] = make_float2(c * p.mscale, s * p.mscale * p.sign);
    }
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

} // extern "C"
