// nxg_attn_rows.hip -- gfx950 attention over packed 16-bit rows, forward and backward, and its C ABI
// (include/nxg_rows.h).
//
// One KV head's queries are taken as "pairs" (token, query head of the group), pair p = token * R + r
// with R = n_head / n_kv_head, so that the R heads that share K and V share their tiles too. Every
// product is an MFMA 32x32x16 with the wave's own 32 rows as the columns of the result:
//
//   forward, dQ   S^T = K Q^T     a lane holds 16 keys' scores of one pair (its column)
//   dK, dV        S   = Q K^T     a lane holds 16 pairs' scores of one key
//
// A lane's registers of such a result are, without a move between lanes, the operand of the product
// that follows (P V, dS K, P^T dO, dS^T Q): 32x32x16 wants 8 values of the contracted index per lane, and
// the order of that index is free as long as the other operand has the same. That other operand is
// the tile in LDS read in columns, which ds_read_b64_tr_b16 does 4 rows at a time.
//
// Softmax statistics, products and sums are fp32. P and dS are rounded to the inputs' type for the second
// products (at most half a step of a value in 0..1, its sign alternating over the keys; the sum stays
// fp32); fp16, whose range they would leave, carries them scaled by powers of two.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "nxg_rows.h"
#include "nxg_internal.h"

namespace {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;

// fp16 alone: P is carried as 2^15 P in the backward pass (P <= 1, fp16 ends at 65504), so that weights
// down to 2^-29 keep all their bits
constexpr int P_SHIFT = 15;
// ... and dS as f 2^15 P (dP - delta), a power of two f for each row that a lane sums up (dQ: a pair, dK: a key). It starts at
// DS_START, for dS down to 2^-74, and is lowered to where the largest value is in 2^9 .. 2^10 whenever one is past DS_TOP.
constexpr float DS_START = 0x1p45f, DS_TOP = 32768.0f;
constexpr int DS_PLACE = 10;

template <class E> struct type_of;
template <> struct type_of<__bf16> {
    typedef v8b v8;
    static constexpr bool HALF = false;
    static __device__ __forceinline__ v16f mfma(v8 a, v8 b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct type_of<_Float16> {
    typedef v8h v8;
    static constexpr bool HALF = true;
    static __device__ __forceinline__ v16f mfma(v8 a, v8 b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

struct rows {
    char * data;
    int64_t ts, hs;            // strides in bytes
};

struct attn_p {
    rows q, k, v, out, dout, dq, dk, dv;
    float * lse;               // [T_q][H]
    float * lse2, * ndelta;    // for the backward pass, a KV head's pairs one after another ([G][T_q R]): log2 of the sums, -delta
    float * part;              // partial sums of the split forward pass
    float * part_q, * part_kv; // partial gradients: [split_q][G][T_q R][D], [split_kv][dK, dV][G][T_k][D]
    const int32_t * cu_q, * cu_k;
    int32_t n_seqs, T_q, T_k, H, G, R, D, left, right, n_split, split_q, split_kv, order;
    float scale;
    uint32_t by_R;             // 2^22 / R, rounded up
    bool near_k, near_q;       // a tile's rows are within 32-bit offsets of its first
    bool even_q;               // pairs lie alike in every tile
};

// ---------------------------------------------------------------------------
// small pieces
// ---------------------------------------------------------------------------

__device__ __align__(16) const uint32_t zeros16[4] = {};

// 16 bytes per lane from global memory straight into LDS (lane l to lds + 16 l). From inline asm, so
// that the compiler does not wait for every prefetch before an LDS read; wait_all() and a barrier do.
__device__ __forceinline__ void dma16(const void * g, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" :: "v"(g), "s"(lds) : "memory", "m0");
}
// The same from a scalar base: lane l copies the 16 bytes at base + off_l.
__device__ __forceinline__ void dma16s(const char * base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
// 4 bytes per lane (lane l's at base + off_l to lds + 4 l).
__device__ __forceinline__ void dma4s(const void * base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" :: "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void wait_all() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_addr(const void * p) { return (uint32_t) (uintptr_t) (lds_void *) p; }

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ const char * uni(const char * p) {
    const uint64_t v = (uint64_t) (uintptr_t) p;
    return (const char *) (uintptr_t) (((uint64_t) (uint32_t) uni((int) (v >> 32)) << 32) | (uint32_t) uni((int) (uint32_t) v));
}

// max over the two halves of the wave
__device__ __forceinline__ float half_max(float x) {
    const v2u r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const v2u r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Row offsets as the caller gave them, kept inside the arrays whatever they hold.
__device__ __forceinline__ int offset(const int32_t * cu, int d, int T) { return min(max(cu[d], 0), T); }

// The document of a tile slot. Document d owns the slots from floor(cu[d] * mul / tile) + d, which are at
// least as many as its ceil(len * mul / tile) tiles, so the slots need no pass over the lengths: T * mul /
// tile + n_seqs of them in all. 64 documents are tried at a time.
__device__ __forceinline__ int64_t slot_of(const int32_t * cu, int d, int T, int mul, int tile) {
    return (int64_t) offset(cu, d, T) * mul / tile + d;
}
__device__ __forceinline__ int find_doc(const int32_t * cu, int n_seqs, int T, int mul, int tile, int slot) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = n_seqs;               // the document is in lo .. lo + n - 1
    while (n > 1) {
        const int step = (n + 63) >> 6;
        const int d = lo + lane * step;
        const bool at = lane * step < n && slot_of(cu, d, T, mul, tile) <= slot;
        const int last = max(__popcll(__ballot(at)) - 1, 0);
        n = min(step, n - last * step);
        lo += last * step;
    }
    return uni(lo);
}

struct doc {
    int q0, n, k0, m;          // first query row, queries, first key row, keys
};
__device__ __forceinline__ doc doc_of(const attn_p & p, int d) {
    doc r;
    r.q0 = uni(offset(p.cu_q, d, p.T_q));
    r.n = uni(max(offset(p.cu_q, d + 1, p.T_q) - r.q0, 0));
    r.k0 = uni(offset(p.cu_k, d, p.T_k));
    r.m = uni(max(offset(p.cu_k, d + 1, p.T_k) - r.k0, 0));
    return r;
}

// Sum of the lanes up to this one.
__device__ __forceinline__ int scan64(int x) {
#define NXG_STEP(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, false)
    NXG_STEP(0x111, 0xf);      // row_shr 1, 2, 4, 8
    NXG_STEP(0x112, 0xf);
    NXG_STEP(0x114, 0xf);
    NXG_STEP(0x118, 0xf);
    NXG_STEP(0x142, 0xa);      // row_bcast 15, 31
    NXG_STEP(0x143, 0xc);
#undef NXG_STEP
    return x;
}

// What a workgroup does: a tile (BM query-head pairs, or keys) of a document.
struct job {
    doc c;
    int tile;                  // -1: nothing
};

// The order of a launch's workgroups, so that the last to start are short ones.
enum { BY_ROWS, BY_LENGTH, BY_LEVEL };

// The slot's job. A document has ceil(len mul / size) tiles, by its queries or its keys (by_keys). BY_ROWS: slots as
// find_doc() gives them. For up to 64 documents, a lane each: BY_LENGTH takes the longest documents first
// (full windows: a tile's work is its document's length), BY_LEVEL the tiles with the most work of all documents
// first (windows open on one side: a tile's work is its number, from the end where from_end).
__device__ __forceinline__ job find_job(const attn_p & p, bool by_keys, int mul, int size, int slot, int order, bool from_end) {
    job r;
    r.tile = -1;
    const int32_t * cu = by_keys ? p.cu_k : p.cu_q;
    const int T = by_keys ? p.T_k : p.T_q;
    if (p.n_seqs > 64) {
        const int d = find_doc(cu, p.n_seqs, T, mul, size, slot);
        r.c = doc_of(p, d);
        const int64_t at = slot - slot_of(cu, d, T, mul, size);
        const int64_t len = (int64_t) (by_keys ? r.c.m : r.c.n) * mul;
        if (at >= 0 && at * size < len) r.tile = uni((int) (from_end ? (len + size - 1) / size - 1 - at : at));
        return r;
    }
    // a document a lane, its offsets in one load each
    const int lane = threadIdx.x & 63, d = min(lane, p.n_seqs - 1);
    const int q0 = offset(p.cu_q, d, p.T_q), n = max(offset(p.cu_q, d + 1, p.T_q) - q0, 0);
    const int k0 = offset(p.cu_k, d, p.T_k), m = max(offset(p.cu_k, d + 1, p.T_k) - k0, 0);
    const int count = lane < p.n_seqs ? (int) (((int64_t) (by_keys ? m : n) * mul + size - 1) / size) : 0;
    auto take = [&](int at, int tile) {
        r.c.q0 = __builtin_amdgcn_readlane(q0, at);
        r.c.n = __builtin_amdgcn_readlane(n, at);
        r.c.k0 = __builtin_amdgcn_readlane(k0, at);
        r.c.m = __builtin_amdgcn_readlane(m, at);
        r.tile = uni(tile);
    };
    if (order == BY_ROWS) {
        const int upto = scan64(count);
        const uint64_t here = __ballot(slot < upto);
        if (!here) return r;
        const int at = __builtin_ctzll(here), left = __builtin_amdgcn_readlane(upto, at) - slot;
        take(at, from_end ? left - 1 : __builtin_amdgcn_readlane(count, at) - left);
        return r;
    }
    int rank = 0;              // documents of more tiles, or as many and before this one
    for (int j = 0; j < p.n_seqs; ++j) {
        const int cj = __builtin_amdgcn_readlane(count, j);
        rank += cj > count || (cj == count && j < lane);
    }
    if (lane >= p.n_seqs) rank = lane;
    const int c = __builtin_amdgcn_ds_permute(rank << 2, count);       // lane r: the r'th most
    const int upto = scan64(c);
    int doc_rank, tile;
    if (order == BY_LENGTH) {
        const uint64_t here = __ballot(slot < upto);
        if (!here) return r;
        doc_rank = __builtin_ctzll(here);
        tile = slot - (__builtin_amdgcn_readlane(upto, doc_rank) - __builtin_amdgcn_readlane(c, doc_rank));
    } else {
        // tiles of the first r + 1 documents above the next one's count
        // (every lane takes part in the move: what a lane that is switched off holds reads as 0)
        const int down = __shfl_down(c, 1), next = lane < 63 ? down : 0;
        const int above = upto - (lane + 1) * next;
        const uint64_t here = __ballot(slot < above);
        if (!here) return r;
        const int last = __builtin_ctzll(here);
        const int k = slot - (last ? __builtin_amdgcn_readlane(above, last - 1) : 0);
        tile = __builtin_amdgcn_readlane(c, last) - 1 - k / (last + 1);
        doc_rank = k % (last + 1);
    }
    const int at = __builtin_ctzll(__ballot(rank == doc_rank));
    if (from_end && order == BY_LEVEL) tile = __builtin_amdgcn_readlane(count, at) - 1 - tile;
    take(at, tile);
    return r;
}

// The same for a whole workgroup: found by its first wave, through LDS (with a barrier).
__device__ __forceinline__ job workgroup_job(const attn_p & p, bool by_keys, int mul, int size, int slot, bool from_end, int * lds) {
    if (p.order == BY_ROWS) return find_job(p, by_keys, mul, size, slot, BY_ROWS, from_end);
    if (uni(threadIdx.x >> 6) == 0) {
        const job f = find_job(p, by_keys, mul, size, slot, p.order, from_end);
        if (threadIdx.x == 0) {
            lds[0] = f.c.q0;
            lds[1] = f.c.n;
            lds[2] = f.c.k0;
            lds[3] = f.c.m;
            lds[4] = f.tile;
        }
    }
    barrier();
    job r;
    r.c.q0 = uni(lds[0]);
    r.c.n = uni(lds[1]);
    r.c.k0 = uni(lds[2]);
    r.c.m = uni(lds[3]);
    r.tile = uni(lds[4]);
    return r;
}

// The keys lo .. hi - 1 of query token t.
__device__ __forceinline__ int key_lo(const attn_p & p, const doc & c, int t) {
    return p.left < 0 ? 0 : min(max(t + c.m - c.n - p.left, 0), c.m);
}
__device__ __forceinline__ int key_hi(const attn_p & p, const doc & c, int t) {
    return p.right < 0 ? c.m : min(max(t + c.m - c.n + p.right + 1, 0), c.m);
}
// The query tokens lo .. hi - 1 that see key j.
__device__ __forceinline__ int tok_lo(const attn_p & p, const doc & c, int j) {
    return p.right < 0 ? 0 : min(max(j - (c.m - c.n) - p.right, 0), c.n);
}
__device__ __forceinline__ int tok_hi(const attn_p & p, const doc & c, int j) {
    return p.left < 0 ? c.n : min(max(j - (c.m - c.n) + p.left + 1, 0), c.n);
}

// ---------------------------------------------------------------------------
// tiles in LDS
// ---------------------------------------------------------------------------
//
// A tile is rows of SP = 64 or 128 values (the head's D, zeros behind it). The 16-byte chunk c of row r is
// at chunk c ^ swz(r) of the row, so that a cycle of LDS (64 banks of 4 bytes) is filled both by 16 rows'
// same chunk (reads of rows, 16 lanes a cycle) and by 4 rows' 4 neighbouring chunks (reads of columns, 32 lanes
// a cycle). swz(a ^ b) = swz(a) ^ swz(b).

template <int DT> constexpr int SP = DT <= 2 ? 64 : 128;

template <int DT>
__device__ __forceinline__ constexpr int swz(int r) {
    return SP<DT> == 64 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : (r & 3) << 2 | ((r >> 2) & 3);
}

// Copies NR rows by the NT threads of a workgroup (NT = 256) or a wave (64) into a tile. A thread's place
// within a tile is computed once; a tile is a new scalar base, and so is each of a thread's rows (STEP
// rows further). Chunks behind D are never written: clear() before.
template <int DT, int NR, int NT>
struct tile_loader {
    static constexpr int CH = SP<DT> / 8, N = NR * CH / NT, STEP = NT / CH;
    int D;
    uint32_t off;              // of the thread's first row r0 from the tile's base
    uint32_t wave_at;          // the wave's first row in the tile
    int64_t step;              // of STEP rows

    static __device__ __forceinline__ int row_of(int t) { return (NT == 64 ? t & 63 : t) / CH; }
    // The chunk of the thread's k'th row, r0 + k STEP = r0 ^ k STEP.
    static __device__ __forceinline__ int chunk_of(int t, int k) { return (t % CH) ^ swz<DT>(row_of(t)) ^ swz<DT>(k * STEP); }

    __device__ __forceinline__ tile_loader(int D_) : D(D_), wave_at(NT == 64 ? 0 : uni((int) (threadIdx.x >> 6)) * 1024) {}
    // Rows ts bytes apart; or pairs, R to a token (R divides STEP), heads hs bytes apart.
    __device__ __forceinline__ void rows_at(int64_t ts) {
        off = (uint32_t) (row_of(threadIdx.x) * ts);
        step = STEP * ts;
    }
    __device__ __forceinline__ void pairs_at(int R, int64_t ts, int64_t hs) {
        const int r0 = row_of(threadIdx.x);
        off = (uint32_t) (r0 / R * ts + r0 % R * hs);
        step = STEP / R * ts;
    }
    __device__ __forceinline__ void load(const char * base, uint32_t lds) const {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int c = chunk_of(threadIdx.x, k);
            if (c * 8 < D) dma16s(base + k * step, off + c * 16, lds + wave_at + k * NT * 16);
        }
    }
    // Pairs from the r0'th of the base's token on, any R (their places differ from tile to tile); by_R = 2^22 / R, rounded up: exact
    // for (64 + R) R < 2^22.
    __device__ __forceinline__ void load_pairs(const char * base, int r0, int R, uint32_t by_R, uint32_t ts, uint32_t hs, uint32_t lds) const {
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const uint32_t x = r0 + row_of(t) + k * STEP, token = x * by_R >> 22;
            const int c = chunk_of(t, k);
            if (c * 8 < D) dma16s(base, token * ts + (x - token * R) * hs + c * 16, lds + wave_at + k * NT * 16);
        }
    }
    // row r from src(r), zeros where that is null
    template <class Src>
    __device__ __forceinline__ void load_each(uint32_t lds, Src src) const {
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));        // few tiles come here: nothing of it is kept in registers
#pragma unroll 1
        for (int k = 0; k < N; ++k) {
            const char * s = src(row_of(t) + k * STEP);
            const int c = chunk_of(t, k);
            if (c * 8 < D) dma16(s ? s + c * 16 : (const char *) zeros16, uni((int) (lds + wave_at + k * NT * 16)));
        }
    }
};

// The tiles of a document's m keys one after another, K and V each by itself; K's start k_ahead keys further.
template <int DT, int NR, int NT>
struct key_stream {
    tile_loader<DT, NR, NT> lk, lv;
    const char * k, * v;       // of the next tile's first rows
    int jk, jv, m, step;       // their keys; keys from one tile to the next
    int64_t kts, vts;
    bool near;

    __device__ __forceinline__ key_stream(const attn_p & p, const doc & c, int g, int first, int step_, int k_ahead = 0)
        : lk(p.D), lv(p.D), jk(first + k_ahead), jv(first), m(c.m), step(step_), kts(p.k.ts), vts(p.v.ts), near(p.near_k) {
        lk.rows_at(kts);
        lv.rows_at(vts);
        k = uni(p.k.data + (c.k0 + (int64_t) jk) * kts + g * p.k.hs);
        v = uni(p.v.data + (c.k0 + (int64_t) jv) * vts + g * p.v.hs);
    }
    __device__ __forceinline__ void next_k(uint32_t lds) {
        if (near && jk + NR <= m) lk.load(k, lds);
        else lk.load_each(lds, [&](int r) { return jk + r < m ? k + r * kts : nullptr; });
        jk += step;
        k += step * kts;
    }
    // the tile before the first, as far as it is within the document (with k_ahead)
    __device__ __forceinline__ void first_k(uint32_t lds) {
        lk.load_each(lds, [&](int r) { return (unsigned) (jk - step + r) < (unsigned) m ? k + (r - step) * kts : nullptr; });
    }
    __device__ __forceinline__ void next_v(uint32_t lds) {
        if (near && jv + NR <= m) lv.load(v, lds);
        else lv.load_each(lds, [&](int r) { return jv + r < m ? v + r * vts : nullptr; });
        jv += step;
        v += step * vts;
    }
    __device__ __forceinline__ void next(uint32_t lds_k, uint32_t lds_v) {
        next_k(lds_k);
        next_v(lds_v);
    }
};

// Zeros the chunks behind D of n tiles' memory (all of it), before the first load.
__device__ __forceinline__ void clear(void * lds, int bytes, int thread, int threads) {
    for (int i = thread * 16; i < bytes; i += threads * 16) *reinterpret_cast<v4i *>((char *) lds + i) = v4i{0, 0, 0, 0};
}

// A lane's places in a tile, as byte offsets whose chunk is varied by an exclusive or.
struct lane_at {
    uint32_t row, col;
};
template <int DT>
__device__ __forceinline__ lane_at lane_places() {
    const int lane = threadIdx.x & 63, r = lane & 31, i = lane & 15, g = lane >> 4;
    const int cr = 4 * (g >> 1) + (i >> 2);
    lane_at o;
    o.row = r * SP<DT> * 2 + (((lane >> 5) ^ swz<DT>(r)) << 4);
    o.col = cr * SP<DT> * 2 + (((2 * (g & 1) + ((i & 3) >> 1)) ^ swz<DT>(cr)) << 4) + (i & 1) * 8;
    return o;
}

// Operand of 32 rows from r0: lane l's row r0 + l % 32, values 16 s + 8 (l / 32) + 0..7. `at`: the tile's LDS
// address + lane_at.row.
template <class E, int DT>
__device__ __forceinline__ typename type_of<E>::v8 row_operand(uint32_t at, int r0, int s) {
    typedef __attribute__((address_space(3))) v4i lds_v4i;
    const v4i x = *(lds_v4i *) (uintptr_t) ((at ^ (s << 5)) + r0 * SP<DT> * 2);
    typename type_of<E>::v8 out;
    __builtin_memcpy(&out, &x, 16);
    return out;
}

// Operand of the 32 columns from 32 d, rows r0 + 4 (l / 32) + {0..3, 8..11}: the rows of registers 0..7 of a
// 32x32 result (r0 a multiple of 16). `at`: the tile's LDS address + lane_at.col.
template <class E, int DT>
__device__ __forceinline__ typename type_of<E>::v8 col_operand(uint32_t at, int r0, int d) {
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    v4s x[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
        x[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *) (uintptr_t) ((at ^ (d << 6 | swz<DT>(8 * k) << 4)) + (r0 + 8 * k) * SP<DT> * 2));
    typename type_of<E>::v8 out;
    __builtin_memcpy(&out, x, 16);
    return out;
}

// Register i of lane l of a 32x32 result is row 8 (i / 4) + 4 (l / 32) + i % 4 of column l % 32.
__device__ __forceinline__ constexpr int reg_row(int i) { return 8 * (i / 4) + i % 4; }

// Sets the registers whose row is not in the lane's lo .. hi - 1 to x; sides: 1 if a row may be below lo, 2 if one may be
// past hi (of the wave's 32 columns; at no side most tiles).
__device__ __forceinline__ void mask_rows(v16f & s, int sides, int lo, int hi, float x) {
    const int h4 = 4 * ((int) (threadIdx.x & 63) >> 5);
    if (sides & 1) {
        const int l = lo - h4;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = reg_row(i) < l ? x : s[i];
    }
    if (sides & 2) {
        const int l = hi - h4;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = reg_row(i) >= l ? x : s[i];
    }
}

// Registers 8 a .. 8 a + 7 as the operand of the next product.
template <class E>
__device__ __forceinline__ typename type_of<E>::v8 pack(const v16f & x, int a) {
    typename type_of<E>::v8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (E) x[8 * a + j];
    return o;
}

// The wave's own 32 rows of D values as operands in registers, from src (this lane's row); one, or two at once.
template <class E, int DT>
__device__ __forceinline__ void issue_operand(v4i (&z)[2 * DT], const char * src, int D) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int s = 0; s < 2 * DT; ++s) {
        z[s] = v4i{0, 0, 0, 0};
        if (16 * s + 8 * h < D) z[s] = *reinterpret_cast<const v4i *>(src + (16 * s + 8 * h) * 2);
    }
}
template <class E, int DT>
__device__ __forceinline__ void take_operand(typename type_of<E>::v8 (&x)[2 * DT], v4i (&z)[2 * DT]) {
    // arrived here, not at their first use: that is in a loop, where the compiler would wait for the tiles
    // under way as well
#pragma unroll
    for (int s = 0; s < 2 * DT; ++s) {
        asm volatile("" : "+v"(z[s]));
        __builtin_memcpy(&x[s], &z[s], 16);
    }
}
template <class E, int DT>
__device__ __forceinline__ void load_operand(typename type_of<E>::v8 (&x)[2 * DT], const char * src, int D) {
    v4i z[2 * DT];
    issue_operand<E, DT>(z, src, D);
    take_operand<E, DT>(x, z);
}
template <class E, int DT>
__device__ __forceinline__ void load_operands(typename type_of<E>::v8 (&x)[2 * DT], const char * x_src, typename type_of<E>::v8 (&y)[2 * DT],
                                              const char * y_src, int D) {
    v4i zx[2 * DT], zy[2 * DT];
    issue_operand<E, DT>(zx, x_src, D);
    issue_operand<E, DT>(zy, y_src, D);
    take_operand<E, DT>(x, zx);
    take_operand<E, DT>(y, zy);
}

// The wave's 32 columns of DT 32x32 results as rows of D values in memory, scaled by f: through a tile
// of 32 rows of LDS, so that a row is written in 16-byte pieces one after another. dst(c): column c's row, or null.
template <class E, int DT, class Dst>
__device__ __forceinline__ void store_columns(E * tile, const v16f (&acc)[DT], float f, int D, Dst dst) {
    typedef E v4e __attribute__((ext_vector_type(4)));
    constexpr int CH = SP<DT> / 8;
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));            // nothing of this is kept in registers over the loop before
    const int col = lane & 31, h = lane >> 5;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v4e e;
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = (E) (acc[d][4 * k + i] * f);
            const int c = (4 * d + k) ^ swz<DT>(col);
            *reinterpret_cast<v4e *>(tile + col * SP<DT> + c * 8 + 4 * h) = e;
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int it = 0; it < 32 * CH / 64; ++it) {
        const int r = (it * 64 + lane) / CH, c = lane % CH;
        char * o = dst(r);
        const v4i x = *reinterpret_cast<const v4i *>(tile + r * SP<DT> + (c ^ swz<DT>(r)) * 8);
        if (o && c * 8 < D) *reinterpret_cast<v4i *>(o + c * 16) = x;
    }
}

// The same as rows of D floats in memory, one after another, the first n of them: a split's share of a sum.
template <int DT>
__device__ __forceinline__ void store_partial(const v16f (&acc)[DT], float f, int D, int n, float * to) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    if ((lane & 31) >= n) return;
    float * o = to + (lane & 31) * D + 4 * (lane >> 5);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (32 * d + 8 * k < D) *reinterpret_cast<v4f *>(o + 32 * d + 8 * k) = v4f{acc[d][4 * k], acc[d][4 * k + 1], acc[d][4 * k + 2], acc[d][4 * k + 3]} * f;
}

// The part of the tiles lo .. hi - 1 that a split takes, every split but the last as many; those behind the last tile
// take none.
struct span {
    int lo, hi;
};
__device__ __forceinline__ int share_of(span x, int n_split) { return (max(x.hi - x.lo, 0) + n_split - 1) / n_split; }
__device__ __forceinline__ span split_of(span x, int n_split, int split) {
    const int share = share_of(x, n_split);
    return {x.lo + split * share, min(x.lo + (split + 1) * share, x.hi)};
}

// ---------------------------------------------------------------------------
// sums taken again
// ---------------------------------------------------------------------------
//
// A product over a tile takes in every row of it, those that a pair does not see with weight 0. If such a row
// holds an infinity or a NaN, 0 times it is NaN. So a result that is not finite, where rows that some
// pair of the wave does not see hold such values, is taken again from the definition, over the seen rows alone.
// That costs nothing until it happens.

// Bit c: column c of the wave's sums (both half waves) is not finite.
template <int DT>
__device__ __forceinline__ uint32_t bad_columns(const v16f (&x)[DT]) {
    float z = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) z = __builtin_fmaf(x[d][i], 0.0f, z);
    const uint64_t b = __ballot(z != 0.0f || z != z);
    return (uint32_t) b | (uint32_t) (b >> 32);
}

// Does any of the rows a .. b - 1 hold a value that is not finite? row(i): its D values.
template <class E, class Row>
__device__ __forceinline__ bool holds_bad(int a, int b, int D, Row row) {
    const int lane = threadIdx.x & 63, chunks = D / 8;
    bool bad = false;
    for (int i = lane; i < (b - a) * chunks; i += 64) {
        const typename type_of<E>::v8 x = *reinterpret_cast<const typename type_of<E>::v8 *>(row(a + i / chunks) + i % chunks * 16);
#pragma unroll
        for (int k = 0; k < 8; ++k) bad |= !(fabsf((float) x[k]) < INFINITY);
    }
    return __any(bad);
}

template <class E>
__device__ __forceinline__ float dot(const char * a, const char * b, int D) {
    float s = 0.0f;
    for (int d = 0; d < D; d += 8) {
        const typename type_of<E>::v8 x = *reinterpret_cast<const typename type_of<E>::v8 *>(a + 2 * d);
        const typename type_of<E>::v8 y = *reinterpret_cast<const typename type_of<E>::v8 *>(b + 2 * d);
#pragma unroll
        for (int k = 0; k < 8; ++k) s = __builtin_fmaf((float) x[k], (float) y[k], s);
    }
    return s;
}

// The wave's sum over j in a .. b - 1 of weight(j) times row(j): lane l has values l and 64 + l. lds: 64 floats.
template <class E, class Weight, class Row>
__device__ __forceinline__ void add_rows(float (&x)[2], int a, int b, int D, float * lds, Weight weight, Row row) {
    const int lane = threadIdx.x & 63;
    for (int j = a; j < b; j += 64) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        lds[lane] = j + lane < b ? weight(j + lane) : 0.0f;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        for (int k = 0; k < min(64, b - j); ++k) {
            const E * r = reinterpret_cast<const E *>(row(j + k));
            const float w = lds[k];
            if (lane < D) x[0] += w * (float) r[lane];
            if (64 + lane < D) x[1] += w * (float) r[64 + lane];
        }
    }
}

template <class E>
__device__ __forceinline__ void store_row(char * to, const float (&x)[2], float f, int D) {
    const int lane = threadIdx.x & 63;
    E * o = reinterpret_cast<E *>(to);
    if (lane < D) o[lane] = (E) (x[0] * f);
    if (64 + lane < D) o[64 + lane] = (E) (x[1] * f);
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int k = 32; k; k >>= 1) x = fmaxf(x, __shfl_xor(x, k));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int k = 32; k; k >>= 1) x += __shfl_xor(x, k);
    return x;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------

// Running softmax of the wave's 32 pairs. mc: the exponentials' reference in powers of two (-inf before the
// first key); l: the half wave's share of sum p; o = sum p v.
template <int DT>
struct fwd_state {
    float mc, l;
    v16f o[DT];

    // some: the lane's pair sees a key at all
    __device__ __forceinline__ void init(bool some) {
        mc = some ? -INFINITY : 0.0f;
        l = 0.0f;
#pragma unroll
        for (int k = 0; k < DT; ++k) o[k] = v16f{};
    }
};

// A sum of weights past which the reference is raised: P stays in either type's range, and the largest score is
// looked for in few tiles, the first and some after it. A raise leaves the largest weight at 2^TOP: bf16 has fp32's exponents,
// fp16 would lose weights below 2^-24, of which a long document's sum has many (one key 17.3 above 65,536 others alike:
// their sum, 0.002 of all, as 0), and so loses those below 2^-34 of the largest.
template <class E> struct reference {
    static constexpr float RAISE = type_of<E>::HALF ? 60000.0f : 16384.0f, TOP = type_of<E>::HALF ? 10.0f : 0.0f;
};

// Scores of the wave's pairs with the 32 keys from row r0 of the tile.
template <class E, int DT>
__device__ __forceinline__ v16f fwd_scores(const typename type_of<E>::v8 (&q)[2 * DT], uint32_t kt, int r0) {
    v16f s = {};
#pragma unroll
    for (int d = 0; d < 2 * DT; ++d) s = type_of<E>::mfma(row_operand<E, DT>(kt, r0, d), q[d], s);
    return s;
}

__device__ __forceinline__ float fwd_exp(v16f & w, const v16f & s, float c, float mc) {
    float t[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -mc));
        t[i & 1] = i < 2 ? w[i] : t[i & 1] + w[i];
    }
    return t[0] + t[1];
}

// The weights of 32 keys from their scores, with a new reference where the old one is passed: the largest
// score so far (fp16: 2^10 below it).
template <class E, int DT>
__device__ __forceinline__ void fwd_weights(v16f & w, const v16f & s, fwd_state<DT> & st, float c) {
    float t = fwd_exp(w, s, c, st.mc);
    if (__any(!(t <= reference<E>::RAISE))) {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        const float mc = fmaxf(st.mc, half_max(mx) * c - reference<E>::TOP);
        const float f = st.mc == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.mc - mc);
        st.mc = mc;
        st.l *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) st.o[d][i] *= f;
        t = fwd_exp(w, s, c, mc == -INFINITY ? 0.0f : mc);
    }
    st.l += t;
}

// o += V^T P^T for the 32 keys from row r0 of the tile.
template <class E, int DT>
__device__ __forceinline__ void fwd_values(fwd_state<DT> & st, const v16f & w, uint32_t vt, int r0) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        const typename type_of<E>::v8 pa = pack<E>(w, a);
#pragma unroll
        for (int d = 0; d < DT; ++d) st.o[d] = type_of<E>::mfma(col_operand<E, DT>(vt, r0 + 16 * a, d), pa, st.o[d]);
    }
}

// One pair's sums again, over its keys among the tiles first, first + step, ... below end of `size` keys: mc, l (its
// whole sum) and o as in fwd_state, lane l with o's values l and 64 + l.
template <class E>
__device__ __forceinline__ void fwd_again(const attn_p & p, const doc & c, int g, int pair, int first, int step, int end, int size,
                                          float * lds, float & mc, float & l, float (&o)[2]) {
    const int tok = pair / p.R, head = g * p.R + pair % p.R, lane = threadIdx.x & 63;
    const int lo = key_lo(p, c, tok), hi = key_hi(p, c, tok);
    const char * q = p.q.data + (c.q0 + tok) * p.q.ts + head * p.q.hs;
    const char * k = p.k.data + c.k0 * p.k.ts + g * p.k.hs, * v = p.v.data + c.k0 * p.v.ts + g * p.v.hs;
    const float cs = p.scale * LOG2E;
    float mx = -INFINITY, t = 0.0f;
    for (int j = first; j < end; j += step)
        for (int i = max(j * size, lo) + lane; i < min((j + 1) * size, hi); i += 64) mx = fmaxf(mx, dot<E>(q, k + i * p.k.ts, p.D));
    mx = wave_max(mx) * cs;
    mc = mx == -INFINITY ? 0.0f : mx;
    o[0] = o[1] = 0.0f;
    for (int j = first; j < end; j += step) {
        add_rows<E>(o, max(j * size, lo), min((j + 1) * size, hi), p.D, lds, [&](int i) {
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(dot<E>(q, k + i * p.k.ts, p.D), cs, -mc));
            t += w;
            return w;
        }, [&](int i) { return v + i * p.v.ts; });
    }
    l = wave_sum(t);
}

// A workgroup: 128 pairs of one document and KV head, a wave each 32 of them; 64 keys at a time. The scores of
// the next 32 keys are computed beside the exponentials of these, which take about as long as both products:
// K's tiles start 32 keys behind V's. Every wave takes every tile of the workgroup (the windows of its 128 pairs
// differ by few keys), so that the loop has no branches between the products.
//
// Bound by the matrix units, and by the power that they and the exponentials beside them draw together: 65,536 tokens,
// 16 heads of 64 on 8, bf16, full: 17.1 ms, 1,030 TFLOP/s (a library product of 8,192^3 reaches 1,138); the LDS copies cost
// 7 to 9% of it, the exponentials 7%. 32 documents of 32,900 tokens, causal: 135 us, 680 TFLOP/s, the rest the starts
// and ends of 4,248 workgroups of 11 tiles (9% of the tiles' pairs are masked). With 128 values a head 8,192 tokens full take 510 us,
// 1,078 TFLOP/s; 8 x 1,024 tokens in a band of 257 keys 24 us, 5 tiles a workgroup, bound by their latency.
template <class E, int DT>
__global__ __launch_bounds__(256, 2) void attn_rows_fwd_kernel(attn_p p) {
    constexpr int BM = 128, BN = 64, TILE = BN * SP<DT>;
    __shared__ __align__(1024) E sk[2][TILE], sv[2][TILE];
    __shared__ int s_job[8];
    const int g = blockIdx.x % p.G;
    const job todo = workgroup_job(p, false, p.R, BM, blockIdx.x / p.G, p.right >= 0 ? p.order == BY_ROWS : p.left >= 0 && p.order != BY_ROWS, s_job);
    if (todo.tile < 0) return;
    const doc c = todo.c;
    const int np = c.n * p.R, p0 = todo.tile * BM;

    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int pw = p0 + 32 * wave;
    const bool active = pw < np;
    const int pc = min(pw + (lane & 31), np - 1), tok = pc / p.R, head = g * p.R + pc % p.R;
    const int lo = key_lo(p, c, tok), hi = key_hi(p, c, tok);
    // keys of the workgroup, and of the wave: some pair's, and every pair's
    const int t_end = (min(p0 + BM, np) - 1) / p.R;
    const int j_lo = key_lo(p, c, p0 / p.R) / BN, j_hi = (key_hi(p, c, t_end) + BN - 1) / BN;
    const int ta = uni(min(pw, np - 1) / p.R), tb = uni(min(pw + 31, np - 1) / p.R);
    const int all_lo = key_lo(p, c, tb), all_hi = key_hi(p, c, ta);

    key_stream<DT, BN, 256> keys(p, c, g, j_lo * BN, BN, 32);
    if (p.D != 32 * DT) {
        clear(sk, sizeof(sk), threadIdx.x, 256);
        clear(sv, sizeof(sv), threadIdx.x, 256);
        barrier();
    }

    fwd_state<DT> st;
    st.init(lo < hi);
    const float cs = p.scale * LOG2E;
    const lane_at at = lane_places<DT>();
    v16f s0, s1, w;
    if (j_lo < j_hi) {
        keys.first_k(lds_addr(sk[1]));
        keys.next_k(lds_addr(sk[0]));
        keys.next_v(lds_addr(sv[0]));
    }
    typename type_of<E>::v8 q[2 * DT];
    load_operand<E, DT>(q, p.q.data + (c.q0 + tok) * p.q.ts + head * p.q.hs, p.D);
    if (j_lo < j_hi) {
        wait_all();
        barrier();
        s0 = fwd_scores<E, DT>(q, lds_addr(sk[1]) + at.row, 32);
    }
    for (int j = j_lo; j < j_hi; ++j) {
        const int buf = (j - j_lo) & 1, j0 = j * BN;
        const uint32_t kt = lds_addr(sk[buf]) + at.row, vt = lds_addr(sv[buf]) + at.col;
        const int sides = (j0 < all_lo ? 1 : 0) | (j0 + BN > all_hi ? 2 : 0);
        wait_all();
        barrier();
        if (j + 1 < j_hi) {
            keys.next_k(lds_addr(sk[buf ^ 1]));
            keys.next_v(lds_addr(sv[buf ^ 1]));
        }
        if (sides) mask_rows(s0, sides, lo - j0, hi - j0, -INFINITY);
        s1 = fwd_scores<E, DT>(q, kt, 0);
        fwd_weights<E, DT>(w, s0, st, cs);
        fwd_values<E, DT>(st, w, vt, 0);
        if (sides) mask_rows(s1, sides, lo - j0 - 32, hi - j0 - 32, -INFINITY);
        s0 = fwd_scores<E, DT>(q, kt, 32);             // of the next tile's first keys
        fwd_weights<E, DT>(w, s1, st, cs);
        fwd_values<E, DT>(st, w, vt, 32);
    }
    barrier();
    if (!active) return;
    const float l = half_sum(st.l);
    if (lane < 32 && pw + lane < np) {
        const int pr = pw + lane;
        p.lse[(int64_t) (c.q0 + pr / p.R) * p.H + g * p.R + pr % p.R] = LN2 * (st.mc + __builtin_amdgcn_logf(l));
    }
    E * tile = (wave < 2 ? sk[0] : sv[0]) + (wave & 1) * 32 * SP<DT>;
    uint32_t bad = bad_columns<DT>(st.o);
    store_columns<E, DT>(tile, st.o, l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l), p.D, [&](int r) -> char * {
        const int pr = pw + r;
        if (pr >= np) return nullptr;
        return p.out.data + (int64_t) (c.q0 + pr / p.R) * p.out.ts + (g * p.R + pr % p.R) * p.out.hs;
    });
    if (!bad) return;
    auto v_row = [&](int j) { return p.v.data + (int64_t) (c.k0 + j) * p.v.ts + g * p.v.hs; };
    if (!holds_bad<E>(j_lo * BN, min(all_lo, c.m), p.D, v_row) && !holds_bad<E>(max(all_hi, 0), min(j_hi * BN, c.m), p.D, v_row)) return;
    for (; bad; bad &= bad - 1) {
        const int pair = pw + __builtin_ctz(bad);
        if (pair >= np) break;
        float mc, l, o[2];
        fwd_again<E>(p, c, g, pair, j_lo, 1, j_hi, BN, reinterpret_cast<float *>(tile), mc, l, o);
        store_row<E>(p.out.data + (int64_t) (c.q0 + pair / p.R) * p.out.ts + (g * p.R + pair % p.R) * p.out.hs, o,
                     l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l), p.D);
    }
}

// Few pairs: a workgroup takes 32 of them, its four waves every fourth 32 keys of the split's share, each through
// LDS of its own; the waves' sums are joined in LDS. With n_split > 1 the shares of a document's keys go to
// different workgroups, which leave sums (o, m, l) that attn_rows_join_kernel joins.
//
// A wave's tiles are its own so that it waits for its own loads alone, no barrier in the loop. Bound by HBM where the cache is
// long (one query over 65,536 keys, 16 heads of 64 on 8: 134 MB in 25 us, 5.4 TB/s, and 4 us of joining), else by the
// chain of loads, products and the join (32 queries over 16 to 2,048 keys, 68 MB: 20 us; 4 texts of 125 tokens: 7 us).
template <class E, int DT>
__global__ __launch_bounds__(256) void attn_rows_few_kernel(attn_p p) {
    constexpr int BM = 32, BN = 32, TILE = BN * SP<DT>;
    __shared__ __align__(1024) E lds[4][2][2][TILE];       // wave, buffer, K or V
    __shared__ float sm[4][32], sl[4][32], s_weights[4][64];
    const int g = blockIdx.x % p.G, rest = blockIdx.x / p.G, split = rest % p.n_split, slot = rest / p.n_split;
    const job todo = find_job(p, false, p.R, BM, slot, BY_ROWS, false);
    if (todo.tile < 0) return;
    const doc c = todo.c;
    const int np = c.n * p.R, p0 = todo.tile * BM;

    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int pc = min(p0 + (lane & 31), np - 1), tok = pc / p.R, head = g * p.R + pc % p.R;
    typename type_of<E>::v8 q[2 * DT];
    load_operand<E, DT>(q, p.q.data + (c.q0 + tok) * p.q.ts + head * p.q.hs, p.D);
    const int lo = key_lo(p, c, tok), hi = key_hi(p, c, tok);
    const int ta = uni(p0 / p.R), tb = uni(min(p0 + 31, np - 1) / p.R);
    const int all_lo = key_lo(p, c, tb), all_hi = key_hi(p, c, ta);
    const int t_lo = key_lo(p, c, ta) / BN, t_hi = (key_hi(p, c, tb) + BN - 1) / BN;
    // the split's share of the tiles t_lo .. t_hi - 1
    const int share = (max(t_hi - t_lo, 0) + p.n_split - 1) / p.n_split;
    const int j_lo = t_lo + split * share, j_hi = min(j_lo + share, t_hi);

    key_stream<DT, BN, 64> keys(p, c, g, (j_lo + wave) * BN, 4 * BN);
    if (p.D != 32 * DT) {
        clear(lds[wave], sizeof(lds[wave]), lane, 64);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    fwd_state<DT> st;
    st.init(lo < hi);
    const float cs = p.scale * LOG2E;
    const lane_at at = lane_places<DT>();
    int buf = 0;
    if (j_lo + wave < j_hi) keys.next(lds_addr(lds[wave][0][0]), lds_addr(lds[wave][0][1]));
    for (int j = j_lo + wave; j < j_hi; j += 4, buf ^= 1) {
        wait_all();
        if (j + 4 < j_hi) keys.next(lds_addr(lds[wave][buf ^ 1][0]), lds_addr(lds[wave][buf ^ 1][1]));
        const int j0 = j * BN;
        v16f s = fwd_scores<E, DT>(q, lds_addr(lds[wave][buf][0]) + at.row, 0), w;
        const int sides = (j0 < all_lo ? 1 : 0) | (j0 + BN > all_hi ? 2 : 0);
        if (sides) mask_rows(s, sides, lo - j0, hi - j0, -INFINITY);
        fwd_weights<E, DT>(w, s, st, cs);
        fwd_values<E, DT>(st, w, lds_addr(lds[wave][buf][1]) + at.col, 0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // read before the next load writes it
    }
    // join the waves: each leaves its sums in its own LDS, [column][d] as fp32 (32 SP values, as 4 tiles hold)
    const float l = half_sum(st.l);
    if (lane < 32) {
        sm[wave][lane] = l == 0.0f ? -INFINITY : st.mc;
        sl[wave][lane] = l;
    }
    float * so = reinterpret_cast<float *>(&lds[wave][0][0][0]);
#pragma unroll
    for (int k = 0; k < DT; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const v4f x = {st.o[k][4 * i], st.o[k][4 * i + 1], st.o[k][4 * i + 2], st.o[k][4 * i + 3]};
            *reinterpret_cast<v4f *>(so + (lane & 31) * SP<DT> + 32 * k + 8 * i + 4 * (lane >> 5)) = x;
        }
    if (uint32_t bad = bad_columns<DT>(st.o)) {
        auto v_row = [&](int j) { return p.v.data + (int64_t) (c.k0 + j) * p.v.ts + g * p.v.hs; };
        if (holds_bad<E>(t_lo * BN, min(all_lo, c.m), p.D, v_row) || holds_bad<E>(max(all_hi, 0), min(t_hi * BN, c.m), p.D, v_row)) {
            for (; bad; bad &= bad - 1) {
                const int col = __builtin_ctz(bad);
                if (p0 + col >= np) break;
                float mc, l, o[2];
                fwd_again<E>(p, c, g, p0 + col, j_lo + wave, 4, j_hi, BN, s_weights[wave], mc, l, o);
                if (lane == 0) {
                    sm[wave][col] = l == 0.0f ? -INFINITY : mc;
                    sl[wave][col] = l;
                }
                so[col * SP<DT> + lane] = o[0];
                if (SP<DT> > 64) so[col * SP<DT> + 64 + lane] = o[1];
            }
        }
    }
    barrier();
    constexpr int CH = SP<DT> / 8;
    constexpr int WAVE_F = 2 * 2 * TILE / 2;                // floats of a wave's LDS
    const float * all = reinterpret_cast<const float *>(&lds[0][0][0][0]);
    for (int idx = threadIdx.x; idx < 32 * CH; idx += 256) {
        const int r = idx / CH, cc = idx % CH, pr = p0 + r;
        if (pr >= np || cc * 8 >= p.D) continue;
        float m = -INFINITY, lt = 0.0f, x[8] = {};
#pragma unroll
        for (int w = 0; w < 4; ++w) m = fmaxf(m, sm[w][r]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = sm[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[w][r] - m);
            lt += f * sl[w][r];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] += sm[w][r] == -INFINITY ? 0.0f : f * all[w * WAVE_F + r * SP<DT> + cc * 8 + i];
        }
        const int64_t row = (int64_t) (c.q0 + pr / p.R) * p.H + g * p.R + pr % p.R;
        if (p.n_split > 1) {
            float * o = p.part + ((int64_t) split * p.T_q * p.H + row) * (p.D + 8);
            *reinterpret_cast<v4f *>(o + 8 + cc * 8) = v4f{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<v4f *>(o + 8 + cc * 8 + 4) = v4f{x[4], x[5], x[6], x[7]};
            if (cc == 0) {
                o[0] = m;
                o[1] = lt;
            }
            continue;
        }
        const float f = lt > 0.0f ? 1.0f / lt : (lt == 0.0f ? 0.0f : lt);
        typename type_of<E>::v8 e;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = (E) (x[i] * f);
        *reinterpret_cast<typename type_of<E>::v8 *>(p.out.data + (int64_t) (c.q0 + pr / p.R) * p.out.ts +
                                                     (g * p.R + pr % p.R) * p.out.hs + cc * 16) = e;
        if (cc == 0) p.lse[row] = m == -INFINITY && lt == 0.0f ? -INFINITY : LN2 * (m + __builtin_amdgcn_logf(lt));
    }
}

// The splits' sums of a (token, head) row joined: a wave a row, L lanes for its values (8 each), 64 / L groups of them
// for every 64 / L'th split, whose loads are independent; the groups' sums added at the end. 4.4 us for 16 rows of 64 values
// in 32 shares: a launch and two rounds of loads.
template <class E, int L>
__global__ __launch_bounds__(256) void attn_rows_join_kernel(attn_p p) {
    const int64_t row = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6), n_rows = (int64_t) p.T_q * p.H;
    const int lane = threadIdx.x & 63, cc = lane % L, first = lane / L;
    if (row >= n_rows) return;
    const int tok = (int) (row / p.H), head = (int) (row % p.H);
    // rows of no document have no sums
    if (tok >= offset(p.cu_q, p.n_seqs, p.T_q) || tok < offset(p.cu_q, 0, p.T_q)) return;
    const float * part = p.part + row * (p.D + 8);
    const int64_t next = n_rows * (p.D + 8);
    // m and l of split `lane` (64 at most); a share without keys has -inf and 0
    const bool mine = lane < p.n_split;
    const float m = mine ? part[lane * next] : -INFINITY, l = mine ? part[lane * next + 1] : 0.0f;
    const float top = wave_max(m);
    const float f = m == -INFINITY && l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    const float total = wave_sum(f * l);
    float x[8] = {};
#pragma unroll 4
    for (int s0 = 0; s0 < p.n_split; s0 += 64 / L) {
        const int s = s0 + first;
        const float fs = __shfl(f, s);
        if (s < p.n_split && cc * 8 < p.D && fs != 0.0f) {
            const v4f a = *reinterpret_cast<const v4f *>(part + s * next + 8 + cc * 8), b = *reinterpret_cast<const v4f *>(part + s * next + 12 + cc * 8);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] += fs * a[i];
                x[4 + i] += fs * b[i];
            }
        }
    }
#pragma unroll
    for (int k = L; k < 64; k *= 2)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += __shfl_xor(x[i], k);
    if (lane == 0) p.lse[row] = top == -INFINITY && total == 0.0f ? -INFINITY : LN2 * (top + __builtin_amdgcn_logf(total));
    if (lane >= L || cc * 8 >= p.D) return;
    const float g = total > 0.0f ? 1.0f / total : (total == 0.0f ? 0.0f : total);
    typename type_of<E>::v8 e;
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = (E) (x[i] * g);
    *reinterpret_cast<typename type_of<E>::v8 *>(p.out.data + (int64_t) tok * p.out.ts + head * p.out.hs + cc * 16) = e;
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float dot8(v8b a, v8b b) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) s = __builtin_amdgcn_fdot2_f32_bf16(v2b{a[i], a[i + 1]}, v2b{b[i], b[i + 1]}, s, false);
    return s;
}
__device__ __forceinline__ float dot8(v8h a, v8h b) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) s = __builtin_amdgcn_fdot2(v2h{a[i], a[i + 1]}, v2h{b[i], b[i + 1]}, s, false);
    return s;
}

// A query of at most EXACT_KEYS keys takes delta from the definition, the sum of P dP over them, not from `out`, whose rounding
// would stay in its gradients: dS = P (dP - delta) cancels the more, the fewer the keys (nothing is left of one), and few
// keys make the largest dS. With 3 keys a query dQ and dK are off by 0.0024 of their norm so, by 0.0032 from out (bf16, of which
// the rounding of dS and of the result make 0.0024); with 17 by 0.0024 and 0.0025. It costs 2 us of 8 with 8 x 1,024 tokens
// in a band, 4 of 28 with 32 documents, where the queries of more keys only have their documents looked up.
constexpr int EXACT_KEYS = 16;
// Documents whose offsets the delta kernel's workgroups hold; those of more are looked up in memory.
constexpr int DELTA_DOCS = 1024;

// The largest d with cu[d] <= t.
__device__ __forceinline__ int doc_of_token(const int32_t * cu, int n_seqs, int T, int t) {
    int lo = 0, hi = n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (offset(cu, mid, T) <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// -delta = -sum(dout out) and log2 of the sums of each (token, head) row. L lanes a row (8 for heads of up to 64). Bound by
// HBM: 32,900 tokens of 16 heads of 64, 135 MB, 33 us, 4.1 TB/s (28.5 without the look-up).
template <class E, int L>
__global__ __launch_bounds__(1024) void attn_rows_delta_kernel(attn_p p) {
    typedef typename type_of<E>::v8 v8;
    constexpr int ROWS = 1024 / L;
    const int cc = threadIdx.x % L, sub = threadIdx.x / L;
    auto sum = [](float x) {
#pragma unroll
        for (int k = L / 2; k; k >>= 1) x += __shfl_xor(x, k, L);
        return x;
    };
    const int q_lo = offset(p.cu_q, 0, p.T_q), q_hi = offset(p.cu_q, p.n_seqs, p.T_q);
    __shared__ int32_t s_cu[2][DELTA_DOCS + 1];
    const bool held = p.n_seqs <= DELTA_DOCS;
    if (held) {
        for (int i = threadIdx.x; i <= p.n_seqs; i += 1024) {
            s_cu[0][i] = p.cu_q[i];
            s_cu[1][i] = p.cu_k[i];
        }
        __syncthreads();
    }
    const int32_t * cu_q = held ? s_cu[0] : p.cu_q, * cu_k = held ? s_cu[1] : p.cu_k;
    const float cs = p.scale * LOG2E;
    // up to 63 documents' offsets a lane each: may a query of the tokens ta .. tb have few keys? (Their number rises, stays
    // and falls over a document, so that its ends tell.)
    const int lane = threadIdx.x & 63;
    const int lane_q = held ? offset(cu_q, min(lane, p.n_seqs), p.T_q) : 0, lane_k = held ? offset(cu_k, min(lane, p.n_seqs), p.T_k) : 0;
    auto few_keys = [&](int ta, int tb) {
        if (p.n_seqs > 63) return true;
        const int d = __popcll(__ballot(lane <= p.n_seqs && lane_q <= ta)) - 1;
        if (d < 0 || d >= p.n_seqs) return true;
        doc c;
        c.q0 = __builtin_amdgcn_readlane(lane_q, d);
        c.n = __builtin_amdgcn_readlane(lane_q, d + 1) - c.q0;
        c.k0 = __builtin_amdgcn_readlane(lane_k, d);
        c.m = max(__builtin_amdgcn_readlane(lane_k, d + 1) - c.k0, 0);
        if (tb >= c.q0 + c.n) return true;
        const int a = ta - c.q0, b = tb - c.q0;
        return min(key_hi(p, c, a) - key_lo(p, c, a), key_hi(p, c, b) - key_lo(p, c, b)) <= EXACT_KEYS;
    };
    // in the order of lse2 and ndelta, a KV head's pairs one after another; two rows at a time under way
    const int n_pairs = p.T_q * p.R, all = p.G * ((n_pairs + 2 * ROWS - 1) / (2 * ROWS));
    for (int w = blockIdx.x; w < all; w += gridDim.x) {
        const int g = w % p.G, p0 = w / p.G * (2 * ROWS) + sub;
        v8 a[2] = {}, b[2] = {};
        int64_t at[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int pr = p0 + ROWS * k;
            at[k] = -1;
            if (pr >= n_pairs) continue;
            const int64_t tok = pr / p.R, head = g * p.R + pr % p.R;
            at[k] = tok * p.H + head;
            if (cc * 8 < p.D) {
                a[k] = *reinterpret_cast<const v8 *>(p.dout.data + tok * p.dout.ts + head * p.dout.hs + cc * 16);
                b[k] = *reinterpret_cast<const v8 *>(p.out.data + tok * p.out.ts + head * p.out.hs + cc * 16);
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int pw = uni(p0 + ROWS * k);
            const bool few = pw < n_pairs && few_keys(pw / p.R, (min(pw + 64 / L, n_pairs) - 1) / p.R);
            if (at[k] < 0) continue;          // a row's lanes alike
            float s = 0.0f;
            if (cc * 8 < p.D) {
#pragma unroll
                for (int i = 0; i < 8; ++i) s += (float) a[k][i] * (float) b[k][i];
            }
            s = sum(s);
            const int tok = (p0 + ROWS * k) / p.R;
            const float lse2 = p.lse[at[k]] * LOG2E;
            if (few && tok >= q_lo && tok < q_hi) {
                const int d = doc_of_token(cu_q, p.n_seqs, p.T_q, tok);
                doc c;
                c.q0 = offset(cu_q, d, p.T_q);
                c.n = max(offset(cu_q, d + 1, p.T_q) - c.q0, 0);
                c.k0 = offset(cu_k, d, p.T_k);
                c.m = max(offset(cu_k, d + 1, p.T_k) - c.k0, 0);
                const int lo = key_lo(p, c, tok - c.q0), hi = key_hi(p, c, tok - c.q0);
                if (hi > lo && hi - lo <= EXACT_KEYS) {
                    const int head = (int) (at[k] - (int64_t) tok * p.H);
                    v8 x = {};
                    if (cc * 8 < p.D) x = *reinterpret_cast<const v8 *>(p.q.data + (int64_t) tok * p.q.ts + head * p.q.hs + cc * 16);
                    s = 0.0f;
                    constexpr int AT = 2;                 // keys whose loads are under way together
                    for (int j = lo; j < hi; j += AT) {
                        v8 y[AT] = {}, z[AT] = {};
                        if (cc * 8 < p.D) {
#pragma unroll
                            for (int i = 0; i < AT; ++i) {
                                const int64_t key = c.k0 + min(j + i, hi - 1);
                                y[i] = *reinterpret_cast<const v8 *>(p.k.data + key * p.k.ts + g * p.k.hs + cc * 16);
                                z[i] = *reinterpret_cast<const v8 *>(p.v.data + key * p.v.ts + g * p.v.hs + cc * 16);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < AT; ++i) {
                            const float t = __builtin_amdgcn_exp2f(__builtin_fmaf(sum(dot8(x, y[i])), cs, -lse2)) * sum(dot8(a[k], z[i]));
                            if (j + i < hi) s += t;
                        }
                    }
                }
            }
            if (cc == 0) {
                const int64_t row = (int64_t) g * n_pairs + p0 + ROWS * k;
                p.lse2[row] = lse2 - (type_of<E>::HALF ? P_SHIFT : 0);
                p.ndelta[row] = -s;
            }
        }
    }
}

// fp16: takes 2^15 dS to what is carried, f times that, within the type: where the lane's largest value is past DS_TOP, f and the
// sum so far are lowered by a power of two, for both half waves of the column alike. So a row's small dS lose bits only
// beside its own large ones (2^-34 of the largest at most), whatever other rows hold. Values that are not finite stay as
// they are. Against one power of two for the launch, from the largest norms: 32 documents full 781 -> 818 us, 8,192 tokens causal
// of 128 values a head 1,038 -> 1,045, 64 documents of 100 tokens 55 -> 50 (no norms to take).
template <int DT>
__device__ __forceinline__ void place_ds(v16f & ds, float & f, v16f (&sum)[DT]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        ds[i] *= f;
        m = fmaxf(m, fabsf(ds[i]));
    }
    if (!__any(!(m <= DS_TOP))) return;
    m = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(ds[i]) < INFINITY ? fabsf(ds[i]) : 0.0f);
    m = half_max(m);
    const float lower = m > DS_TOP ? ldexpf(1.0f, DS_PLACE - __builtin_amdgcn_frexp_expf(m)) : 1.0f;
    f *= lower;
#pragma unroll
    for (int i = 0; i < 16; ++i) ds[i] *= lower;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[d][i] *= lower;
}
// What turns a sum of carried dS into one of dS.
template <class E>
__device__ __forceinline__ float ds_unit(float f) { return type_of<E>::HALF ? 1.0f / ldexpf(f, P_SHIFT) : 1.0f; }

// dQ: the forward pass's tiling. dQ^T = scale K^T dS^T.
template <class E, int DT>
__device__ __forceinline__ void dq_tile(v16f (&dq)[DT], const typename type_of<E>::v8 (&q)[2 * DT],
                                        const typename type_of<E>::v8 (&go)[2 * DT], lane_at at, uint32_t kt, uint32_t vt, float c,
                                        float lse2, float ndelta, float & f, int sides, int lo, int hi) {
    typedef type_of<E> TY;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        v16f s = {}, dp = {};
#pragma unroll
        for (int d = 0; d < 2 * DT; ++d) s = TY::mfma(row_operand<E, DT>(kt + at.row, 32 * a, d), q[d], s);
#pragma unroll
        for (int d = 0; d < 2 * DT; ++d) dp = TY::mfma(row_operand<E, DT>(vt + at.row, 32 * a, d), go[d], dp);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -lse2));
            s[i] = pr * (dp[i] + ndelta);
        }
        if (sides) mask_rows(s, sides, lo - 32 * a, hi - 32 * a, 0.0f);
        if constexpr (TY::HALF) place_ds<DT>(s, f, dq);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const typename TY::v8 ds = pack<E>(s, b);
#pragma unroll
            for (int d = 0; d < DT; ++d) dq[d] = TY::mfma(col_operand<E, DT>(kt + at.col, 32 * a + 16 * b, d), ds, dq[d]);
        }
    }
}

// P and dS of a pair and a key from the definition.
struct weights {
    float p, ds;
};
template <class E>
__device__ __forceinline__ weights weights_of(const attn_p & p, const doc & c, int g, int pair, const char * k, const char * v) {
    const int tok = pair / p.R, head = g * p.R + pair % p.R;
    const int64_t row = ((int64_t) g * p.T_q + c.q0) * p.R + pair;
    const char * q = p.q.data + (c.q0 + tok) * p.q.ts + head * p.q.hs, * d = p.dout.data + (c.q0 + tok) * p.dout.ts + head * p.dout.hs;
    weights w;
    w.p = __builtin_amdgcn_exp2f(dot<E>(q, k, p.D) * p.scale * LOG2E - (p.lse2[row] + (type_of<E>::HALF ? P_SHIFT : 0)));
    w.ds = w.p * (dot<E>(d, v, p.D) + p.ndelta[row]);
    return w;
}
template <class E, class K, class V>
__device__ __forceinline__ void add_ds(float (&x)[2], const attn_p & p, const doc & c, int g, int pair, int lo, int hi, float * lds, K k_row, V v_row) {
    add_rows<E>(x, lo, hi, p.D, lds, [&](int j) { return weights_of<E>(p, c, g, pair, k_row(j), v_row(j)).ds; }, k_row);
}

// The tiles of 64 keys that the 128 pairs from p0 see some of, and of 64 pairs that see some of the 128 keys from kb0.
__device__ __forceinline__ span keys_of(const attn_p & p, const doc & c, int p0) {
    const int t_end = (min(p0 + 128, c.n * p.R) - 1) / p.R;
    return {key_lo(p, c, p0 / p.R) / 64, (key_hi(p, c, t_end) + 63) / 64};
}
__device__ __forceinline__ span pairs_of(const attn_p & p, const doc & c, int kb0) {
    const int k_end = min(kb0 + 128, c.m) - 1;
    return {tok_lo(p, c, kb0) * p.R / 64, (tok_hi(p, c, k_end) * p.R + 63) / 64};
}

// dQ: a workgroup has 128 pairs, a wave 32 of them with q and dout in registers, and goes over the keys that they see, 64 at a
// time: S^T = K Q^T and dP^T = V dO^T from the tiles' rows, dQ^T += K^T dS^T from K's columns. P and dS are computed here again
// rather than shared with dK and dV, whose sums over pairs would need atomics, in no fixed order.
template <class E, int DT>
struct dq_lds {
    E sk[2][64 * SP<DT>], sv[2][64 * SP<DT>];
};
template <class E, int DT>
__device__ __forceinline__ void dq_workgroup(const attn_p & p, int block, dq_lds<E, DT> & lds, int * s_job) {
    constexpr int BM = 128, BN = 64;
    auto & sk = lds.sk;
    auto & sv = lds.sv;
    const int g = block % p.G, split = block / p.G % p.split_q;
    const job todo = workgroup_job(p, false, p.R, BM, block / (p.G * p.split_q), p.right >= 0 ? p.order == BY_ROWS : p.left >= 0 && p.order != BY_ROWS, s_job);
    if (todo.tile < 0) return;
    const doc c = todo.c;
    const int np = c.n * p.R, p0 = todo.tile * BM;

    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int pw = p0 + 32 * wave;
    const bool active = pw < np;
    const int pc = min(pw + (lane & 31), np - 1), tok = pc / p.R, head = g * p.R + pc % p.R;

    const int lo = key_lo(p, c, tok), hi = key_hi(p, c, tok);
    const span mine = split_of(keys_of(p, c, p0), p.split_q, split);
    const int j_lo = uni(mine.lo), j_hi = uni(mine.hi);
    if (p.split_q > 1 && j_lo >= j_hi) return;
    const int ta = uni(min(pw, np - 1) / p.R), tb = uni(min(pw + 31, np - 1) / p.R);
    const int some_lo = key_lo(p, c, ta), some_hi = key_hi(p, c, tb), all_lo = key_lo(p, c, tb), all_hi = key_hi(p, c, ta);

    key_stream<DT, BN, 256> keys(p, c, g, j_lo * BN, BN);
    if (p.D != 32 * DT) {
        clear(sk, sizeof(sk), threadIdx.x, 256);
        clear(sv, sizeof(sv), threadIdx.x, 256);
        barrier();
    }
    v16f dq[DT];
#pragma unroll
    for (int k = 0; k < DT; ++k) dq[k] = v16f{};
    const float cs = p.scale * LOG2E;
    const lane_at at = lane_places<DT>();
    if (j_lo < j_hi) keys.next(lds_addr(sk[0]), lds_addr(sv[0]));
    typename type_of<E>::v8 q[2 * DT], go[2 * DT];
    load_operands<E, DT>(q, p.q.data + (c.q0 + tok) * p.q.ts + head * p.q.hs, go, p.dout.data + (c.q0 + tok) * p.dout.ts + head * p.dout.hs, p.D);
    const int64_t row = ((int64_t) g * p.T_q + c.q0) * p.R + pc;
    float f = DS_START;
    float lse2 = p.lse2[row], ndelta = p.ndelta[row];
    asm volatile("" : "+v"(lse2), "+v"(ndelta));
    for (int j = j_lo; j < j_hi; ++j) {
        const int buf = (j - j_lo) & 1, j0 = j * BN;
        wait_all();
        barrier();
        if (j + 1 < j_hi) keys.next(lds_addr(sk[buf ^ 1]), lds_addr(sv[buf ^ 1]));
        if (!active || j0 >= some_hi || j0 + BN <= some_lo) continue;
        dq_tile<E, DT>(dq, q, go, at, lds_addr(sk[buf]), lds_addr(sv[buf]), cs, lse2, ndelta, f, (j0 < all_lo ? 1 : 0) | (j0 + BN > all_hi ? 2 : 0), lo - j0, hi - j0);
    }
    barrier();
    if (!active) return;
    E * tile = (wave < 2 ? sk[0] : sv[0]) + (wave & 1) * 32 * SP<DT>;
    uint32_t bad = bad_columns<DT>(dq);
    float * part = p.part_q + (((int64_t) split * p.G + g) * p.T_q + c.q0) * p.R * p.D;
    if (p.split_q > 1) {
        store_partial<DT>(dq, p.scale * ds_unit<E>(f), p.D, np - pw, part + (int64_t) pw * p.D);
    } else {
        store_columns<E, DT>(tile, dq, p.scale * ds_unit<E>(f), p.D, [&](int r) -> char * {
            const int pr = pw + r;
            if (pr >= np) return nullptr;
            return p.dq.data + (int64_t) (c.q0 + pr / p.R) * p.dq.ts + (g * p.R + pr % p.R) * p.dq.hs;
        });
    }
    if (!bad) return;
    auto k_row = [&](int j) { return p.k.data + (int64_t) (c.k0 + j) * p.k.ts + g * p.k.hs; };
    auto v_row = [&](int j) { return p.v.data + (int64_t) (c.k0 + j) * p.v.ts + g * p.v.hs; };
    if (!holds_bad<E>(j_lo * BN, min(all_lo, c.m), p.D, k_row) && !holds_bad<E>(max(all_hi, 0), min(j_hi * BN, c.m), p.D, k_row)) return;
    for (; bad; bad &= bad - 1) {
        const int pair = pw + __builtin_ctz(bad);
        if (pair >= np) break;
        float x[2] = {0.0f, 0.0f};
        const int t = pair / p.R;
        add_ds<E>(x, p, c, g, pair, max(key_lo(p, c, t), j_lo * BN), min(key_hi(p, c, t), j_hi * BN), reinterpret_cast<float *>(tile), k_row, v_row);
        if (p.split_q > 1) store_row<float>((char *) (part + (int64_t) pair * p.D), x, p.scale, p.D);
        else store_row<E>(p.dq.data + (int64_t) (c.q0 + t) * p.dq.ts + (g * p.R + pair % p.R) * p.dq.hs, x, p.scale, p.D);
    }
}

// Ends a phase of N products of one LDS read each, with two reads ahead of the products: more would not
// fit the registers.
template <int N>
__device__ __forceinline__ void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
    for (int i = 0; i < N - 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
    __builtin_amdgcn_sched_barrier(0);
}

// dK, dV: a wave has 32 keys, the workgroup goes over the pairs that see its 128, 64 at a time, a wave 32 at a
// time: qt, ot their rows of q and dout, lse2, ndelta (LDS addresses as well) their sums, pairs lo .. hi - 1 of them seen by the key.
template <class E, int DT>
__device__ __forceinline__ void dkv_tile(v16f (&dk)[DT], v16f (&dv)[DT], const typename type_of<E>::v8 (&k)[2 * DT],
                                         const typename type_of<E>::v8 (&v)[2 * DT], lane_at at, uint32_t qt, uint32_t ot,
                                         uint32_t lse2, uint32_t ndelta, float c, float & f, int sides, int lo, int hi) {
    typedef type_of<E> TY;
    typedef __attribute__((address_space(3))) v4f lds_v4f;
    const uint32_t h16 = (threadIdx.x & 32) >> 1;      // 4 values for the second half wave
    v16f s = {}, dp;
#pragma unroll
    for (int d = 0; d < 2 * DT; ++d) s = TY::mfma(row_operand<E, DT>(qt + at.row, 0, d), k[d], s);
    if (DT >= 3) reads_ahead<2 * DT>();
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {              // dP - delta: the sums start there
        const v4f de = *(lds_v4f *) (uintptr_t) (ndelta + h16 + 32 * i4);
#pragma unroll
        for (int j = 0; j < 4; ++j) dp[4 * i4 + j] = de[j];
    }
#pragma unroll
    for (int d = 0; d < 2 * DT; ++d) dp = TY::mfma(row_operand<E, DT>(ot + at.row, 0, d), v[d], dp);
    if (DT >= 3) reads_ahead<2 * DT>();
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
        const v4f ls = *(lds_v4f *) (uintptr_t) (lse2 + h16 + 32 * i4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = 4 * i4 + j;
            s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -ls[j]));
            dp[i] *= s[i];
        }
    }
    if (sides) {
        mask_rows(s, sides, lo, hi, 0.0f);
        mask_rows(dp, sides, lo, hi, 0.0f);
    }
    if constexpr (TY::HALF) place_ds<DT>(dp, f, dk);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const typename TY::v8 pp = pack<E>(s, b), ds = pack<E>(dp, b);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            dv[d] = TY::mfma(col_operand<E, DT>(ot + at.col, 16 * b, d), pp, dv[d]);
            dk[d] = TY::mfma(col_operand<E, DT>(qt + at.col, 16 * b, d), ds, dk[d]);
        }
    }
}

// A workgroup: 128 keys, 4 waves of 32 with k and v in registers; tiles of q and dout are read in rows for S and dP, in columns for
// dV += dO^T P and dK += Q^T dS: four products a tile, the other operand of each matrix instruction read from LDS.
template <class E, int DT>
struct dkv_lds {
    E sq[2][64 * SP<DT>], so[2][64 * SP<DT>];
    float s_lse[2][64], s_delta[2][64];
};
template <class E, int DT>
__device__ __forceinline__ void dkv_workgroup(const attn_p & p, int block, dkv_lds<E, DT> & lds, int * s_job) {
    constexpr int BK = 128, BQ = 64;
    auto & sq = lds.sq;
    auto & so = lds.so;
    auto & s_lse = lds.s_lse;
    auto & s_delta = lds.s_delta;
    const int g = block % p.G, split = block / p.G % p.split_kv;
    const job todo = workgroup_job(p, true, 1, BK, block / (p.G * p.split_kv), p.right >= 0 && p.order != BY_ROWS, s_job);
    if (todo.tile < 0) return;
    const doc c = todo.c;
    const int np = c.n * p.R, kb0 = todo.tile * BK;

    const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int kw = kb0 + 32 * wave;
    const bool active = kw < c.m;
    const int key = min(kw + (lane & 31), c.m - 1);

    const span mine = split_of(pairs_of(p, c, kb0), p.split_kv, split);
    const int j_lo = uni(mine.lo), j_hi = uni(mine.hi);
    if (p.split_kv > 1 && j_lo >= j_hi) return;
    const int ka = uni(min(kw, c.m - 1)), ke = uni(min(kw + 31, c.m - 1));
    const int some_lo = tok_lo(p, c, ka) * p.R, some_hi = tok_hi(p, c, ke) * p.R;
    const int all_lo = tok_lo(p, c, ke) * p.R, all_hi = tok_hi(p, c, ka) * p.R;

    tile_loader<DT, BQ, 256> lq(p.D), l_out(p.D);
    lq.pairs_at(p.R, p.q.ts, p.q.hs);
    l_out.pairs_at(p.R, p.dout.ts, p.dout.hs);
    if (p.D != 32 * DT) {
        clear(sq, sizeof(sq), threadIdx.x, 256);
        clear(so, sizeof(so), threadIdx.x, 256);
        barrier();
    }
    auto load = [&](int j, int buf) {
        const int j0 = j * BQ;
        if (p.near_q && !p.even_q && j0 + BQ <= np) {
            const int t0 = j0 / p.R, r0 = j0 - t0 * p.R;
            lq.load_pairs(uni(p.q.data + (int64_t) (c.q0 + t0) * p.q.ts + g * p.R * p.q.hs), r0, p.R, p.by_R, (uint32_t) p.q.ts, (uint32_t) p.q.hs, lds_addr(sq[buf]));
            l_out.load_pairs(uni(p.dout.data + (int64_t) (c.q0 + t0) * p.dout.ts + g * p.R * p.dout.hs), r0, p.R, p.by_R, (uint32_t) p.dout.ts, (uint32_t) p.dout.hs, lds_addr(so[buf]));
        } else if (p.near_q && j0 + BQ <= np) {
            lq.load(uni(p.q.data + (int64_t) (c.q0 + j0 / p.R) * p.q.ts + g * p.R * p.q.hs), lds_addr(sq[buf]));
            l_out.load(uni(p.dout.data + (int64_t) (c.q0 + j0 / p.R) * p.dout.ts + g * p.R * p.dout.hs), lds_addr(so[buf]));
        } else {
            auto at = [&](const rows & x, int r) -> const char * {
                const int pr = j0 + r;
                return pr < np ? x.data + (int64_t) (c.q0 + pr / p.R) * x.ts + (g * p.R + pr % p.R) * x.hs : nullptr;
            };
            lq.load_each(lds_addr(sq[buf]), [&](int r) { return at(p.q, r); });
            l_out.load_each(lds_addr(so[buf]), [&](int r) { return at(p.dout, r); });
        }
        // the pairs' sums, by waves 0 and 1 (behind the document: whatever is there, masked)
        if (wave < 2) {
            int t = threadIdx.x;
            asm volatile("" : "+v"(t));
            const float * from = (wave ? p.ndelta : p.lse2) + ((int64_t) g * p.T_q + c.q0) * p.R + j0;
            dma4s(uni((const char *) from), (t & 63) * 4, lds_addr(wave ? s_delta[buf] : s_lse[buf]));
        }
    };
    v16f dk[DT], dv[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) dk[i] = dv[i] = v16f{};
    const float cs = p.scale * LOG2E;
    const lane_at at = lane_places<DT>();
    if (j_lo < j_hi) load(j_lo, 0);
    typename type_of<E>::v8 k[2 * DT], v[2 * DT];
    load_operands<E, DT>(k, p.k.data + (int64_t) (c.k0 + key) * p.k.ts + g * p.k.hs, v, p.v.data + (int64_t) (c.k0 + key) * p.v.ts + g * p.v.hs, p.D);
    float f = DS_START;
    for (int j = j_lo; j < j_hi; ++j) {
        const int buf = (j - j_lo) & 1, j0 = j * BQ;
        wait_all();
        barrier();
        if (j + 1 < j_hi) load(j + 1, buf ^ 1);
        if (active && j0 < some_hi && j0 + BQ > some_lo) {
            const int sides = (j0 < all_lo ? 1 : 0) | (j0 + BQ > all_hi ? 2 : 0);
            int lo = 0, hi = 0;
            if (sides) {               // few tiles: the lane's bounds are not kept in registers
                int t = threadIdx.x;
                asm volatile("" : "+v"(t));
                const int j = min(kw + (t & 31), c.m - 1);
                lo = tok_lo(p, c, j) * p.R - j0;
                hi = tok_hi(p, c, j) * p.R - j0;
            }
#pragma unroll 1
            for (int a = 0; a < BQ; a += 32) {
                dkv_tile<E, DT>(dk, dv, k, v, at, lds_addr(sq[buf]) + a * SP<DT> * 2, lds_addr(so[buf]) + a * SP<DT> * 2, lds_addr(s_lse[buf]) + 4 * a,
                                lds_addr(s_delta[buf]) + 4 * a, cs, f, sides, lo - a, hi - a);
            }
        }
    }
    barrier();
    if (!active) return;
    E * tile = (wave < 2 ? sq[0] : so[0]) + (wave & 1) * 32 * SP<DT>;
    auto dst = [&](const rows & x) {
        return [&, x](int r) -> char * { return kw + r < c.m ? x.data + (int64_t) (c.k0 + kw + r) * x.ts + g * x.hs : nullptr; };
    };
    uint32_t bad = bad_columns<DT>(dv) | bad_columns<DT>(dk);
    const int64_t part_v = (int64_t) p.G * p.T_k * p.D;
    float * part = p.part_kv + 2 * split * part_v + ((int64_t) g * p.T_k + c.k0) * p.D;
    if (p.split_kv > 1) {
        store_partial<DT>(dv, type_of<E>::HALF ? 1.0f / (1 << P_SHIFT) : 1.0f, p.D, c.m - kw, part + part_v + (int64_t) kw * p.D);
        store_partial<DT>(dk, p.scale * ds_unit<E>(f), p.D, c.m - kw, part + (int64_t) kw * p.D);
    } else {
        store_columns<E, DT>(tile, dv, type_of<E>::HALF ? 1.0f / (1 << P_SHIFT) : 1.0f, p.D, dst(p.dv));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        store_columns<E, DT>(tile, dk, p.scale * ds_unit<E>(f), p.D, dst(p.dk));
    }
    if (!bad) return;
    auto pair_row = [&](const rows & x) {
        return [&, x](int pr) { return (const char *) x.data + (int64_t) (c.q0 + pr / p.R) * x.ts + (g * p.R + pr % p.R) * x.hs; };
    };
    const int a0 = j_lo * BQ, a1 = min(all_lo, np), b0 = max(all_hi, 0), b1 = min(j_hi * BQ, np);
    if (!holds_bad<E>(a0, a1, p.D, pair_row(p.q)) && !holds_bad<E>(a0, a1, p.D, pair_row(p.dout)) &&
        !holds_bad<E>(b0, b1, p.D, pair_row(p.q)) && !holds_bad<E>(b0, b1, p.D, pair_row(p.dout))) return;
    for (; bad; bad &= bad - 1) {
        const int j = kw + __builtin_ctz(bad);
        if (j >= c.m) break;
        const char * k_row = p.k.data + (int64_t) (c.k0 + j) * p.k.ts + g * p.k.hs, * v_row = p.v.data + (int64_t) (c.k0 + j) * p.v.ts + g * p.v.hs;
        const int lo = max(tok_lo(p, c, j) * p.R, j_lo * BQ), hi = min(tok_hi(p, c, j) * p.R, j_hi * BQ);
        float x[2] = {0.0f, 0.0f}, y[2] = {0.0f, 0.0f};
        add_rows<E>(x, lo, hi, p.D, reinterpret_cast<float *>(tile), [&](int pr) { return weights_of<E>(p, c, g, pr, k_row, v_row).p; }, pair_row(p.dout));
        add_rows<E>(y, lo, hi, p.D, reinterpret_cast<float *>(tile), [&](int pr) { return weights_of<E>(p, c, g, pr, k_row, v_row).ds; }, pair_row(p.q));
        if (p.split_kv > 1) {
            store_row<float>((char *) (part + part_v + (int64_t) j * p.D), x, 1.0f, p.D);
            store_row<float>((char *) (part + (int64_t) j * p.D), y, p.scale, p.D);
        } else {
            store_row<E>(p.dv.data + (int64_t) (c.k0 + j) * p.dv.ts + g * p.dv.hs, x, 1.0f, p.D);
            store_row<E>(p.dk.data + (int64_t) (c.k0 + j) * p.dk.ts + g * p.dk.hs, y, p.scale, p.D);
        }
    }
}

// Both in one launch, dK and dV's workgroups first (they are the longer ones), so that the end of the one is
// filled by the others: against a launch each, 8 x 1,024 tokens banded 71 -> 58 us, one document of 8,192 causal
// 720 -> 535 us (64 values a head) and 1,176 -> 1,037 (128).
//
// Bound by the matrix units with the exponentials and the LDS reads between them (the products of one wave wait for
// each other; two workgroups' waves a CU fill part of that): of the five products that the gradients need (seven are
// taken, S and dP on both sides), 8,192 tokens full, 16 heads of 64 on 8: 975 us, 705 TFLOP/s, 987 with the two taken twice;
// 128 values a head 1,715 us, 802. Taking P for the next tile beside dP of this (841 against 759 us), V's tile in LDS, and
// other priorities of the waves were no faster.
template <class E, int DT>
__global__ __launch_bounds__(256, 2) void attn_rows_grad_kernel(attn_p p, int n_dkv, int order_dq) {
    __shared__ __align__(1024) union {
        dq_lds<E, DT> dq;
        dkv_lds<E, DT> dkv;
    } lds;
    __shared__ int s_job[8];
    if ((int) blockIdx.x < n_dkv) {
        dkv_workgroup<E, DT>(p, blockIdx.x, lds.dkv, s_job);
    } else {
        p.order = order_dq;
        dq_workgroup<E, DT>(p, blockIdx.x - n_dkv, lds.dq, s_job);
    }
}

// The splits' shares of the gradients joined, a workgroup a tile of them: the first n_kv workgroups dK and dV, the
// others dQ. Summed in the splits' order. Bound by the shares' reads: 2,048 tokens, 16 heads of 64 on 8, in three and two
// shares 6.6 us.
template <class E>
__global__ __launch_bounds__(1024) void attn_rows_grad_join_kernel(attn_p p, int n_kv) {
    const int chunks = p.D / 8;
    auto sum = [&](const float * from, int64_t step, int n, char * to) {
        float x[8] = {};
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
            const v4f a = *reinterpret_cast<const v4f *>(from + k * step), b = *reinterpret_cast<const v4f *>(from + k * step + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] += a[i];
                x[4 + i] += b[i];
            }
        }
        typename type_of<E>::v8 e;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = (E) x[i];
        *reinterpret_cast<typename type_of<E>::v8 *>(to) = e;
    };
    const bool kv = (int) blockIdx.x < n_kv;
    const int block = kv ? blockIdx.x : blockIdx.x - n_kv, g = block % p.G;
    const job todo = find_job(p, kv, kv ? 1 : p.R, 128, block / p.G, BY_ROWS, false);
    if (todo.tile < 0) return;
    const doc c = todo.c;
    const int first = todo.tile * 128, rows_here = min(128, (kv ? c.m : c.n * p.R) - first), n_split = kv ? p.split_kv : p.split_q;
    const span all = kv ? pairs_of(p, c, first) : keys_of(p, c, first);
    const int share = share_of(all, n_split), n = share ? (all.hi - all.lo + share - 1) / share : 0;
    if (kv) {
        const int64_t part_v = (int64_t) p.G * p.T_k * p.D;
        for (int i = threadIdx.x; i < 2 * rows_here * chunks; i += 1024) {
            const int which = i >= rows_here * chunks, at = i - which * rows_here * chunks, row = c.k0 + first + at / chunks, d = at % chunks * 8;
            const rows & to = which ? p.dv : p.dk;
            sum(p.part_kv + which * part_v + ((int64_t) g * p.T_k + row) * p.D + d, 2 * part_v, n, to.data + row * to.ts + g * to.hs + 2 * d);
        }
    } else {
        const int64_t part_g = (int64_t) p.T_q * p.R * p.D;
        for (int i = threadIdx.x; i < rows_here * chunks; i += 1024) {
            const int pair = first + i / chunks, d = i % chunks * 8;
            sum(p.part_q + g * part_g + ((int64_t) c.q0 * p.R + pair) * p.D + d, p.G * part_g, n,
                p.dq.data + (int64_t) (c.q0 + pair / p.R) * p.dq.ts + (g * p.R + pair % p.R) * p.dq.hs + 2 * d);
        }
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

int64_t slots(int64_t T, int64_t mul, int64_t tile, int64_t n_seqs) { return T * mul / tile + n_seqs; }

constexpr int64_t MAX_T = 1 << 30;
constexpr int MAX_R = 1 << 16;                 // the pieces of 128 tokens' pairs fit 32 bits
constexpr int64_t MAX_GRID = (1 << 24) - 1;    // workgroups of a launch: less than 2^32 threads

int32_t check_params(const char * what, const nxg_attention_rows_params * a, attn_p & p) {
    if (!a) return nxg_fail(NXG_EINVAL, "%s: null parameters", what);
    if (a->type != NXG_TYPE_F16 && a->type != NXG_TYPE_BF16) {
        return nxg_fail(NXG_EINVAL, "%s: type %d (rows must be F16 or BF16)", what, a->type);
    }
    if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8) {
        return nxg_fail(NXG_EINVAL, "%s: head_dim=%d (a multiple of 8 up to 128)", what, a->head_dim);
    }
    if (a->n_head < 1 || a->n_kv_head < 1 || a->n_head % a->n_kv_head) {
        return nxg_fail(NXG_EINVAL, "%s: n_head=%d n_kv_head=%d", what, a->n_head, a->n_kv_head);
    }
    if (a->n_head / a->n_kv_head > MAX_R) return nxg_fail(NXG_EINVAL, "%s: n_head=%d n_kv_head=%d (up to %d to one)", what, a->n_head, a->n_kv_head, MAX_R);
    if (a->T_q < 0 || a->T_k < 0 || a->n_seqs < 0 || a->T_q > MAX_T || a->T_k > MAX_T) {
        return nxg_fail(NXG_EINVAL, "%s: T_q=%d T_k=%d n_seqs=%d", what, a->T_q, a->T_k, a->n_seqs);
    }
    if (a->left < -1 || a->right < -1) return nxg_fail(NXG_EINVAL, "%s: left=%d right=%d (-1: no limit)", what, a->left, a->right);
    if (!(a->scale > 0.0f) || !(a->scale < INFINITY)) return nxg_fail(NXG_EINVAL, "%s: scale must be positive and finite", what);
    p = attn_p{};
    p.H = a->n_head;
    p.G = a->n_kv_head;
    p.R = p.H / p.G;
    p.D = a->head_dim;
    p.T_q = a->T_q;
    p.T_k = a->T_k;
    p.n_seqs = a->n_seqs;
    p.left = std::min(a->left, (int32_t) MAX_T - 1);
    p.right = std::min(a->right, (int32_t) MAX_T - 1);
    p.scale = a->scale;
    p.cu_q = a->cu_q;
    p.cu_k = a->cu_k;
    if ((int64_t) p.T_q * p.H > INT32_MAX - 256 || (int64_t) p.T_k * p.G > INT32_MAX ||
        (slots(p.T_q, p.R, 128, p.n_seqs) + slots(p.T_k, 1, 128, p.n_seqs)) * p.G > MAX_GRID) {
        return nxg_fail(NXG_EINVAL, "%s: T_q=%d T_k=%d of %d heads is too large", what, p.T_q, p.T_k, p.H);
    }
    p.n_split = 1;
    return NXG_OK;
}

// Whether 64 rows' offsets from the first fit 32 bits: keys one after another, and pairs.
bool near_rows(const rows & x) { return x.ts <= (INT32_MAX - 4096) / 64; }
bool near_pairs(const rows & x, int R) {
    return R <= 1024 && x.ts <= (INT32_MAX - 4096) / 128 && x.hs <= (INT32_MAX - 4096) / 2 / R;
}

int32_t check_rows(const char * what, const char * name, const nxg_rows * x, int64_t T, int n_head, int D, bool written, rows & r) {
    if (T == 0) return NXG_OK;
    if (!x || !x->data) return nxg_fail(NXG_EINVAL, "%s: %s is null", what, name);
    if ((uintptr_t) x->data & 15) return nxg_fail(NXG_EINVAL, "%s: %s must be 16-byte aligned", what, name);
    r.data = (char *) x->data;
    r.ts = T == 1 ? 0 : x->token_stride;
    r.hs = n_head == 1 ? 0 : x->head_stride;
    const int64_t most = INT64_MAX / 16;
    if (r.ts < 0 || r.hs < 0 || r.ts % 8 || r.hs % 8 || r.ts > most / T || r.hs > most / n_head) {
        return nxg_fail(NXG_EINVAL, "%s: %s has strides %lld, %lld (multiples of 8)", what, name, (long long) r.ts, (long long) r.hs);
    }
    if (written) {           // no two rows of an output overlap
        const int64_t in_n = r.hs <= r.ts || T == 1 ? n_head : T, in_s = r.hs <= r.ts || T == 1 ? r.hs : r.ts;
        const int64_t out_n = in_s == r.hs ? T : n_head, out_s = in_s == r.hs ? r.ts : r.hs;
        if ((in_n > 1 && in_s < D) || (out_n > 1 && out_s < (in_n - 1) * in_s + D)) {
            return nxg_fail(NXG_EINVAL, "%s: rows of %s overlap (strides %lld, %lld)", what, name, (long long) r.ts, (long long) r.hs);
        }
    }
    r.ts *= 2;
    r.hs *= 2;
    return NXG_OK;
}

#define NXG_TRY(call) do { const int32_t rc_ = (call); if (rc_) return rc_; } while (0)

// Refuses an output that is another row array of the call.
int32_t check_apart(const char * what, const char * name, const rows & out, std::initializer_list<const rows *> others) {
    for (const rows * r : others) {
        if (out.data && out.data == r->data) return nxg_fail(NXG_EINVAL, "%s: %s is another tensor of the call too", what, name);
    }
    return NXG_OK;
}

// Values of a row array of the backward pass: one a (token, head), and a tile's reach behind the last.
int64_t row_values(const attn_p & p) { return ((int64_t) p.T_q * p.H + 67) / 4 * 4; }
int64_t part_q_values(const attn_p & p) { return p.split_q > 1 ? (int64_t) p.split_q * p.T_q * p.H * p.D : 0; }
int64_t part_kv_values(const attn_p & p) { return p.split_kv > 1 ? (int64_t) p.split_kv * 2 * p.T_k * p.G * p.D : 0; }
int64_t backward_bytes(const attn_p & p) { return (2 * row_values(p) + part_q_values(p) + part_kv_values(p)) * 4; }

// The length that a split is reckoned for, of which only the sum is known here: one document's, two's average, twice
// that of more (mixed lengths: with the average 17 documents of 5 queries over 405 keys take 32 us, so 25).
int64_t long_document(int64_t T, int n_seqs) { return n_seqs <= 2 ? T / std::max(1, n_seqs) : 2 * T / n_seqs; }

// Keys that a window leaves of them for `tokens` queries next to each other, and the other way round.
int64_t within_window(const attn_p & p, int64_t length, int64_t tokens) {
    return p.left >= 0 && p.right >= 0 ? std::min(length, (int64_t) p.left + p.right + tokens) : length;
}

// Where there are few tiles of keys, or of pairs, what each goes over is split until there are two workgroups a CU
// (2,048 tokens causal 107 -> 59 us; four a CU cost more in the join: 2 documents of 1,840 tokens, 32 heads of 128 on 4:
// 200 us with two, 241 with four). Where there are up to two a CU anyhow but documents of mixed lengths, and windows that
// leave their tiles mixed work, in two: the longest document's would be the launch's last (17 documents of 3,700 tokens,
// the longest of 1,700: 204 -> 147 us; not for 11 documents of 260, 45 -> 57). A share is two tiles of 64 at least (a
// document of 750 tokens, 8 heads on one: 104 us with 4, 87 with 2), and fewer than 6 tiles are not shared out
// (5 documents of 410 in a window of 16: 50 -> 56 us).
constexpr int MAX_SPLIT = 16;
void plan_backward(attn_p & p) {
    const int64_t cus = nxg_device_cus(), pairs = within_window(p, long_document(p.T_q, p.n_seqs), 128) * p.R,
                  keys = within_window(p, long_document(p.T_k, p.n_seqs), (128 + p.R - 1) / p.R);
    const bool mixed = p.n_seqs > 1 && (p.left < 0 || p.right < 0);
    auto split = [&](int64_t workgroups, int64_t rows) {
        const int64_t tiles = rows / 64;
        int64_t n = 2 * cus / std::max<int64_t>(1, workgroups);
        if (n == 1 && mixed && tiles >= 24) n = 2;
        return tiles < 6 ? 1 : (int) std::max<int64_t>(1, std::min({n, tiles / 2, (int64_t) MAX_SPLIT}));
    };
    p.split_kv = split(slots(p.T_k, 1, 128, p.n_seqs) * p.G, pairs);
    p.split_q = split(slots(p.T_q, p.R, 128, p.n_seqs) * p.G, keys);
}

// Launches one of a kernel's instances by type and head size.
#define NXG_BY_TYPE(type, D, LAUNCH)                                               \
    do {                                                                           \
        if ((type) == NXG_TYPE_BF16) { typedef __bf16 E; NXG_BY_DIM(D, LAUNCH); }  \
        else { typedef _Float16 E; NXG_BY_DIM(D, LAUNCH); }                        \
    } while (0)
#define NXG_BY_DIM(D, LAUNCH)                                                      \
    do {                                                                           \
        if ((D) <= 32) { constexpr int DT = 1; LAUNCH; }                           \
        else if ((D) <= 64) { constexpr int DT = 2; LAUNCH; }                      \
        else if ((D) <= 96) { constexpr int DT = 3; LAUNCH; }                      \
        else { constexpr int DT = 4; LAUNCH; }                                     \
    } while (0)

// Documents in the order of their rows where the workgroups fit the CUs at once, where there is one
// document or more than a wave has lanes, or where every tile's work is alike.
int work_order(const attn_p & p, int64_t workgroups) {
    if (p.n_seqs < 2 || p.n_seqs > 64 || workgroups <= 2 * nxg_device_cus() || (p.left >= 0 && p.right >= 0)) return BY_ROWS;
    return p.left < 0 && p.right < 0 ? BY_LENGTH : BY_LEVEL;
}

// The few-pairs kernel where tiles of 128 pairs would be nearly empty, or would leave CUs idle and tiles of 32 run in
// one round (two workgroups a CU by LDS with up to 64 values a head, else one: 4 documents of 766 tokens, 8 heads of 96 on
// one, 45 us in three rounds, 19 with tiles of 128; 3 documents of 339 tokens of 64 values, 12 us in one, and 14). Its keys are split until there is a workgroup a CU (more only add sums to join: 8 x 1
// query over 8,192 keys of 128 values 50.0, 54.1 and 63.1 us with one, two and four a CU), 256 keys to each at least.
struct fwd_plan {
    bool few;
    int n_split;
};
fwd_plan plan_forward(const attn_p & p) {
    const int64_t cus = nxg_device_cus(), wgs = slots(p.T_q, p.R, 32, p.n_seqs) * p.G;
    fwd_plan f{false, 1};
    const bool empty_tiles = (int64_t) p.T_q * p.R <= 32LL * p.n_seqs, idle = slots(p.T_q, p.R, 128, p.n_seqs) * p.G < cus;
    if (!empty_tiles && !(idle && wgs <= cus * (p.D <= 64 ? 2 : 1))) return f;
    f.few = true;
    const int64_t keys = within_window(p, long_document(p.T_k, p.n_seqs), (32 + p.R - 1) / p.R);
    f.n_split = (int) std::max<int64_t>(1, std::min({cus / wgs, keys / 256, (int64_t) 64}));
    return f;
}

} // namespace

extern "C" {

int64_t nxg_attention_rows_workspace_bytes(const nxg_attention_rows_params * a) {
    attn_p p;
    const int32_t rc = check_params("attention_rows_workspace_bytes", a, p);
    if (rc) return -rc;
    if (p.T_q == 0 || p.n_seqs == 0) return 0;
    const fwd_plan f = plan_forward(p);
    return f.n_split > 1 ? (int64_t) f.n_split * p.T_q * p.H * (p.D + 8) * 4 : 0;
}

int32_t nxg_attention_rows(const nxg_attention_rows_params * a, const nxg_rows * q, const nxg_rows * k, const nxg_rows * v,
                           const nxg_rows * out, float * lse, void * workspace, int64_t workspace_bytes, void * stream) {
    const char * what = "attention_rows";
    attn_p p;
    NXG_TRY(check_params(what, a, p));
    NXG_TRY(check_rows(what, "q", q, p.T_q, p.H, p.D, false, p.q));
    NXG_TRY(check_rows(what, "k", k, p.T_k, p.G, p.D, false, p.k));
    NXG_TRY(check_rows(what, "v", v, p.T_k, p.G, p.D, false, p.v));
    NXG_TRY(check_rows(what, "out", out, p.T_q, p.H, p.D, true, p.out));
    if (workspace_bytes < 0 || (workspace_bytes > 0 && !workspace) || ((uintptr_t) workspace & 15)) {
        return nxg_fail(NXG_EINVAL, "%s: workspace must be 16-byte aligned memory of workspace_bytes", what);
    }
    if (p.T_q == 0 || p.n_seqs == 0) return NXG_OK;
    if (!p.cu_q || !p.cu_k || !lse) return nxg_fail(NXG_EINVAL, "%s: cu_q, cu_k or lse is null", what);
    NXG_TRY(check_apart(what, "out", p.out, {&p.q, &p.k, &p.v}));
    NXG_TRY(nxg_check_device());
    p.lse = lse;
    p.near_k = near_rows(p.k) && near_rows(p.v);
    fwd_plan f = plan_forward(p);
    if (f.n_split > 1) f.n_split = (int) std::min<int64_t>(f.n_split, workspace_bytes / ((int64_t) p.T_q * p.H * (p.D + 8) * 4));
    f.n_split = std::max(1, f.n_split);
    p.n_split = f.n_split;
    p.part = (float *) workspace;
    hipStream_t s = (hipStream_t) stream;
    const unsigned grid = (unsigned) (slots(p.T_q, p.R, f.few ? 32 : 128, p.n_seqs) * p.G * p.n_split);
    if (f.few) {
        NXG_BY_TYPE(a->type, p.D, (attn_rows_few_kernel<E, DT><<<grid, 256, 0, s>>>(p)));
        NXG_TRY(nxg_launch_check(what));
        if (p.n_split == 1) return NXG_OK;
        const unsigned rows_grid = (unsigned) (((int64_t) p.T_q * p.H + 3) / 4);
        if (a->type == NXG_TYPE_BF16) {
            if (p.D <= 64) attn_rows_join_kernel<__bf16, 8><<<rows_grid, 256, 0, s>>>(p);
            else attn_rows_join_kernel<__bf16, 16><<<rows_grid, 256, 0, s>>>(p);
        } else {
            if (p.D <= 64) attn_rows_join_kernel<_Float16, 8><<<rows_grid, 256, 0, s>>>(p);
            else attn_rows_join_kernel<_Float16, 16><<<rows_grid, 256, 0, s>>>(p);
        }
        return nxg_launch_check(what);
    }
    p.order = work_order(p, grid);
    NXG_BY_TYPE(a->type, p.D, (attn_rows_fwd_kernel<E, DT><<<grid, 256, 0, s>>>(p)));
    return nxg_launch_check(what);
}

int64_t nxg_attention_rows_backward_workspace_bytes(const nxg_attention_rows_params * a) {
    attn_p p;
    const int32_t rc = check_params("attention_rows_backward_workspace_bytes", a, p);
    if (rc) return -rc;
    plan_backward(p);
    return backward_bytes(p);
}

int32_t nxg_attention_rows_backward(const nxg_attention_rows_params * a, const nxg_rows * dout, const nxg_rows * q,
                                    const nxg_rows * k, const nxg_rows * v, const nxg_rows * out, const float * lse,
                                    const nxg_rows * dq, const nxg_rows * dk, const nxg_rows * dv, void * workspace,
                                    int64_t workspace_bytes, void * stream) {
    const char * what = "attention_rows_backward";
    attn_p p;
    NXG_TRY(check_params(what, a, p));
    NXG_TRY(check_rows(what, "dout", dout, p.T_q, p.H, p.D, false, p.dout));
    NXG_TRY(check_rows(what, "q", q, p.T_q, p.H, p.D, false, p.q));
    NXG_TRY(check_rows(what, "k", k, p.T_k, p.G, p.D, false, p.k));
    NXG_TRY(check_rows(what, "v", v, p.T_k, p.G, p.D, false, p.v));
    NXG_TRY(check_rows(what, "out", out, p.T_q, p.H, p.D, false, p.out));
    NXG_TRY(check_rows(what, "dq", dq, p.T_q, p.H, p.D, true, p.dq));
    NXG_TRY(check_rows(what, "dk", dk, p.T_k, p.G, p.D, true, p.dk));
    NXG_TRY(check_rows(what, "dv", dv, p.T_k, p.G, p.D, true, p.dv));
    if (p.n_seqs == 0 || (p.T_q == 0 && p.T_k == 0)) return NXG_OK;
    if (!p.cu_q || !p.cu_k || (p.T_q > 0 && !lse)) return nxg_fail(NXG_EINVAL, "%s: cu_q, cu_k or lse is null", what);
    plan_backward(p);
    if (!workspace || ((uintptr_t) workspace & 15) || workspace_bytes < backward_bytes(p)) {
        return nxg_fail(NXG_EINVAL, "%s: workspace must be 16-byte aligned memory of %lld bytes", what,
                        (long long) backward_bytes(p));
    }
    NXG_TRY(check_apart(what, "dq", p.dq, {&p.dout, &p.q, &p.k, &p.v, &p.out}));
    NXG_TRY(check_apart(what, "dk", p.dk, {&p.dout, &p.q, &p.k, &p.v, &p.out, &p.dq}));
    NXG_TRY(check_apart(what, "dv", p.dv, {&p.dout, &p.q, &p.k, &p.v, &p.out, &p.dq, &p.dk}));
    NXG_TRY(nxg_check_device());
    p.lse = (float *) lse;
    p.near_k = near_rows(p.k) && near_rows(p.v);
    p.near_q = near_pairs(p.q, p.R) && near_pairs(p.dout, p.R);
    p.even_q = 16 % p.R == 0;              // the rows of a thread's step
    p.by_R = ((1u << 22) + p.R - 1) / p.R;
    p.lse2 = (float *) workspace;
    p.ndelta = p.lse2 + row_values(p);
    p.part_q = p.ndelta + row_values(p);
    p.part_kv = p.part_q + part_q_values(p);
    hipStream_t s = (hipStream_t) stream;
    if (p.T_q > 0) {
        const int L = p.D <= 64 ? 8 : 16;
        const int64_t n = ((int64_t) p.T_q * p.R + 2048 / L - 1) / (2048 / L) * p.G;
        const unsigned grid = (unsigned) std::min<int64_t>(n, 1024);
        if (a->type == NXG_TYPE_BF16) {
            if (L == 8) attn_rows_delta_kernel<__bf16, 8><<<grid, 1024, 0, s>>>(p);
            else attn_rows_delta_kernel<__bf16, 16><<<grid, 1024, 0, s>>>(p);
        } else {
            if (L == 8) attn_rows_delta_kernel<_Float16, 8><<<grid, 1024, 0, s>>>(p);
            else attn_rows_delta_kernel<_Float16, 16><<<grid, 1024, 0, s>>>(p);
        }
        NXG_TRY(nxg_launch_check(what));
    }
    const unsigned n_dq = p.T_q > 0 ? (unsigned) (slots(p.T_q, p.R, 128, p.n_seqs) * p.G) : 0;
    const unsigned n_dkv = p.T_k > 0 ? (unsigned) (slots(p.T_k, 1, 128, p.n_seqs) * p.G) : 0;
    p.order = work_order(p, n_dkv);
    const unsigned wgs_dkv = n_dkv * p.split_kv, wgs = wgs_dkv + n_dq * p.split_q;
    NXG_BY_TYPE(a->type, p.D, (attn_rows_grad_kernel<E, DT><<<wgs, 256, 0, s>>>(p, (int) wgs_dkv, work_order(p, n_dq))));
    const unsigned join_kv = p.split_kv > 1 ? n_dkv : 0, joins = join_kv + (p.split_q > 1 ? n_dq : 0);
    if (joins == 0) return nxg_launch_check(what);
    NXG_TRY(nxg_launch_check(what));
    if (a->type == NXG_TYPE_BF16) attn_rows_grad_join_kernel<__bf16><<<joins, 1024, 0, s>>>(p, (int) join_kv);
    else attn_rows_grad_join_kernel<_Float16><<<joins, 1024, 0, s>>>(p, (int) join_kv);
    return nxg_launch_check(what);
}

} // extern "C"
