// Attention over a paged cache: the arguments, the ragged batch's geometry and the division of the work, shared by the kernel for
// few rows per sequence (ttq_paged.cu) and the tensor-memory kernel (ttq_paged_tc.cu).
//
// The rows of a sequence that attend with one kv head are its new tokens times the G = hq / hkv query heads of that kv head, row
// r = token r / G, head r % G: K and V are read once for all of them.  An item is a tile of such rows; its keys are walked in
// units of a fixed number of keys.  All units of a call are numbered through (the tensor-memory kernel: weighted) -- sequence, row tile, kv head, unit -- and every CTA
// takes an equal, contiguous share of the numbers, found from the lengths in device memory by each CTA for itself (a captured graph
// follows them, the host never waits).  An item that one CTA sees whole is finished there; of an item cut by share borders
// every CTA leaves a partial result (running maximum, sum, unnormalised output) in the plan's workspace, at most two per CTA
// whatever the batch looks like.  They are added in the order of the keys, hence to the same bits every time: by the CTA that
// arrives last (few rows), or by a launch of its own (hundreds of rows).
#pragma once

#include <cuda.h>

#include <climits>

#include "ttq_internal.cuh"

namespace ttq {

struct PagedArgs {
    const void *q;
    void *out;
    int64_t ld_q, ld_out;
    int64_t n_tokens;
    int B;
    const int *q_start, *kv_len, *block_table;
    int64_t ld_table;
    int table_len;
    int prefix_len;
    const int *prefix_table;
    int prefix_pass;            // 1: all rows of the batch against the shared prefix's keys, results to pre_o / pre_lse
    int hq, hkv, G, page_shift, n_pages;
    int tokens;                 // tensor-memory kernel: tokens of a stream, 128 / G
    float inv_tokens2, inv_G;   // 1 / (2 tokens), 1 / G
    int window, sinks;          // window 0: none
    float scale2;               // scale * log2(e): scores and maxima are kept in units of log2
    float *pre_o, *pre_lse;     // [n_tokens][hq][d] normalised, [n_tokens][hq]; read by the other pass (nullptr: no prefix)
    float *part;                // partial results, two per CTA
    unsigned *counters;         // few rows: arrivals, one per CTA, zero between launches; else the records of cut items
    int *status;
    int sms;
};

// 2^x (x <= 8 or so, 2 ulp; results below 2^-126 are zero)
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The softmax weights enter the second product in the 16-bit type, the only operand that the tensor cores take beside 16-bit values: a
// rounding of half a step of each weight (2^-8 relative in bf16, 2^-11 in f16), where the contiguous step's kernel (ttq_decode.cu)
// multiplies in 32 bits.  Weights are 2^(score - reference); in f16, whose range ends at 2^-14 (2^-24 in steps), the reference
// lies 2^9 below the maximum that it was taken from, so that a weight is rounded relative to itself down to 2^-23 of the row's
// largest and is off by no more than 2^-34 of it below.  Their sum is of the unrounded ones.
template <bool BF16>
constexpr float PAGED_BELOW = BF16 ? 0.f : 9.f;
constexpr int PAGED_BAD_INDEX = 8;  // status bit: page id or position outside the cache

// Lengths and positions are 32-bit.  A sequence of no or negative length has no positions: its tokens count down from -1.  Positions end
// a few units before 2^31, so that the first key behind a unit is still a number.
constexpr int PAGED_MAX_LEN = INT_MAX - 4095;
__device__ __forceinline__ int paged_len(const PagedArgs &a, int b) { return max(0, a.kv_len[b]); }
// First key (of `end`; in the coordinates of a table that begins at position `base`) that the window of a token at `pos` holds.
__device__ __forceinline__ int paged_window_start(const PagedArgs &a, int pos, int base, int end) {
    const int64_t first = (int64_t)pos - a.window + 1 - base;
    return (int)max((int64_t)0, min((int64_t)end, first));
}

// One sequence's rows and keys (prefix pass: the one group of all rows).  Keys are in the coordinates of its page table.
struct PagedSeq {
    int q0, n;      // first row and number of new tokens
    int pos0;       // absolute position of token 0 (own pass)
    int key_end;    // keys 0 .. key_end - 1 exist
    int lo;         // first key behind the sinks that any token sees
    int sink;       // keys 0 .. sink - 1 are visible as sinks (sink <= lo)
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs &a, int b, int min_pos) {
    PagedSeq s;
    const int T = (int)a.n_tokens;
    int end, pmin;
    if (a.prefix_pass) {
        s.q0 = 0;
        s.n = max(0, min(a.q_start[a.B], T));
        s.pos0 = 0;
        end = a.prefix_len;
        pmin = min_pos;
    } else {
        s.q0 = max(0, min(a.q_start[b], T));
        s.n = max(0, min(a.q_start[b + 1], T) - s.q0);
        const int L = paged_len(a, b);
        s.pos0 = L - s.n;
        const int64_t cap = min((int64_t)a.table_len << a.page_shift, max((int64_t)0, PAGED_MAX_LEN - (int64_t)a.prefix_len));
        end = max(0, L - a.prefix_len);
        if (end > cap) {
            if (s.n > 0) atomicOr(a.status, PAGED_BAD_INDEX);
            end = (int)cap;
        }
        pmin = s.pos0;
    }
    s.key_end = end;
    const int base = a.prefix_pass ? 0 : a.prefix_len;
    s.lo = 0;
    s.sink = 0;
    if (a.window > 0) {
        s.lo = paged_window_start(a, pmin, base, end);
        s.sink = max(0, min(s.lo, a.sinks - base));
    }
    return s;
}

// Units of U keys that a row tile of the sequence walks: those of the sinks, then those from the window's start on.
struct PagedUnits {
    int sink, first, count;
};
template <int U>
__device__ __forceinline__ PagedUnits paged_units(const PagedSeq &s) {
    PagedUnits u;
    u.first = s.lo / U;
    u.sink = min((s.sink + U - 1) / U, u.first);
    const int last = (s.key_end + U - 1) / U;
    u.count = max(1, u.sink + max(0, last - u.first));  // a row without keys is still written
    return u;
}
__device__ __forceinline__ int paged_unit_index(const PagedUnits &u, int i) { return i < u.sink ? i : u.first + i - u.sink; }

// Position of a row's token in the prefix pass (the sequence that holds it by bisection), INT_MIN for a row of no sequence.
__device__ __forceinline__ int paged_row_pos(const PagedArgs &a, int token) {
    int lo = 0, hi = a.B;  // q_start[lo] <= token < q_start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.q_start[mid] <= token) lo = mid;
        else hi = mid;
    }
    return paged_len(a, lo) - (a.q_start[lo + 1] - token);
}

// Quotients.  The compiler's 64-bit division is several hundred clocks of a warp's time, its 32-bit one a hundred and more, and a CTA
// stands behind a dozen of them before its first copy.
__device__ __forceinline__ int64_t paged_div(int64_t x, int64_t d) {
    return ((uint64_t)x | (uint64_t)d) >> 32 ? x / d : (int64_t)((uint32_t)x / (uint32_t)d);
}
__device__ __forceinline__ int paged_div(int x, int d, float inv) {  // x >= 0
    if (x >= 1 << 22) return x / d;
    const int q = (int)((float)x * inv), r = x - q * d;  // (the product is off by less than one)
    return q + (r >= d ? 1 : 0) - (r < 0 ? 1 : 0);
}
// Shares of `total` numbers for N owners: the first `total % N` have one more than the others.  Owner of number u:
__device__ __forceinline__ int paged_owner(int64_t u, int64_t total, int N) {
    const int64_t size = paged_div(total, N), longer = total - size * N, edge = longer * (size + 1);
    return (int)(u < edge ? paged_div(u, size + 1) : longer + paged_div(u - edge, size));
}

// What one CTA finds out before it starts.
struct PagedShare {
    int64_t total;   // all units of the call
    int64_t u0, u1;  // this CTA's
    int64_t seq_u;   // number of the first unit of the sequence that holds u0
    int b;           // that sequence
    int N;           // CTAs that have a share
    int min_pos;     // prefix pass: smallest position of any token that has one (INT_MAX: none does)
};

// Number of shares: of at least MIN_SHARE numbers each, at most one per CTA.
template <int MIN_SHARE>
__device__ __forceinline__ int paged_shares(int64_t total) {
    const int64_t most = total / MIN_SHARE;
    return total == 0 ? 0 : (int)(most < 1 ? 1 : (most < gridDim.x ? most : gridDim.x));
}
// Called by all THREADS of the CTA.  `cost(b, ok, min_pos)`: units of sequence b (ok false: none), whole warps at a time.  red: shared, at least THREADS / 32 + 4 int64.
template <int THREADS, int MIN_SHARE, class Cost>
__device__ __forceinline__ PagedShare paged_share(const PagedArgs &a, int64_t *red, Cost &&cost) {
    constexpr int W = THREADS / 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    PagedShare sh;
    sh.min_pos = 0;
    const int nb = a.prefix_pass ? 1 : a.B;
    if (a.prefix_pass && a.window > 0) {
        int mp = INT_MAX;
        for (int b = tid; b < a.B; b += THREADS) {
            const int n = a.q_start[b + 1] - a.q_start[b], L = paged_len(a, b);
            if (n > 0 && L > 0) mp = min(mp, max(0, L - n));  // (padding, a token of no position, sees nothing)
        }
        mp = __reduce_min_sync(0xffffffffu, mp);
        if (lane == 0) red[warp] = mp;
        __syncthreads();
        for (int w = 0; w < W; w++) mp = min(mp, (int)red[w]);
        __syncthreads();
        sh.min_pos = mp;
    }
    // total, then the sequence that holds the share's first unit (one pass over the lengths when they fit one chunk)
    int64_t total = 0, u0 = 0, u1 = 0;
    auto bounds = [&]() {
        sh.N = paged_shares<MIN_SHARE>(total);
        u0 = u1 = total;
        if ((int)blockIdx.x < sh.N) {
            const int64_t size = paged_div(total, sh.N), longer = total - size * sh.N, c = blockIdx.x;
            u0 = c * size + (c < longer ? c : longer);
            u1 = u0 + size + (c < longer ? 1 : 0);
        }
    };
    for (int pass = 0; pass < 2; pass++) {
        int64_t running = 0;
        for (int base = 0; base < nb; base += THREADS) {
            const int b = base + tid;
            const int64_t c = cost(b, b < nb, sh.min_pos);
            int64_t incl = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            if (lane == 31) red[warp] = incl;
            __syncthreads();
            int64_t before = running, chunk = 0;
            for (int w = 0; w < W; w++) {
                if (w < warp) before += red[w];
                chunk += red[w];
            }
            if (nb <= THREADS) {
                total = chunk;
                bounds();
                pass = 1;
            }
            const int64_t at = before + incl - c;
            if (pass == 1 && c > 0 && at <= u0 && u0 < at + c) {
                red[W] = b;
                red[W + 1] = at;
            }
            running += chunk;
            __syncthreads();
        }
        if (pass == 0) {
            total = running;
            bounds();
        }
    }
    sh.total = total;
    sh.u0 = u0;
    sh.u1 = u1;
    sh.b = sh.u1 > sh.u0 ? (int)red[W] : 0;
    sh.seq_u = sh.u1 > sh.u0 ? red[W + 1] : 0;
    __syncthreads();
    return sh;
}

// Eight consecutive results of one row: normalised, joined with the shared prefix's part, written.  m, l: running maximum (log2
// units) and sum of the row.
template <bool BF16>
__device__ __forceinline__ void paged_finish8(const PagedArgs &a, int D, int token, int head, int col, float m, float l, float (&v)[8]) {
    const int64_t row = (int64_t)token * a.hq + head;
    if (a.prefix_pass) {
        const float inv = l > 0.f ? 1.f / l : 0.f;
        float4 *dst = reinterpret_cast<float4 *>(a.pre_o + row * D + col);
        dst[0] = make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        dst[1] = make_float4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
        if (col == 0) a.pre_lse[row] = l > 0.f ? m + log2f(l) : -INFINITY;
        return;
    }
    float wo = l > 0.f ? 1.f / l : 0.f;
    if (a.pre_o != nullptr) {
        const float lse = a.pre_lse[row];
        if (lse != -INFINITY) {
            const float mx = fmaxf(m, lse), own = m == -INFINITY ? 0.f : ex2(m - mx), pre = ex2(lse - mx), inv = 1.f / (l * own + pre);
            const float4 *src = reinterpret_cast<const float4 *>(a.pre_o + row * D + col);
            const float4 p0 = src[0], p1 = src[1];
            const float wp = pre * inv;
            wo = own * inv;
            v[0] = v[0] * wo + p0.x * wp; v[1] = v[1] * wo + p0.y * wp; v[2] = v[2] * wo + p0.z * wp; v[3] = v[3] * wo + p0.w * wp;
            v[4] = v[4] * wo + p1.x * wp; v[5] = v[5] * wo + p1.y * wp; v[6] = v[6] * wo + p1.z * wp; v[7] = v[7] * wo + p1.w * wp;
            wo = 1.f;
        }
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (BF16) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i] * wo, v[2 * i + 1] * wo);
            w[i] = *reinterpret_cast<const uint32_t *>(&t);
        } else {
            const __half2 t = __floats2half2_rn(v[2 * i] * wo, v[2 * i + 1] * wo);
            w[i] = *reinterpret_cast<const uint32_t *>(&t);
        }
    }
    uint16_t *dst = reinterpret_cast<uint16_t *>(a.out) + (int64_t)token * a.ld_out + (int64_t)head * D + col;
    *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Adds the partials of eight results of one row in the order of the keys: maximum, sum and unnormalised output.
// part: [2 N][ROWS][D + 2] = (outputs, then maximum and sum per row).  The item's units are in the shares of CTAs c0 .. c1; it starts
// in c0's last segment (slot 2 c0 + 1) and continues in the first ones of the others (slots 2 c).
template <int ROWS>
__device__ __forceinline__ void paged_gather8(const PagedArgs &a, int D, int c0, int c1, int r, int col, float &m, float &l, float (&v)[8]) {
    const int64_t pitch = (int64_t)ROWS * (D + 2);
    const float *ml = a.part + (int64_t)ROWS * D + 2 * r;
    m = -INFINITY;
#pragma unroll 8
    for (int c = c0; c <= c1; c++) m = fmaxf(m, __ldcg(ml + (2 * c + (c == c0)) * pitch));
    l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = 0.f;
    if (m == -INFINITY) return;
    const float *o = a.part + (int64_t)r * D + col;
#pragma unroll 4
    for (int c = c0; c <= c1; c++) {
        const int64_t at = (2 * c + (c == c0)) * pitch;
        const float2 s = __ldcg(reinterpret_cast<const float2 *>(ml + at));
        const float4 x = __ldcg(reinterpret_cast<const float4 *>(o + at)), y = __ldcg(reinterpret_cast<const float4 *>(o + at + 4));
        const float w = ex2(s.x - m);
        l = fmaf(w, s.y, l);
        v[0] = fmaf(w, x.x, v[0]); v[1] = fmaf(w, x.y, v[1]); v[2] = fmaf(w, x.z, v[2]); v[3] = fmaf(w, x.w, v[3]);
        v[4] = fmaf(w, y.x, v[4]); v[5] = fmaf(w, y.y, v[5]); v[6] = fmaf(w, y.z, v[6]); v[7] = fmaf(w, y.w, v[7]);
    }
}

// Four-dimensional tiled copies of the pages: (element of the head, slot, kv head, page).
__device__ __forceinline__ void tma_prefetch(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap *map, int x, int slot, int head, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(bar)
        : "memory");
}

struct PagedMaps {
    CUtensorMap k, v, q;  // q: the tensor-memory kernel only
};
// One launch of a pass (own keys, or the shared prefix's).
cudaError_t launch_paged_rows(const PagedArgs &a, int dt, int d, const PagedMaps &maps, cudaStream_t st);
constexpr int PAGED_ROWS16_CTAS = 2;  // resident CTAs per SM of the kernel for few rows
cudaError_t launch_paged_tc(const PagedArgs &a, int dt, int d, const PagedMaps &maps, int box_rows, cudaStream_t st);
int64_t paged_tc_part_floats(int d, int sms);
int64_t paged_tc_words(int sms);  // records of cut items
// Workspace of a plan: partial results in floats, arrival counters of the kernel for few rows.
int64_t paged_part_floats(int d, int sms);
int64_t paged_counters(int sms);
struct PagedAppend {
    const void *qkv, *q_norm, *k_norm, *cosv, *sinv;
    void *q_out, *k, *v;
    int64_t ld_qkv, ld_q, page_stride, head_stride, token_stride;
    float eps;
    int dt, rope_dt, n_rope, d;
};
cudaError_t launch_paged_append(const PagedArgs &a, const PagedAppend &p, cudaStream_t st);

}  // namespace ttq
