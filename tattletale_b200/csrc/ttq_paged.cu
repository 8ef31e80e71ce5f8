// Paged key/value cache: append with rotation, and attention for few rows per sequence (decode steps, short drafts).
//
//   paged_append_kernel   one CTA per few tokens: finds the tokens' sequences, normalises and rotates q and k heads, writes q
//                         out and k, v into the pages
//   paged_rows_kernel     attention of tiles of 16 rows (tokens x query heads of one kv head), one or two of them per sequence; memory
//                         bound: every key and value is read once per tile and feeds two products from registers
#include <climits>

#include "ttq_devutil.cuh"
#include "ttq_paged.cuh"

namespace ttq {
namespace {

// ---- append ----------------------------------------------------------------------------------------
// Reads and writes 2 bytes per element of the fused rows and the cos / sin rows of each position: memory bound from a few hundred
// tokens on, a launch below.  A thread holds elements 8 c .. 8 c + 7 of both halves of a head, so that a rotated pair is in one
// thread; the D / 16 threads of a head sum its squares by shuffles.  The heads of a CTA's tokens are dealt out evenly and four CTAs share
// an SM: cos, sin and the norm's weights come again and again from its cache, which leaves registers for as many.  8101 tokens of 48
// heads: 55 us (3.7 TB/s), 79 with cos and sin held in registers (two CTAs), 61 to 82 with two to four heads of a thread in flight.
constexpr int APPEND_THREADS = 256;

struct AppendArgs {
    PagedArgs a;
    PagedAppend p;
};

__device__ __forceinline__ void unpack8(const uint4 &raw, bool bf16, float (&f)[8]) { xh_unpack(raw, bf16 ? TTQ_DT_BF16 : TTQ_DT_F16, f); }
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (BF16) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&t);
        } else {
            const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&t);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void load8(const void *p, int dt, int64_t i, float (&f)[8]) {
    if (dt == TTQ_DT_F32) {
        const float4 *q = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + i);
        const float4 x = q[0], y = q[1];
        f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w; f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
    } else {
        unpack8(*reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(p) + i), dt == TTQ_DT_BF16, f);
    }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(APPEND_THREADS, 4) paged_append_kernel(const __grid_constant__ AppendArgs args, int per_cta) {
    constexpr int C = D / 16;                       // threads of a head
    constexpr int SLOTS = APPEND_THREADS / C;       // heads in flight
    constexpr int MAX_TOKENS = 16;
    __shared__ int64_t dst_s[MAX_TOKENS];           // element offset of the token's slot in the pages (head 0)
    __shared__ int pos_s[MAX_TOKENS];               // -1: nothing is written for the token
    const PagedArgs &a = args.a;
    const PagedAppend &p = args.p;
    grid_launch_dependents();
    grid_dependency_wait();
    const int tid = threadIdx.x;
    const int t0 = blockIdx.x * per_cta;
    const int t1 = (int)(t0 + per_cta < a.n_tokens ? t0 + per_cta : a.n_tokens);
    if (tid < per_cta) pos_s[tid] = -1;
    __syncthreads();
    for (int b = tid; b < a.B; b += APPEND_THREADS) {
        const int s = max(a.q_start[b], 0), e = a.q_start[b + 1];
        const int lo = max(s, t0), hi = min(e, t1);
        if (lo < hi) {
            const int L = paged_len(a, b);
            for (int t = lo; t < hi; t++) {
                const int pos = L - (e - t), own = pos >= a.prefix_len ? pos - a.prefix_len : 0, idx = own >> a.page_shift;
                int page = -1;
                if (pos >= a.prefix_len && idx < a.table_len && pos < p.n_rope) page = a.block_table[(int64_t)b * a.ld_table + idx];
                if (page >= 0 && page < a.n_pages) {
                    dst_s[t - t0] = (int64_t)page * p.page_stride + (int64_t)(own & ((1 << a.page_shift) - 1)) * p.token_stride;
                    pos_s[t - t0] = pos;
                } else {
                    atomicOr(a.status, PAGED_BAD_INDEX);
                }
            }
        }
    }
    __syncthreads();
    const int c = tid % C, slot = tid / C;
    const int heads = a.hq + 2 * a.hkv, pairs = (t1 - t0) * heads;
    const float inv_heads = 1.f / (float)heads;
    // the C threads of a head are consecutive lanes and take the same branches
    const unsigned group = C == 32 ? 0xffffffffu : ((1u << C) - 1u) << ((tid & 31) / C * C);
    for (int x = slot; x < pairs; x += SLOTS) {
        const int t = paged_div(x, heads, inv_heads), h = x - t * heads;
        if (pos_s[t] < 0) continue;
        const uint16_t *src = reinterpret_cast<const uint16_t *>(p.qkv) + (int64_t)(t0 + t) * p.ld_qkv + (int64_t)h * D;
        uint4 r0 = __ldcs(reinterpret_cast<const uint4 *>(src + 8 * c)), r1 = __ldcs(reinterpret_cast<const uint4 *>(src + D / 2 + 8 * c));
        uint16_t *out;
        if (h < a.hq) out = reinterpret_cast<uint16_t *>(p.q_out) + (int64_t)(t0 + t) * p.ld_q + (int64_t)h * D;
        else if (h < a.hq + a.hkv) out = reinterpret_cast<uint16_t *>(p.k) + dst_s[t] + (int64_t)(h - a.hq) * p.head_stride;
        else out = reinterpret_cast<uint16_t *>(p.v) + dst_s[t] + (int64_t)(h - a.hq - a.hkv) * p.head_stride;
        if (h < a.hq + a.hkv) {
            float x0[8], x1[8], w[8];
            unpack8(r0, BF16, x0);
            unpack8(r1, BF16, x1);
            const void *norm = h < a.hq ? p.q_norm : p.k_norm;
            if (norm != nullptr) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) ss = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], ss));
#pragma unroll
                for (int o = C / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(group, ss, o);
                const float inv = rsqrtf(ss / (float)D + p.eps);
                load8(norm, p.dt, 8 * c, w);
#pragma unroll
                for (int i = 0; i < 8; i++) x0[i] = x0[i] * inv * w[i];
                load8(norm, p.dt, D / 2 + 8 * c, w);
#pragma unroll
                for (int i = 0; i < 8; i++) x1[i] = x1[i] * inv * w[i];
            }
            const int64_t row = (int64_t)pos_s[t] * D;
            float y[8];
            load8(p.cosv, p.rope_dt, row + 8 * c, w);
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = x0[i] * w[i];
            load8(p.sinv, p.rope_dt, row + 8 * c, w);
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] -= x1[i] * w[i];
            r0 = pack8<BF16>(y);
            load8(p.cosv, p.rope_dt, row + D / 2 + 8 * c, w);
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = x1[i] * w[i];
            load8(p.sinv, p.rope_dt, row + D / 2 + 8 * c, w);
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] += x0[i] * w[i];
            r1 = pack8<BF16>(y);
        }
        *reinterpret_cast<uint4 *>(out + 8 * c) = r0;
        *reinterpret_cast<uint4 *>(out + D / 2 + 8 * c) = r1;
    }
}

// ---- attention, tiles of 16 rows -------------------------------------------------------------------
// Memory bound: 4 d flops per key, row and 2 bytes x 2 d of cache; 16 rows are 32 flops a byte, a hundred TFLOP/s at the
// card's bandwidth, which m16n8k16 products reach with few warps.  A CTA of four warps takes units of 64 keys (d = 64: 128), each
// warp 16 (32) of them as a pipeline of its own: its lanes issue the tiled copies of 16 slots of one page into the warp's ring
// (128-byte swizzle, read by ldmatrix without conflicts), wait for their own stage only and keep maximum, sum and output of the
// tile in registers; the warps meet once per item.  Three 8 KB stages per warp, two CTAs per SM: 192 KB in flight per SM,
// several times what the memory's latency asks for, which covers the table look-ups and item ends in between.  A stage's
// bookkeeping takes about as long as 4 KB do (23 windows of 4096 keys, d = 64: 55 us with stages of 16 keys).
constexpr int ROWS_WARPS = 4;
constexpr int ROWS_THREADS = ROWS_WARPS * 32;
constexpr int ROWS_TILE = 16;

template <int D>
struct RowsCfg {
    static constexpr int STAGES = 3;
    static constexpr int KT = 128 / D;                     // blocks of 16 keys in a warp's tile
    static constexpr int KEYS = 16 * KT, UNIT = KEYS * ROWS_WARPS;
    static constexpr int TILE_BYTES = KEYS * D * 2;        // a tile of K (or V)
    static constexpr int STAGE_BYTES = 2 * TILE_BYTES;
    static constexpr int RING = ROWS_WARPS * STAGES * STAGE_BYTES;
    static constexpr int OPITCH = D + 4;                   // floats
    static constexpr int OBUF = ROWS_TILE * OPITCH * 4;
    static constexpr int SMEM = RING + OBUF + 1024;        // + alignment of the ring
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (BF16) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&t);
    } else {
        const __half2 t = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&t);
    }
}

// Walk through the units of consecutive sequences: row tiles, kv heads, units.
struct RowsWalk {
    PagedSeq s;
    PagedUnits u;
    int b, rt, head, unit;
};
__device__ __forceinline__ int rows_tiles(const PagedArgs &a, int n) { return (n * a.G + ROWS_TILE - 1) / ROWS_TILE; }
template <int U>
__device__ __forceinline__ void rows_enter(const PagedArgs &a, RowsWalk &w, int min_pos) {
    const int nb = a.prefix_pass ? 1 : a.B;
    for (; w.b < nb; w.b++) {
        w.s = paged_seq(a, w.b, min_pos);
        if (w.s.n > 0) break;
    }
    w.u = paged_units<U>(w.s);
    w.rt = w.head = w.unit = 0;
}
template <int U>
__device__ __forceinline__ void rows_next(const PagedArgs &a, RowsWalk &w, int min_pos, bool more) {
    if (++w.unit == w.u.count) {
        w.unit = 0;
        if (++w.head == a.hkv) {
            w.head = 0;
            if (++w.rt == rows_tiles(a, w.s.n) && more) {
                w.b++;
                rows_enter<U>(a, w, min_pos);
            }
        }
    }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(ROWS_THREADS, PAGED_ROWS16_CTAS) paged_rows_kernel(const __grid_constant__ PagedArgs a,
                                                                                    const __grid_constant__ CUtensorMap kmap,
                                                                                    const __grid_constant__ CUtensorMap vmap) {
    using C = RowsCfg<D>;
    constexpr int HALVES = D / 64, KT = C::KT, KEYS = C::KEYS, UNIT = C::UNIT;
    extern __shared__ uint8_t smem_raw[];
    __shared__ alignas(8) uint64_t full_s[ROWS_WARPS * C::STAGES];
    __shared__ int64_t red[ROWS_WARPS + 4];
    __shared__ float2 ml_s[ROWS_WARPS][ROWS_TILE];
    __shared__ int last_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const uint32_t ring_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    float *obuf = reinterpret_cast<float *>(smem_raw + (ring_base - smem_u32(smem_raw)) + C::RING);
    const uint32_t ring = ring_base + (uint32_t)warp * C::STAGES * C::STAGE_BYTES;
    const uint32_t bars = smem_u32(full_s) + (uint32_t)warp * C::STAGES * 8;
    if (tid == 0) {
        tma_prefetch(&kmap);
        tma_prefetch(&vmap);
    }
    if (lane == 0) {
        for (int i = 0; i < C::STAGES; i++) mbar_init(bars + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    grid_launch_dependents();
    grid_dependency_wait();

    const PagedShare sh = paged_share<ROWS_THREADS, 1>(a, red, [&](int b, bool ok, int min_pos) -> int64_t {
        if (!ok) return 0;
        const PagedSeq s = paged_seq(a, b, min_pos);
        return s.n > 0 ? (int64_t)a.hkv * rows_tiles(a, s.n) * paged_units<UNIT>(s).count : 0;
    });
    if (sh.u0 >= sh.u1) return;

    RowsWalk cw;  // the unit being computed
    cw.b = sh.b;
    rows_enter<UNIT>(a, cw, sh.min_pos);
    {
        const int64_t off = sh.u0 - sh.seq_u;
        const int item = (int)paged_div(off, cw.u.count);
        cw.unit = (int)(off - (int64_t)item * cw.u.count);
        cw.rt = item / a.hkv;
        cw.head = item - cw.rt * a.hkv;
    }
    RowsWalk lw = cw;  // the unit whose copy is issued next
    int64_t lpos = sh.u0;
    int issued = 0, taken = 0;
    int page_cache[KT], cache_first = -1, cache_b = -1;  // lane i: pages of this warp's keys in unit cache_first + i of sequence cache_b

    const int base_pos = a.prefix_pass ? 0 : a.prefix_len;  // absolute position of key 0
    auto wanted = [&](const RowsWalk &w, int k0, int keys) {
        return k0 < w.s.key_end && (a.window == 0 || k0 + keys > w.s.lo || k0 < w.s.sink);
    };
    auto fill = [&]() {
        while (lpos < sh.u1 && issued - taken < C::STAGES) {
            const int k0 = paged_unit_index(lw.u, lw.unit) * UNIT + KEYS * warp;
            if (wanted(lw, k0, KEYS)) {
                if (cache_b != lw.b || lw.unit < cache_first || lw.unit >= cache_first + 32) {
                    cache_b = lw.b;
                    cache_first = lw.unit;
                    const int ku = lw.unit + lane < lw.u.count ? paged_unit_index(lw.u, lw.unit + lane) * UNIT + KEYS * warp : -1;
#pragma unroll
                    for (int t = 0; t < KT; t++) {
                        page_cache[t] = a.n_pages;  // zeros are read from beyond the last page
                        if (ku >= 0 && wanted(lw, ku + 16 * t, 16)) {
                            const int page = a.prefix_pass ? a.prefix_table[(ku + 16 * t) >> a.page_shift] : a.block_table[(int64_t)lw.b * a.ld_table + ((ku + 16 * t) >> a.page_shift)];
                            if (page >= 0 && page < a.n_pages) page_cache[t] = page;
                            else atomicOr(a.status, PAGED_BAD_INDEX);
                        }
                    }
                }
                int page[KT];
#pragma unroll
                for (int t = 0; t < KT; t++) page[t] = __shfl_sync(0xffffffffu, page_cache[t], lw.unit - cache_first);
                const int st = issued % C::STAGES;
                const uint32_t dst = ring + (uint32_t)st * C::STAGE_BYTES, bar = bars + 8 * st;
                if (elect_one()) {
                    mbar_expect_tx(bar, C::STAGE_BYTES);
                    const int head = lw.head, mask = (1 << a.page_shift) - 1;
#pragma unroll
                    for (int t = 0; t < KT; t++)
#pragma unroll
                        for (int h = 0; h < HALVES; h++) {
                            tma_load_page(dst + t * 2048 + h * 2048, &kmap, 64 * h, (k0 + 16 * t) & mask, head, page[t], bar);
                            tma_load_page(dst + C::TILE_BYTES + t * 2048 + h * 2048, &vmap, 64 * h, (k0 + 16 * t) & mask, head, page[t], bar);
                        }
                }
                __syncwarp();
                issued++;
            }
            lpos++;
            rows_next<UNIT>(a, lw, sh.min_pos, lpos < sh.u1);
        }
    };
    fill();

    // fragments of the tile's rows: this thread's are g and g + 8
    uint32_t qf[D / 16][4];
    float o[D / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // references of the weights, and their sums
    int pos0 = 0, pos1 = 0, min_row = 0, max_row = 0, lo_row = 0;  // lo_row: smallest position of a row that has one
    auto row_of = [&](int r, int &token, int &head) {
        const int x = cw.rt * ROWS_TILE + r, i = paged_div(x, a.G, a.inv_G);
        token = cw.s.q0 + i;
        head = cw.head * a.G + (x - i * a.G);
        return i < cw.s.n;
    };
    auto begin = [&]() {
#pragma unroll
        for (int r = 0; r < 2; r++) {
            int token, head;
            const bool ok = row_of(g + 8 * r, token, head);
            int pos = -1;
            if (ok) pos = a.prefix_pass ? paged_row_pos(a, token) : cw.s.pos0 + token - cw.s.q0;
            const uint32_t *src = reinterpret_cast<const uint32_t *>(reinterpret_cast<const uint16_t *>(a.q) + (ok ? (int64_t)token * a.ld_q + (int64_t)head * D : 0)) + t4;
#pragma unroll
            for (int ks = 0; ks < D / 16; ks++) {
                qf[ks][r] = ok ? src[8 * ks] : 0u;
                qf[ks][2 + r] = ok ? src[8 * ks + 4] : 0u;
            }
            if (r == 0) pos0 = pos;
            else pos1 = pos;
            const int lo = __reduce_min_sync(0xffffffffu, ok ? pos : INT_MAX), hi = __reduce_max_sync(0xffffffffu, ok ? pos : -1);
            min_row = r == 0 ? lo : min(min_row, lo);
            max_row = r == 0 ? hi : max(max_row, hi);
        }
        lo_row = max(min_row, 0);
        if (a.prefix_pass && min_row < 0)  // (rows of other sequences, which may be padding)
            lo_row = __reduce_min_sync(0xffffffffu, min(pos0 >= 0 ? pos0 : INT_MAX, pos1 >= 0 ? pos1 : INT_MAX));
#pragma unroll
        for (int n = 0; n < D / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.f;
    };
    begin();
    int64_t seg_start = sh.u0;

    for (int64_t pos = sh.u0; pos < sh.u1; pos++) {
        const int k0 = paged_unit_index(cw.u, cw.unit) * UNIT + KEYS * warp;
        if (wanted(cw, k0, KEYS)) {
            const int st = taken % C::STAGES;
            const uint32_t kt = ring + (uint32_t)st * C::STAGE_BYTES, vt = kt + C::TILE_BYTES;
            mbar_wait_bounded(bars + 8 * st, (taken / C::STAGES) & 1, a.status);
            float s[2 * KT][4] = {};
#pragma unroll
            for (int t = 0; t < KT; t++) {
                const int r = (lane & 7) + ((lane >> 4) << 3), cc = (lane >> 3) & 1;
                const uint32_t row = kt + t * 2048 + r * 128;
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++) {
                    uint32_t b[4];
                    const int c = 2 * ks + cc;
                    ldsm4(row + (c >> 3) * 2048 + (((c & 7) ^ (r & 7)) << 4), b);
                    mma16816<BF16>(s[2 * t], qf[ks], b[0], b[1]);
                    mma16816<BF16>(s[2 * t + 1], qf[ks], b[2], b[3]);
                }
            }
            // visibility: whole tiles need no test
            const int j0 = k0 + base_pos;
            const bool whole = j0 + KEYS - 1 <= min_row && k0 + KEYS <= cw.s.key_end && (a.window == 0 || j0 > max_row - a.window || j0 + KEYS <= a.sinks);
            uint32_t vm[2 * KT];
#pragma unroll
            for (int n = 0; n < 2 * KT; n++) {
                vm[n] = 0xffffffffu;
#pragma unroll
                for (int i = 0; i < 4; i++) s[n][i] *= a.scale2;
            }
            if (!whole) {
#pragma unroll
                for (int n = 0; n < 2 * KT; n++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int k = k0 + 8 * n + 2 * t4 + e, j = k + base_pos;
                        const bool in = k < cw.s.key_end;
                        const bool v0 = in && j <= pos0 && (a.window == 0 || j > pos0 - a.window || j < a.sinks);
                        const bool v1 = in && j <= pos1 && (a.window == 0 || j > pos1 - a.window || j < a.sinks);
                        if (!v0) s[n][e] = -INFINITY;
                        if (!v1) s[n][2 + e] = -INFINITY;
                        // values that no row sees may be anything: zero them
                        const bool any = in && j <= max_row && (a.window == 0 || j > lo_row - a.window || j < a.sinks);
                        if (!any) vm[n] &= e == 0 ? 0xffff0000u : 0x0000ffffu;
                    }
                }
            }
            float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2 * KT; n++) {
                x0 = fmaxf(x0, fmaxf(s[n][0], s[n][1]));
                x1 = fmaxf(x1, fmaxf(s[n][2], s[n][3]));
            }
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) {
                x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
                x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
            }
            // the reference follows the maximum only when a score exceeds it by RISE: weights stay finite in f16
            constexpr float BELOW = PAGED_BELOW<BF16>, RISE = BF16 ? 8.f : 15.f;
            if (__any_sync(0xffffffffu, x0 > m0 + RISE || x1 > m1 + RISE)) {
                const float n0 = fmaxf(m0, x0 - BELOW), n1 = fmaxf(m1, x1 - BELOW);
                const float c0 = m0 == -INFINITY ? 0.f : ex2(m0 - n0), c1 = m1 == -INFINITY ? 0.f : ex2(m1 - n1);
                m0 = n0;
                m1 = n1;
                l0 *= c0;
                l1 *= c1;
#pragma unroll
                for (int n = 0; n < D / 8; n++) {
                    o[n][0] *= c0; o[n][1] *= c0;
                    o[n][2] *= c1; o[n][3] *= c1;
                }
            }
            const float z0 = m0 == -INFINITY ? 0.f : m0, z1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
            for (int n = 0; n < 2 * KT; n++) {
                s[n][0] = ex2(s[n][0] - z0); s[n][1] = ex2(s[n][1] - z0);
                s[n][2] = ex2(s[n][2] - z1); s[n][3] = ex2(s[n][3] - z1);
                l0 += s[n][0] + s[n][1];
                l1 += s[n][2] + s[n][3];
            }
#pragma unroll
            for (int t = 0; t < KT; t++) {
                const uint32_t p[4] = {pack2<BF16>(s[2 * t][0], s[2 * t][1]), pack2<BF16>(s[2 * t][2], s[2 * t][3]), pack2<BF16>(s[2 * t + 1][0], s[2 * t + 1][1]),
                                       pack2<BF16>(s[2 * t + 1][2], s[2 * t + 1][3])};
                const int r = (lane & 7) + (((lane >> 3) & 1) << 3), cc = lane >> 4;
                const uint32_t row = vt + t * 2048 + r * 128;
#pragma unroll
                for (int np = 0; np < D / 16; np++) {
                    uint32_t b[4];
                    const int c = 2 * np + cc;
                    ldsm4t(row + (c >> 3) * 2048 + (((c & 7) ^ (r & 7)) << 4), b);
                    mma16816<BF16>(o[2 * np], p, b[0] & vm[2 * t], b[1] & vm[2 * t + 1]);
                    mma16816<BF16>(o[2 * np + 1], p, b[2] & vm[2 * t], b[3] & vm[2 * t + 1]);
                }
            }
            taken++;
            __syncwarp();  // all lanes have read the stage
            fill();
        }
        const bool item_end = cw.unit + 1 == cw.u.count;
        if (!item_end && pos + 1 < sh.u1) {
            cw.unit++;
            continue;
        }
        // ---- end of the item or of the share: the four warps' results into one ----
        const int64_t item_start = pos - cw.unit, item_stop = item_start + cw.u.count;
        const bool complete = item_end && seg_start == item_start;
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, d);
            l1 += __shfl_xor_sync(0xffffffffu, l1, d);
        }
        if (t4 == 0) {
            ml_s[warp][g] = make_float2(m0, l0);
            ml_s[warp][g + 8] = make_float2(m1, l1);
        }
        __syncthreads();
        auto joint = [&](int r, float &m, float &l) {
            m = -INFINITY;
            l = 0.f;
#pragma unroll
            for (int w = 0; w < ROWS_WARPS; w++) m = fmaxf(m, ml_s[w][r].x);
#pragma unroll
            for (int w = 0; w < ROWS_WARPS; w++)
                if (ml_s[w][r].x != -INFINITY) l = fmaf(ml_s[w][r].y, ex2(ml_s[w][r].x - m), l);
        };
        const int rows = min(ROWS_TILE, cw.s.n * a.G - cw.rt * ROWS_TILE);
        const bool apart = pos + 1 == sh.u1;
        const int together = apart || rows <= 4 ? 4 : (rows <= 8 ? 2 : 1);
        {
            float M0, M1, x;
            joint(g, M0, x);
            joint(g + 8, M1, x);
            const float c0 = m0 == -INFINITY ? 0.f : ex2(m0 - M0), c1 = m1 == -INFINITY ? 0.f : ex2(m1 - M1);
            // At the share's end the warps' rings are free and take a result each.  Before, `together` warps at a time put theirs into the one
            // buffer there is (a second one would cost the second CTA of the SM), all four where the tile has four rows.
            float *mine = apart ? reinterpret_cast<float *>(smem_raw + (ring - smem_u32(smem_raw))) : obuf + (warp % together) * (ROWS_TILE / together) * C::OPITCH;
            for (int turn = 0; turn < ROWS_WARPS / together; turn++) {
                if (warp / together == turn) {
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const float c = r == 0 ? c0 : c1;
                        float *to = mine + (g + 8 * r) * C::OPITCH + 2 * t4;
                        if (g + 8 * r < rows) {
#pragma unroll
                            for (int n = 0; n < D / 8; n++) {
                                float2 v = make_float2(o[n][2 * r] * c, o[n][2 * r + 1] * c);
                                if (turn > 0) {
                                    const float2 x = *reinterpret_cast<const float2 *>(to + 8 * n);
                                    v.x += x.x;
                                    v.y += x.y;
                                }
                                *reinterpret_cast<float2 *>(to + 8 * n) = v;
                            }
                        }
                    }
                }
                __syncthreads();
            }
        }
        const int own_slot = 2 * blockIdx.x + (seg_start == item_start ? 1 : 0);
        float *part = a.part + (int64_t)own_slot * ROWS_TILE * (D + 2);
        for (int i = tid; i < rows * (D / 8); i += ROWS_THREADS) {
            const int r = i / (D / 8), col = i % (D / 8) * 8;
            float m, l, v[8];
            joint(r, m, l);
#pragma unroll
            for (int x = 0; x < 8; x++) v[x] = 0.f;
#pragma unroll
            for (int w = 0; w < ROWS_WARPS; w++)
                if (w < together) {
                    const float *from = apart ? reinterpret_cast<const float *>(smem_raw + (ring_base - smem_u32(smem_raw)) + w * C::STAGES * C::STAGE_BYTES)
                                              : obuf + w * (ROWS_TILE / together) * C::OPITCH;
                    const float4 *src = reinterpret_cast<const float4 *>(from + r * C::OPITCH + col);
                    const float4 y0 = src[0], y1 = src[1];
                    v[0] += y0.x; v[1] += y0.y; v[2] += y0.z; v[3] += y0.w;
                    v[4] += y1.x; v[5] += y1.y; v[6] += y1.z; v[7] += y1.w;
                }
            if (complete) {
                int token, head;
                row_of(r, token, head);
                paged_finish8<BF16>(a, D, token, head, col, m, l, v);
            } else {
                float4 *d = reinterpret_cast<float4 *>(part + r * D + col);
                d[0] = make_float4(v[0], v[1], v[2], v[3]);
                d[1] = make_float4(v[4], v[5], v[6], v[7]);
                if (col == 0) *reinterpret_cast<float2 *>(part + ROWS_TILE * D + 2 * r) = make_float2(m, l);
            }
        }
        if (!complete) {
            const int c0 = paged_owner(item_start, sh.total, sh.N), c1 = paged_owner(item_stop - 1, sh.total, sh.N);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const unsigned seen = atomicAdd(a.counters + c0, 1u);
                last_s = seen == (unsigned)(c1 - c0);
                if (last_s) a.counters[c0] = 0;
            }
            __syncthreads();
            if (last_s) {
                __threadfence();
                for (int i = tid; i < rows * (D / 8); i += ROWS_THREADS) {
                    const int r = i / (D / 8), col = i % (D / 8) * 8;
                    float m, l, v[8];
                    paged_gather8<ROWS_TILE>(a, D, c0, c1, r, col, m, l, v);
                    int token, head;
                    row_of(r, token, head);
                    paged_finish8<BF16>(a, D, token, head, col, m, l, v);
                }
            }
        }
        if (pos + 1 < sh.u1) {
            __syncthreads();  // obuf, ml_s and last_s are written again
            rows_next<UNIT>(a, cw, sh.min_pos, true);
            seg_start = pos + 1;
            begin();
        }
    }
}

template <int D, bool BF16>
cudaError_t launch_rows_t(const PagedArgs &a, const PagedMaps &maps, cudaStream_t st) {
    using C = RowsCfg<D>;
    auto kernel = paged_rows_kernel<D, BF16>;
    static OncePerDevice once;
    const cudaError_t e = once([&]() { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM); });
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3((unsigned)(PAGED_ROWS16_CTAS * a.sms)), dim3(ROWS_THREADS), C::SMEM, st, a, maps.k, maps.v);
}

template <int D>
cudaError_t launch_append_t(const AppendArgs &args, int per_cta, cudaStream_t st) {
    const dim3 grid((unsigned)((args.a.n_tokens + per_cta - 1) / per_cta));
    if (args.p.dt == TTQ_DT_BF16) return launch_pdl(paged_append_kernel<D, true>, grid, dim3(APPEND_THREADS), 0, st, args, per_cta);
    return launch_pdl(paged_append_kernel<D, false>, grid, dim3(APPEND_THREADS), 0, st, args, per_cta);
}

}  // namespace

int64_t paged_part_floats(int d, int sms) {
    const int64_t rows = (int64_t)2 * PAGED_ROWS16_CTAS * sms * ROWS_TILE * (d + 2), tc = paged_tc_part_floats(d, sms);
    return rows > tc ? rows : tc;
}
int64_t paged_counters(int sms) { return PAGED_ROWS16_CTAS * sms; }

cudaError_t launch_paged_rows(const PagedArgs &a, int dt, int d, const PagedMaps &maps, cudaStream_t st) {
    if (d == 128) return dt == TTQ_DT_BF16 ? launch_rows_t<128, true>(a, maps, st) : launch_rows_t<128, false>(a, maps, st);
    return dt == TTQ_DT_BF16 ? launch_rows_t<64, true>(a, maps, st) : launch_rows_t<64, false>(a, maps, st);
}

cudaError_t launch_paged_append(const PagedArgs &a, const PagedAppend &p, cudaStream_t st) {
    AppendArgs args{a, p};
    // one token per CTA while the card holds all of them at once, several from there on (the search for their sequences is shared)
    const int per_cta = a.n_tokens <= 4 * (int64_t)a.sms ? 1 : 4;
    return p.d == 128 ? launch_append_t<128>(args, per_cta, st) : launch_append_t<64>(args, per_cta, st);
}

}  // namespace ttq
