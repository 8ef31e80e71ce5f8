// Attention over a paged cache on the tensor cores (tcgen05): prompts, pieces of prompts, and rows of a whole batch against a shared
// prefix.
//
// An item is a tile of up to 2 x 128 rows -- twice floor(128 / G) tokens times the G query heads of one kv head -- walked in units of
// 128 keys.  Its two halves are two streams that take turns: while the softmax of one runs on the CUDA cores, the tensor core multiplies for the other.
//   S = Q K^T     128 rows x 64 keys (half a unit), Q and K in shared memory (K-major, 128-byte swizzle), S in one of the stream's two
//                 score buffers in tensor memory
//   softmax       a thread per row: 64 scores from tensor memory, reference and sum in registers, weights in the 16-bit type
//                 back into the columns that the scores had
//   O += P V      P from tensor memory, V as it lies in its pages (keys as rows: the transposed operand form), O in tensor memory
// The scores of half j + 1 are complete while the softmax works on half j.  With one buffer of 128 keys per stream the softmax
// waited for the product and the product for the softmax: 4260 clocks per unit of both streams instead of 3500.
// An item of one half gives both streams the same rows and every other unit of keys; the two results meet in tensor
// memory, whose lanes the warps of both streams reach.  Tensor memory is full: 2 x 2 x 64 columns of scores, 2 x d of output.
//
// Warps 0-3 and 4-7: softmax of the two streams, and their rows' results.  Warps 8 and 11 issue the streams' products -- one
// warp for both would leave the tensor core idle during its waits, since the issue of a product blocks until the queue before it has
// drained -- warp 9 the tiled copies of the pages into a ring of slots.  Warp 10 walks the batch, hands the other warps one
// record per item, so that they keep their registers for scores, and copies the queries (one copy per stream and 64 columns: the
// G heads of a run of tokens are the rows of a tile as they lie).  Products of one stream execute in the order of issue, so the scores of half
// j + 2 may follow the product that reads the weights of half j from the same columns.  The softmax warps rescale the output in
// place, which they do only when the weights outgrow their reference and once the last product that they asked for is complete.
//
// Bound: 4 d flops and one exponential per key and row; at d = 128 the special-function unit (16 a clock and SM) takes as long for a
// unit's exponentials as the tensor core for its products, 2048 clocks for both streams.  Measured: prompts of 1111 to 4300
// tokens 301 us among other passes on changing inputs (737 TFLOP/s, 44 % of the measured bf16 rate), 285 back to back on the same ones; 24000
// shared keys 172 and 157 us (774 and 847 TFLOP/s).
#include <climits>

#include "ttq_devutil.cuh"
#include "ttq_paged.cuh"

namespace ttq {
namespace {

constexpr int TC_UNIT = 128;       // keys per unit (of copies and of shares)
constexpr int TC_HALF = 64;        // keys per product
constexpr int TC_ROWS = 128;       // rows per stream
constexpr int TC_ITEM_ROWS = 2 * TC_ROWS;
constexpr int TC_MMA_WARP = 8, TC_TMA_WARP = 9, TC_WALK_WARP = 10, TC_MMA1_WARP = 11;
constexpr int TC_THREADS = 384, TC_SOFTMAX_THREADS = 256;
// The block is launched with 168 registers a thread (65536 / 384, in steps of 8); a softmax thread, which holds a row of scores,
// gets 208, a thread of the third warpgroup keeps 88: 8 x 208 + 4 x 88 = 12 x 168.
constexpr int TC_SOFTMAX_REGS = 208, TC_OTHER_REGS = 88;

// One item, or the part of it that is in this CTA's share.
struct TcSeg {
    int m;                    // units (0: the share ends)
    int unit, u_sink, u_first;   // first unit; numbers of the item's units as PagedUnits has them
    int key_end, lo, sink;
    int pair;                 // the streams have rows of their own
    int tok0, n;              // first token of the item, tokens of the sequence
    int b, head, q0, pos0;
    int complete, slot;       // the item is whole; else where its partial goes
};
constexpr int TC_SEGS = 4, TC_SEG_READERS = 11;  // (8 softmax warps, copies, two product warps)
// An item that begins in one CTA's share and ends in CTA c1's (rows 0: none), left for the kernel that joins the parts.
struct TcSplit {
    int c1, rows, tok0, n, q0, head;
};
__device__ __forceinline__ int tc_tokens(const PagedArgs &a) { return a.tokens; }  // of a stream

template <int D>
struct TcCfg {
    static constexpr int HALVES = D / 64;
    static constexpr int HALF_BYTES = 128 * 128;               // 128 rows x 64 elements
    static constexpr int SLOT_BYTES = HALVES * HALF_BYTES;     // a unit of K or of V; a stream's queries
    static constexpr int SLOTS = D == 128 ? 4 : 8;             // a fifth (tenth) changed nothing; its room is the results'
    static constexpr int S_COL = 0, O_COL = 256;               // streams 128 columns, resp. D columns apart
    // shared memory: queries, ring, 4 KB per softmax warp through which results leave, then barriers and exchange
    static constexpr int RING_AT = 2 * SLOT_BYTES;
    static constexpr int OUT_AT = RING_AT + SLOTS * SLOT_BYTES;
    static constexpr int BAR_AT = OUT_AT + 8 * 4096;
    static constexpr int N_BARS = 2 * SLOTS + 14 + 1 + 2 * TC_SEGS;
    static constexpr int ML_AT = BAR_AT + (N_BARS * 8 + 15) / 16 * 16;
    static constexpr int SEG_AT = ML_AT + 2 * TC_ROWS * 8;
    static constexpr int MISC_AT = SEG_AT + (TC_SEGS * (int)sizeof(TcSeg) + 15) / 16 * 16;
    static constexpr int SMEM = MISC_AT + 16 * 8 + 16;
};

template <bool BF16>
__host__ __device__ constexpr uint32_t tc_idesc(int n, bool b_rows_are_k) {
    return (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (b_rows_are_k ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// V: element (key, column) of a unit is row `key` of 128 bytes in the half of its column.  As the transposed operand: 8-key groups
// 1024 bytes apart (stride offset), 64-column blocks a half apart (leading offset), 128-byte swizzle.
__device__ __forceinline__ uint64_t tc_desc_v(uint32_t addr, int half_bytes) {
    const uint32_t lo = ((addr & 0x3ffffu) >> 4) | ((uint32_t)(half_bytes >> 4) << 16);
    const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// rows of a stream's queries: (element of the head, head, token)
__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap *map, int x, int head, int token, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(x),
        "r"(head), "r"(token), "r"(bar)
        : "memory");
}
// 32 columns of this thread's lane
__device__ __forceinline__ void tc_ld32(uint32_t taddr, float *v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
        "%29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
// the wait, through which the loaded registers pass
__device__ __forceinline__ void tc_ld_wait32(float *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]),
                   "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]),
                   "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]),
                   "+f"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
        "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
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

__device__ __forceinline__ void tc_ld16(uint32_t taddr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]),
          "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr)
        : "memory");
}
// ---- pairs of floats -----------------------------------------------------------------------------------
__device__ __forceinline__ uint64_t f2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void f2_split(uint64_t v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// How the work is numbered: a unit of keys counts once for an item of one stream, twice for one of two; an item's start and end
// count like TC_ITEM_WEIGHT of them.
constexpr int TC_PAIR_WEIGHT = 2, TC_ITEM_WEIGHT = 6;
// Row tile rt of a sequence: its rows, and the keys that any of them sees.
struct TcItem {
    PagedSeq k;      // key_end, lo, sink of this item (the rest as the sequence's)
    PagedUnits u;
    int tok0, tokens;
    int shift, size;    // a unit has 1 << shift numbers; numbers of the whole item
    // units whose number is below p; unit i stands at TC_ITEM_WEIGHT + (i << shift)
    __device__ __forceinline__ int units_before(int p) const { return max(0, min(u.count, (p - TC_ITEM_WEIGHT + (1 << shift) - 1) >> shift)); }
};
__device__ __forceinline__ int tc_tiles(const PagedArgs &a, int n) { return paged_div(n + 2 * tc_tokens(a) - 1, 2 * tc_tokens(a), a.inv_tokens2); }
__device__ __forceinline__ TcItem tc_item(const PagedArgs &a, const PagedSeq &s, int rt) {
    TcItem it;
    it.k = s;
    it.tok0 = rt * 2 * tc_tokens(a);
    it.tokens = min(2 * tc_tokens(a), s.n - it.tok0);
    if (!a.prefix_pass) {
        it.k.key_end = max(0, min(s.key_end, s.pos0 + it.tok0 + it.tokens - a.prefix_len));
        it.k.lo = it.k.sink = 0;
        if (a.window > 0) {
            it.k.lo = paged_window_start(a, s.pos0 + it.tok0, a.prefix_len, it.k.key_end);
            it.k.sink = max(0, min(it.k.lo, a.sinks - a.prefix_len));
        }
    }
    it.u = paged_units<TC_UNIT>(it.k);
    it.shift = it.tokens > tc_tokens(a) ? 1 : 0;
    it.size = TC_ITEM_WEIGHT + (it.u.count << it.shift);
    return it;
}
// Numbers of one kv head's items of a sequence, by the whole warp (`s`: the same in all lanes).
__device__ __forceinline__ int64_t tc_seq_units(const PagedArgs &a, const PagedSeq &s, int lane) {
    const int nt = tc_tiles(a, s.n);
    int64_t sum = 0;
    for (int rt = lane; rt < nt; rt += 32) sum += tc_item(a, s, rt).size;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// Walk through the items of consecutive sequences: kv heads, and their row tiles.  Every warp walks for itself.
struct TcWalk {
    PagedSeq s;
    TcItem it;
    int b, head, rt, nt;
    int at;          // number within the item
    int64_t pos;     // the same, of the call

    __device__ __forceinline__ void enter(const PagedArgs &a, int min_pos) {
        const int nb = a.prefix_pass ? 1 : a.B;
        for (; b < nb; b++) {
            s = paged_seq(a, b, min_pos);
            if (s.n > 0) break;
        }
        nt = tc_tiles(a, s.n);
        head = rt = at = 0;
        it = tc_item(a, s, 0);
    }
    // to the share's first number (the whole warp)
    __device__ __forceinline__ void start(const PagedArgs &a, const PagedShare &sh, int lane) {
        b = sh.b;
        enter(a, sh.min_pos);
        int64_t off = sh.u0 - sh.seq_u;
        pos = sh.u0;
        if (nt == 1) {
            head = (int)paged_div(off, it.size);
            at = (int)(off - (int64_t)head * it.size);
            return;
        }
        const int64_t per_head = tc_seq_units(a, s, lane);
        head = (int)paged_div(off, per_head);
        off -= head * per_head;
#pragma unroll 1
        for (int base = 0;; base += 32) {
            const int c = base + lane < nt ? tc_item(a, s, base + lane).size : 0;
            int incl = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, off < incl);
            if (hit) {
                const int l = __ffs(hit) - 1;
                rt = base + l;
                at = (int)off - __shfl_sync(0xffffffffu, incl - c, l);
                break;
            }
            if (base + 32 >= nt) break;  // (not reached)
            off -= __shfl_sync(0xffffffffu, incl, 31);
        }
        it = tc_item(a, s, rt);
    }
    // numbers of this item in the share
    __device__ __forceinline__ int here(const PagedShare &sh) const {
        const int64_t left = sh.u1 - pos;
        return (int)(left < it.size - at ? left : it.size - at);
    }
    __device__ __forceinline__ void next(const PagedArgs &a, const PagedShare &sh) {
        pos += here(sh);
        at = 0;
        if (pos >= sh.u1) return;
        if (++rt == nt) {
            rt = 0;
            if (++head == a.hkv) {
                b++;
                enter(a, sh.min_pos);
                return;
            }
        }
        it = tc_item(a, s, rt);
    }
};

// Named barriers of the two softmax warps that share a scheduler: TC_TURN_BAR + 2 (warp & 3) + stream.
constexpr int TC_TURN_BAR = 2;
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void pair_arrive(int id) { asm volatile("bar.arrive %0, 64;" ::"r"(id) : "memory"); }

template <int D, bool BF16>
__global__ void __launch_bounds__(TC_THREADS, 1) paged_tc_kernel(const __grid_constant__ PagedArgs a, const __grid_constant__ CUtensorMap kmap,
                                                                 const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap qmap,
                                                                 int box_rows) {
    using C = TcCfg<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = smem_u32(smem);
    const uint32_t bars = base + C::BAR_AT;
    const uint32_t kv_full = bars, kv_empty = kv_full + 8 * C::SLOTS, q_full = kv_empty + 8 * C::SLOTS, s_full = q_full + 16, p_full = s_full + 32,
                   o_full = p_full + 32, q_empty = o_full + 16, fix_bar = q_empty + 16, seg_full = fix_bar + 8, seg_empty = seg_full + 8 * TC_SEGS;
    float2 *ml = reinterpret_cast<float2 *>(smem + C::ML_AT);
    TcSeg *segs = reinterpret_cast<TcSeg *>(smem + C::SEG_AT);
    int64_t *red = reinterpret_cast<int64_t *>(smem + C::MISC_AT);
    volatile uint32_t *slot_word = reinterpret_cast<volatile uint32_t *>(smem + C::MISC_AT + 16 * 8);
    TcSplit *splits = reinterpret_cast<TcSplit *>(a.counters);
    if (tid == 0) {
        tma_prefetch(&kmap);
        tma_prefetch(&vmap);
        tma_prefetch(&qmap);
        for (int i = 0; i < C::SLOTS; i++) {
            mbar_init(kv_full + 8 * i, 1);
            mbar_init(kv_empty + 8 * i, 2);  // one arrival per stream
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(q_full + 8 * i, 1);
            mbar_init(q_empty + 8 * i, 1);
            for (int h = 0; h < 2; h++) {
                mbar_init(s_full + 8 * (2 * i + h), 1);
                mbar_init(p_full + 8 * (2 * i + h), 4);
            }
            mbar_init(o_full + 8 * i, 1);
        }
        mbar_init(fix_bar, 1);
        for (int i = 0; i < TC_SEGS; i++) {
            mbar_init(seg_full + 8 * i, 1);
            mbar_init(seg_empty + 8 * i, TC_SEG_READERS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    grid_launch_dependents();
    grid_dependency_wait();
    const PagedShare sh = paged_share<TC_THREADS, TC_PAIR_WEIGHT>(a, red, [&](int b, bool ok, int min_pos) -> int64_t {
        PagedSeq s{};
        if (ok) s = paged_seq(a, b, min_pos);
        const int nt = ok ? tc_tiles(a, s.n) : 0;
        int64_t units = 0;
        if (nt <= 2)
            for (int rt = 0; rt < nt; rt++) units += tc_item(a, s, rt).size;
        // long prompts: the warp's lanes share the row tiles
        for (unsigned many = __ballot_sync(0xffffffffu, nt > 2); many; many &= many - 1) {
            const int l = __ffs(many) - 1;
            PagedSeq t;
            t.q0 = 0;
            t.n = __shfl_sync(0xffffffffu, s.n, l);
            t.pos0 = __shfl_sync(0xffffffffu, s.pos0, l);
            t.key_end = __shfl_sync(0xffffffffu, s.key_end, l);
            t.lo = __shfl_sync(0xffffffffu, s.lo, l);
            t.sink = __shfl_sync(0xffffffffu, s.sink, l);
            const int64_t sum = tc_seq_units(a, t, lane);
            if (lane == l) units = sum;
        }
        return units * a.hkv;
    });
    if (sh.u0 >= sh.u1) {
        if (tid == 0) splits[blockIdx.x].rows = 0;
        return;
    }
    if (warp == TC_MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void *)slot_word)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot_word;

    // a reader's next record, and its release
    auto seg_wait = [&](int k) { return tc_wait(seg_full + 8 * (k % TC_SEGS), (uint32_t)((k / TC_SEGS) & 1), a.status); };
    auto seg_done = [&](int k) {
        __syncwarp();
        if (lane == 0) mbar_arrive(seg_empty + 8 * (k % TC_SEGS));
    };
    if (warp < TC_MMA_WARP) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TC_SOFTMAX_REGS));
        // ------------------------------------------------------------------------------------------ softmax: a thread per row
        const int st = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's quarter of the tensor memory's lanes
        const uint32_t tsc = tmem + C::S_COL + st * TC_UNIT + lanes, to = tmem + C::O_COL + st * D + lanes;
        const int r_tok = r / a.G, r_head = r - r_tok * a.G;
        const int base_pos = a.prefix_pass ? 0 : a.prefix_len;
        const uint64_t scale_2 = f2(a.scale2, a.scale2);
        bool alive = true;
        uint32_t halves = 0, par[2] = {0u, 0u};  // halves done so far; parities of the buffers
        if (st == 1) pair_arrive(TC_TURN_BAR + 2 * (warp & 3));  // stream 0 begins
        for (int k = 0; seg_wait(k); k++) {
            const TcSeg &g = segs[k % TC_SEGS];
            const int m = g.m;
            if (m == 0) break;
            const bool joint = !g.pair;   // both streams work on the same rows
            const int tok = g.tok0 + (joint ? 0 : st * tc_tokens(a)) + r_tok;
            const bool valid = r_tok < tc_tokens(a) && tok < g.n;
            int pos = -1;
            if (valid) pos = a.prefix_pass ? paged_row_pos(a, g.q0 + tok) : g.pos0 + tok;
            const int min_row = __reduce_min_sync(0xffffffffu, valid ? pos : INT_MAX), max_row = __reduce_max_sync(0xffffffffu, valid ? pos : -1);
            float mx = valid ? -INFINITY : 0.f, l = 0.f;  // maximum that the reference goes by (unscaled), and sum
            const int step = joint ? 2 : 1, first = joint ? st : 0;
            const uint32_t halves0 = halves;
            for (int i = first; i < m; i += step) {
                const int ui = g.unit + i, k_unit = (ui < g.u_sink ? ui : g.u_first + ui - g.u_sink) * TC_UNIT;
#pragma unroll 1
                for (int h = 0; h < 2; h++, halves++) {
                    const int k0 = k_unit + h * TC_HALF;
                    const uint32_t ts = tsc + h * TC_HALF;
                    if (alive) alive = tc_wait(s_full + 8 * (2 * st + h), par[h], a.status);
                    par[h] ^= 1u;
                    __syncwarp();
                    tc_fence_after();
                    float s[TC_HALF];
#pragma unroll
                    for (int c = 0; c < 2; c++) tc_ld32(ts + 32 * c, s + 32 * c);
#pragma unroll
                    for (int c = 0; c < 2; c++) tc_ld_wait32(s + 32 * c);
                    const int j0 = k0 + base_pos;
                    const bool whole = j0 + TC_HALF - 1 <= min_row && k0 + TC_HALF <= g.key_end && (a.window == 0 || j0 > max_row - a.window || j0 + TC_HALF <= a.sinks);
                    if (!whole) {
                        // key kk of the half is visible from `from` to `end` and below `sink`
                        const int end = min(pos - base_pos + 1, g.key_end) - k0, from = a.window > 0 ? pos - a.window + 1 - base_pos - k0 : INT_MIN,
                                  sink = a.sinks - base_pos - k0;
#pragma unroll
                        for (int kk = 0; kk < TC_HALF; kk++)
                            if (!(kk < end && (kk >= from || kk < sink))) s[kk] = -INFINITY;
                    }
                    // The weights are taken relative to the row's reference (`mx` less PAGED_BELOW), which follows the maximum only when they
                    // grow too large (by their sum: every weight is finite in f16, where 64 weights of 2^9 are 2^15): the maximum of 64
                    // scores costs a fifth of their softmax.
                    // The streams' exponentials take turns.  Each alone keeps the special-function unit busy (590 clocks for 64 rows' weights of a
                    // warp, 512 at the unit's rate); both at once take as long as one after the other, and then both wait for
                    // their next scores at once, the unit idle.  The turn passes on half way, which hides the hand-over (back to
                    // back, prompts of 8116 tokens: 308 us without turns, 291 with, 284 passing on half way; 24000 shared keys: 176, 170, 158).
                    if (!joint) pair_sync(TC_TURN_BAR + 2 * (warp & 3) + st);
                    float sum;
                    bool redo = mx == -INFINITY;
#pragma unroll 1
                    for (int turn = 0;; turn++) {
                        if (__any_sync(0xffffffffu, redo)) {
                            float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                            for (int kk = 4; kk < TC_HALF - 4; kk += 8)
#pragma unroll
                                for (int x = 0; x < 4; x++) tops[x] = max3(tops[x], s[kk + x], s[kk + 4 + x]);
#pragma unroll
                            for (int x = 0; x < 4; x++) tops[x] = fmaxf(tops[x], s[TC_HALF - 4 + x]);
                            const float next = fmaxf(mx, fmaxf(max3(tops[0], tops[1], tops[2]), tops[3])), f = mx == -INFINITY ? 0.f : ex2((mx - next) * a.scale2);
                            mx = next;
                            l *= f;
                            tc_st_wait();
                            if (halves != halves0) {  // (the first half starts the accumulator)
                                if (alive) alive = tc_wait(o_full + 8 * st, (halves - 1) & 1, a.status);
                                __syncwarp();
                                tc_fence_after();
#pragma unroll 1
                                for (int c = 0; c < D / 16; c++) {
                                    float o[16];
                                    tc_ld16(to + 16 * c, o);
                                    uint32_t q[16];
#pragma unroll
                                    for (int x = 0; x < 16; x++) q[x] = __float_as_uint(o[x] * f);
                                    tc_st16(to + 16 * c, q);
                                }
                            }
                        }
                        const float off = mx == -INFINITY ? 0.f : fmaf(-mx, a.scale2, PAGED_BELOW<BF16>);
                        const uint64_t off_2 = f2(off, off);
                        uint64_t sums[2] = {0ull, 0ull};
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            uint32_t q[16];
#pragma unroll
                            for (int x = 0; x < 16; x++) {
                                float e0, e1;
                                f2_split(fma2(f2(s[32 * c + 2 * x], s[32 * c + 2 * x + 1]), scale_2, off_2), e0, e1);
                                e0 = ex2(e0);
                                e1 = ex2(e1);
                                sums[x & 1] = add2(sums[x & 1], f2(e0, e1));
                                q[x] = pack2<BF16>(e0, e1);
                            }
                            tc_st16(ts + 16 * c, q);
                            if (c == 0 && turn == 0 && !joint) pair_arrive(TC_TURN_BAR + 2 * (warp & 3) + 1 - st);
                        }
                        float x, y;
                        f2_split(add2(sums[0], sums[1]), x, y);
                        sum = x + y;
                        redo = valid && !(sum <= (BF16 ? 32768.f : 61440.f));  // (rows of no token hold anything)
                        if (turn > 0 || !__any_sync(0xffffffffu, redo)) break;
                    }
                    l += sum;
                    tc_st_wait();
                    // A parity tells a phase only from its neighbours, so the last product is waited for from the one before it, which is
                    // waited for here, where the last one cannot be under way yet.
                    if (h == 1 && i + step >= m && alive) alive = tc_wait(o_full + 8 * st, (halves - 1) & 1, a.status);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full + 8 * (2 * st + h));
                }
            }
            // ---- results ----
            if (first < m && alive) alive = tc_wait(o_full + 8 * st, (halves - 1) & 1, a.status);
            __syncwarp();
            tc_fence_after();
            const float m2 = mx == -INFINITY ? -INFINITY : -fmaf(-mx, a.scale2, PAGED_BELOW<BF16>);  // the reference in log2
            const bool complete = g.complete;
            const int token = g.q0 + tok, head = g.head * a.G + r_head;
            float M = m2, L = l, f0 = 1.f, f1 = 0.f;
            if (joint) {
                ml[st * TC_ROWS + r] = make_float2(m2, l);
                tc_fence_before();
                named_barrier(1, TC_SOFTMAX_THREADS);
                tc_fence_after();
                const float2 x = ml[r], y = ml[TC_ROWS + r];
                M = fmaxf(x.x, y.x);
                f0 = x.x == -INFINITY ? 0.f : ex2(x.x - M);
                f1 = y.x == -INFINITY ? 0.f : ex2(y.x - M);
                L = x.y * f0 + y.y * f1;
            }
            // what the row's accumulator is multiplied by (0: the other stream's too), and its share of the shared prefix's result
            float w0 = f0, w1 = f1, wp = 0.f;
            if (complete) {
                float inv = L > 0.f ? 1.f / L : 0.f;
                if (a.prefix_pass) {
                    if (valid && (!joint || st == 0)) a.pre_lse[(int64_t)token * a.hq + head] = L > 0.f ? M + log2f(L) : -INFINITY;
                } else if (a.pre_o != nullptr && valid) {
                    const float lse = a.pre_lse[(int64_t)token * a.hq + head];
                    if (lse != -INFINITY) {
                        const float top = fmaxf(M, lse), own = M == -INFINITY ? 0.f : ex2(M - top), pre = ex2(lse - top);
                        inv = 1.f / (L * own + pre);
                        wp = pre * inv;
                        inv *= own;
                    }
                }
                w0 *= inv;
                w1 *= inv;
            }
            float *part = a.part + (int64_t)g.slot * TC_ITEM_ROWS * (D + 2);
            if (!complete && valid && (!joint || st == 0))
                *reinterpret_cast<float2 *>(part + (int64_t)TC_ITEM_ROWS * D + 2 * (joint ? r : st * TC_ROWS + r)) = make_float2(M, L);
            // 32 columns at a time through the warp's 4 KB (16-byte chunks, swizzled), then four rows of 128 bytes per instruction: a store by
            // the row's own thread would touch 32 lines.  Joint: each stream finishes half of the columns from both accumulators.
            const uint32_t stage = base + C::OUT_AT + (uint32_t)warp * 4096u;
            const int c_first = joint ? st * (D / 64) : 0, c_last = joint ? c_first + D / 64 : D / 32;
            const int my_token = valid ? token : -1, width = complete && !a.prefix_pass ? 2 : 4;
            uint8_t *dst[8];    // where this lane's part of rows 4 e + lane / 8 goes
            float pw[8];
            int prow[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int rr = 4 * e + (lane >> 3), t = __shfl_sync(0xffffffffu, my_token, rr), hd = __shfl_sync(0xffffffffu, head, rr);
                pw[e] = __shfl_sync(0xffffffffu, wp, rr);
                prow[e] = t * a.hq + hd;
                uint8_t *row;
                if (!complete) row = reinterpret_cast<uint8_t *>(part + (int64_t)((joint ? 0 : st * TC_ROWS) + (warp & 3) * 32 + rr) * D);
                else if (a.prefix_pass) row = reinterpret_cast<uint8_t *>(a.pre_o + (int64_t)prow[e] * D);
                else row = reinterpret_cast<uint8_t *>(reinterpret_cast<uint16_t *>(a.out) + (int64_t)t * a.ld_out + (int64_t)hd * D);
                dst[e] = t < 0 ? nullptr : row + 4 * (lane & 7) * width;
            }
            const bool with_prefix = __any_sync(0xffffffffu, wp != 0.f);
#pragma unroll 1
            for (int c = c_first; c < c_last; c++) {
                float o[32];
                tc_ld32(joint ? tmem + C::O_COL + lanes + 32 * c : to + 32 * c, o);
                tc_ld_wait32(o);
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] *= w0;
                if (joint && m > 1) {
                    float x[32];
                    tc_ld32(tmem + C::O_COL + D + lanes + 32 * c, x);
                    tc_ld_wait32(x);
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = fmaf(x[e], w1, o[e]);
                }
#pragma unroll
                for (int e = 0; e < 8; e++) sts128f<0>(stage + lane * 128 + ((e ^ (lane & 7)) << 4), o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                __syncwarp();
                float4 v[8];
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = lds128f<0>(stage + (4 * e + (lane >> 3)) * 128 + (((lane & 7) ^ ((4 * e + (lane >> 3)) & 7)) << 4));
                if (with_prefix) {
                    float4 x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (dst[e] != nullptr && pw[e] != 0.f) x[e] = *reinterpret_cast<const float4 *>(a.pre_o + (int64_t)prow[e] * D + 32 * c + 4 * (lane & 7));
                        else x[e] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        v[e] = make_float4(fmaf(x[e].x, pw[e], v[e].x), fmaf(x[e].y, pw[e], v[e].y), fmaf(x[e].z, pw[e], v[e].z), fmaf(x[e].w, pw[e], v[e].w));
                }
                if (width == 2) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (dst[e] != nullptr) *reinterpret_cast<uint2 *>(dst[e] + 64 * c) = make_uint2(pack2<BF16>(v[e].x, v[e].y), pack2<BF16>(v[e].z, v[e].w));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (dst[e] != nullptr) *reinterpret_cast<float4 *>(dst[e] + 128 * c) = v[e];
                }
                __syncwarp();
            }
            tc_fence_before();
            if (joint) named_barrier(1, TC_SOFTMAX_THREADS);  // the exchange and the other's accumulator are used again
            seg_done(k);
        }
        if (st == 0) pair_sync(TC_TURN_BAR + 2 * (warp & 3));    // stream 1's last arrival
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TC_OTHER_REGS));
        if (warp == TC_TMA_WARP) {
        // ------------------------------------------------------------------------------------------ copies of the pages
        int n = 0;  // slots filled so far
        bool alive = true;
        uint32_t fix_par = 0;
        const int page_mask = (1 << a.page_shift) - 1;
        // K and V of a unit into the next two slots: boxes of box_rows slots of one page.  Boxes that no row sees are left out of K
        // (their scores are masked) and are zeros in V; rows of a page that no row sees are zeroed in V, where a weight of zero would
        // meet them.  One warp's instruction latency bounds this loop, so what can be shared between K and V is.
        int cache_first = 0, page_cache = 0;  // lane i: page number cache_first + i of the item's table
        const int boxes = TC_UNIT / box_rows, box_bytes = box_rows * 128;
        for (int k = 0; seg_wait(k); k++) {
            const TcSeg &g = segs[k % TC_SEGS];
            const int m = g.m, u0 = g.unit, u_sink = g.u_sink, u_first = g.u_first, key_end = g.key_end, lo = g.lo, sink = g.sink, head = g.head, seq = g.b;
            if (m == 0) break;
            seg_done(k);
            bool cached = false;  // (the entries are those of this item's keys: the next one of the sequence sees further)
            auto visible = [&](int from, int rows) { return from < key_end && (from + rows > lo || from < sink); };
#pragma unroll 1
            for (int i = u0; i < u0 + m; i++) {
                const int k0 = (i < u_sink ? i : u_first + i - u_sink) * TC_UNIT, idx = k0 >> a.page_shift;
                if (!cached || idx < cache_first || idx + boxes > cache_first + 32) {
                    cached = true;
                    cache_first = idx;
                    const int at = idx + lane;
                    page_cache = a.n_pages;  // beyond the last page: zeros
                    if (at <= (key_end - 1) >> a.page_shift) {
                        page_cache = a.prefix_pass ? a.prefix_table[at] : a.block_table[(int64_t)seq * a.ld_table + at];
                        if (page_cache < 0 || page_cache >= a.n_pages) {
                            page_cache = a.n_pages;
                            if (visible(at << a.page_shift, page_mask + 1)) atomicOr(a.status, PAGED_BAD_INDEX);
                        }
                    }
                }
                const int mine = __shfl_sync(0xffffffffu, page_cache, (idx - cache_first + lane) & 31);
                const uint32_t seen = __ballot_sync(0xffffffffu, lane < boxes && visible(k0 + lane * box_rows, box_rows));
                const int page = seen >> lane & 1u ? mine : a.n_pages;
                const bool edge = k0 + TC_UNIT > key_end || (k0 < lo && k0 + TC_UNIT > sink);
                // (four boxes at a time: a launch begins with cold instruction caches, and all sixteen copies unrolled took 10000 clocks for the
                // first unit; one by one, pages of 16 slots keep the products waiting)
#pragma unroll 1
                for (int kv = 0; kv < 2; kv++, n++) {
                    const uint32_t slot = base + C::RING_AT + (uint32_t)(n % C::SLOTS) * C::SLOT_BYTES, full = kv_full + 8 * (n % C::SLOTS);
                    const uint32_t wanted = kv == 0 ? seen : (1u << boxes) - 1u;
                    const bool fix = kv == 1 && edge;
                    const uint32_t bar = fix ? fix_bar : full;
                    const CUtensorMap *map = kv == 0 ? &kmap : &vmap;
                    if (n >= C::SLOTS && alive) alive = tc_wait(kv_empty + 8 * (n % C::SLOTS), (uint32_t)((n / C::SLOTS - 1) & 1), a.status);
                    __syncwarp();
                    if (elect_one()) {
                        if (wanted) mbar_expect_tx(bar, (uint32_t)(__popc(wanted) * box_bytes * C::HALVES));
                        else mbar_arrive(bar);
                    }
                    __syncwarp();
#pragma unroll 1
                    for (int r0 = 0; r0 < boxes; r0 += 4) {
                        int pg[4];
#pragma unroll
                        for (int r = 0; r < 4; r++) pg[r] = __shfl_sync(0xffffffffu, page, r0 + r);
                        if (elect_one()) {
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                if (wanted >> (r0 + r) & 1u) {
#pragma unroll
                                    for (int h = 0; h < C::HALVES; h++)
                                        tma_load_page(slot + (uint32_t)(h * C::HALF_BYTES + (r0 + r) * box_bytes), map, 64 * h, (k0 + (r0 + r) * box_rows) & page_mask, head,
                                                      pg[r], bar);
                                }
                        }
                        __syncwarp();
                    }
                    if (fix) {
                        if (alive) alive = tc_wait(fix_bar, fix_par, a.status);
                        fix_par ^= 1u;
                        for (int r = lane / 8; r < TC_UNIT; r += 4) {
                            const int key = k0 + r;
                            if (key >= key_end || (key < lo && key >= sink)) {
#pragma unroll
                                for (int h = 0; h < C::HALVES; h++) sts128<0>(slot + (uint32_t)(h * C::HALF_BYTES + r * 128 + (lane & 7) * 16), 0u, 0u, 0u, 0u);
                            }
                        }
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(full);
                    }
                }
            }
        }
        // the last copies have landed before the CTA may end: the product warps wait for every fill
    } else if (warp == TC_MMA_WARP || warp == TC_MMA1_WARP) {
        // ------------------------------------------------------------------------------------------ products of a stream
        const int st = warp == TC_MMA_WARP ? 0 : 1;
        bool alive = true;
        int n = 0, seen = 0;             // fills of the ring: of earlier items; that this warp has seen
        uint32_t q_par = 0u, p_par[2] = {0u, 0u};
        constexpr uint32_t idesc_s = tc_idesc<BF16>(TC_HALF, false), idesc_o = tc_idesc<BF16>(D, true);
        const uint32_t sc = tmem + C::S_COL + st * TC_UNIT, o = tmem + C::O_COL + st * D;
        const uint64_t qd = smem_desc_sw128(base + (uint32_t)st * C::SLOT_BYTES);
        auto slot_addr = [&](int i) { return base + C::RING_AT + (uint32_t)(i % C::SLOTS) * C::SLOT_BYTES; };
        for (int k = 0; seg_wait(k); k++) {
            const TcSeg &g = segs[k % TC_SEGS];
            const int m = g.m;
            if (m == 0) break;
            const bool pair = g.pair;
            seg_done(k);
            // A parity tells a phase only from its neighbours: each of the two warps sees every fill of the ring in turn, and lets go of the
            // other stream's at once (a warp that skipped them would take the copy before its own for it, where that one is still under
            // way and the streams' slots have changed places).  They have been asked for before the warp's own next one: no time lost.
            auto see = [&](int last) {
                for (; seen <= last; seen++) {
                    if (alive) alive = tc_wait(kv_full + 8 * (seen % C::SLOTS), (uint32_t)((seen / C::SLOTS) & 1), a.status);
                    if (!pair && (((seen - n) >> 1) & 1) != st) {
                        __syncwarp();  // (no lane still asks for this phase)
                        if (lane == 0) mbar_arrive(kv_empty + 8 * (seen % C::SLOTS));
                    }
                }
            };
            // slots in the order of the copies: K V K V ...
            auto k_slot = [&](int i) { return n + 2 * i; };
            auto v_slot = [&](int i) { return n + 2 * i + 1; };
            const int first = pair ? 0 : st, step = pair ? 1 : 2;
            if (first < m) {
                if (alive) alive = tc_wait(q_full + 8 * st, q_par, a.status);
                q_par ^= 1u;
            }
            for (int i = first - step; i < m; i += step) {
                // half by half: O += P V of unit i, then S = Q K^T of the next one into the same buffer
                const bool with_v = i >= first, with_k = i + step < m;
                const int vs = with_v ? v_slot(i) : 0, ks = with_k ? k_slot(i + step) : 0;
                if (with_v) see(vs);
                if (with_k) see(ks);
#pragma unroll 1
                for (int h = 0; h < 2; h++) {
                    if (with_v) {
                        if (alive) alive = tc_wait(p_full + 8 * (2 * st + h), p_par[h], a.status);
                        p_par[h] ^= 1u;
                    }
                    __syncwarp();
                    tc_fence_after();
                    if (elect_one()) {
                        if (with_v) {
                            const uint64_t vd = tc_desc_v(slot_addr(vs) + (uint32_t)(h * TC_HALF * 128), C::HALF_BYTES);
#pragma unroll
                            for (int kk = 0; kk < TC_HALF / 16; kk++)
                                tc_mma_ts(o, sc + h * TC_HALF + 8 * kk, vd + (uint64_t)((kk * 2048) >> 4), idesc_o, i == first && h + kk == 0 ? 0u : 1u);
                            umma_commit(o_full + 8 * st);
                            if (h == 1) umma_commit(kv_empty + 8 * (vs % C::SLOTS));
                        }
                        if (with_k) {
                            const uint64_t kd = smem_desc_sw128(slot_addr(ks) + (uint32_t)(h * TC_HALF * 128));
#pragma unroll
                            for (int x = 0; x < C::HALVES; x++)
#pragma unroll
                                for (int kk = 0; kk < 4; kk++)
                                    tc_mma_ss(sc + h * TC_HALF, qd + (uint64_t)(x * (C::HALF_BYTES >> 4) + 2 * kk), kd + (uint64_t)(x * (C::HALF_BYTES >> 4) + 2 * kk),
                                              idesc_s, x + kk > 0 ? 1u : 0u);
                            umma_commit(s_full + 8 * (2 * st + h));
                            if (h == 1) {
                                if (i + 2 * step >= m) umma_commit(q_empty + 8 * st);
                                umma_commit(kv_empty + 8 * (ks % C::SLOTS));
                            }
                        }
                    }
                    __syncwarp();
                }
            }
            see(n + 2 * m - 1);
            n += 2 * m;
        }
    } else if (warp == TC_WALK_WARP) {
        // ------------------------------------------------------------------------------------------ the batch, item by item
        TcWalk w;
        w.start(a, sh, lane);
        if (lane == 0) splits[blockIdx.x].rows = 0;
        bool alive = true;
        int used[2] = {0, 0};
        const uint32_t bytes = (uint32_t)(tc_tokens(a) * a.G * 128 * C::HALVES);
        // Queries of item k, once the scores of the last item are complete (the record of the one after it comes in time for the copies of
        // its pages: with the scores of this one still to be made).  A stream without a unit gets none.
        auto queries = [&](int k) {
            const TcSeg &g = segs[k % TC_SEGS];
            for (int st = 0; st < (g.m == 0 ? 0 : (g.pair || g.m > 1 ? 2 : 1)); st++) {
                if (used[st] > 0 && alive) alive = tc_wait(q_empty + 8 * st, (uint32_t)((used[st] - 1) & 1), a.status);
                used[st]++;
                __syncwarp();
                if (elect_one()) {
                    mbar_expect_tx(q_full + 8 * st, bytes);
#pragma unroll
                    for (int h = 0; h < C::HALVES; h++)
                        tma_load_rows(base + (uint32_t)(st * C::SLOT_BYTES + h * C::HALF_BYTES), &qmap, 64 * h, g.head * a.G,
                                      g.q0 + g.tok0 + (g.pair ? st * tc_tokens(a) : 0), q_full + 8 * st);
                }
                __syncwarp();
            }
        };
        for (int k = 0;;) {
            const bool end = w.pos >= sh.u1;
            const int first = end ? 0 : w.it.units_before(w.at), units = end ? 0 : w.it.units_before(w.at + w.here(sh)) - first;
            if (!end && units == 0) {  // (only numbers that stand for no unit)
                w.next(a, sh);
                continue;
            }
            if (k >= TC_SEGS && alive) alive = tc_wait(seg_empty + 8 * (k % TC_SEGS), (uint32_t)((k / TC_SEGS - 1) & 1), a.status);
            if (!alive) break;
            if (lane == 0) {
                TcSeg g{};
                if (!end) {
                    g.m = units;
                    g.unit = first; g.u_sink = w.it.u.sink; g.u_first = w.it.u.first;
                    g.key_end = w.it.k.key_end; g.lo = w.it.k.lo; g.sink = w.it.k.sink;
                    g.pair = w.it.tokens > tc_tokens(a);
                    g.tok0 = w.it.tok0; g.n = w.s.n;
                    g.b = w.b; g.head = w.head; g.q0 = w.s.q0; g.pos0 = w.s.pos0;
                    g.complete = units == w.it.u.count;
                    g.slot = 2 * (int)blockIdx.x + (first == 0 ? 1 : 0);
                }
                segs[k % TC_SEGS] = g;
                mbar_arrive(seg_full + 8 * (k % TC_SEGS));
            }
            __syncwarp();
            if (end) break;
            queries(k);
            // an item that begins here and goes on elsewhere is the share's last
            if (lane == 0 && first == 0 && units < w.it.u.count)
                splits[blockIdx.x] = {paged_owner(w.pos - w.at + TC_ITEM_WEIGHT + ((int64_t)(w.it.u.count - 1) << w.it.shift), sh.total, sh.N),
                                      w.it.tokens > tc_tokens(a) ? TC_ITEM_ROWS : TC_ROWS, w.it.tok0, w.s.n, w.s.q0, w.head};
            w.next(a, sh);
            k++;
        }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == TC_MMA_WARP)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// Joins the parts of the items that share borders have cut: CTA (c, y) takes 256 groups of eight results of the item that begins in
// share c, one thread each.  A launch of its own, since a single CTA reads the parts of a widely cut item (two hundred rows against a
// long prefix: 2 MB) at a hundred GB/s: 95 us of 187 us when the last CTA to arrive did it (48 decode rows, prefix of 12345).
constexpr int TC_JOIN_THREADS = 256, TC_JOIN_PARTS = 160;  // (a grid has no more CTAs than an item may have parts; the card: 148)
template <int D, bool BF16>
__global__ void __launch_bounds__(TC_JOIN_THREADS) paged_tc_join_kernel(const __grid_constant__ PagedArgs a) {
    grid_launch_dependents();
    grid_dependency_wait();
    constexpr int PER_ROW = D / 8, ROWS = TC_JOIN_THREADS / PER_ROW;
    __shared__ float2 w_s[TC_JOIN_PARTS][ROWS];  // a part's weight for a row, and its weighted sum
    const int c0 = blockIdx.x;
    const TcSplit sp = reinterpret_cast<const TcSplit *>(a.counters)[c0];
    const int first_row = blockIdx.y * ROWS, lr = threadIdx.x / PER_ROW, r = first_row + lr, lane = threadIdx.x % PER_ROW, col = lane * 8;
    if (first_row >= sp.rows) return;
    const int parts = sp.c1 - c0 + 1;
    const int64_t pitch = (int64_t)TC_ITEM_ROWS * (D + 2);
    auto part_of = [&](int i) { return (int64_t)(2 * (c0 + i) + (i == 0 ? 1 : 0)) * pitch; };
    const int rr = r % TC_ROWS, t = paged_div(rr, a.G, a.inv_G), tok = sp.tok0 + r / TC_ROWS * tc_tokens(a) + t;
    const bool valid = t < tc_tokens(a) && tok < sp.n;
    float m, l = 0.f, v[8];
    // the threads of a row share the parts' maxima and sums, then every thread adds its columns with all loads in flight
    const float *ml = a.part + (int64_t)TC_ITEM_ROWS * D + 2 * r;
    const unsigned group = __activemask();  // (whole warps)
    m = -INFINITY;
    if (valid)
        for (int i = lane; i < parts; i += PER_ROW) {
            const float2 x = __ldcg(reinterpret_cast<const float2 *>(ml + part_of(i)));
            w_s[i][lr] = x;
            m = fmaxf(m, x.x);
        }
#pragma unroll
    for (int o = PER_ROW / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(group, m, o));
    if (valid)
        for (int i = lane; i < parts; i += PER_ROW) {
            const float2 x = w_s[i][lr];
            const float w = x.x == -INFINITY ? 0.f : ex2(x.x - m);
            w_s[i][lr].x = w;
            w_s[i][lr].y = x.y * w;
        }
    __syncwarp();
#pragma unroll
    for (int x = 0; x < 8; x++) v[x] = 0.f;
    if (!valid) return;
    const float *o = a.part + (int64_t)r * D + col;
#pragma unroll 8
    for (int i = 0; i < parts; i++) {
        const float4 x = __ldcg(reinterpret_cast<const float4 *>(o + part_of(i))), y = __ldcg(reinterpret_cast<const float4 *>(o + part_of(i) + 4));
        const float w = w_s[i][lr].x;
        l += w_s[i][lr].y;
        v[0] = fmaf(w, x.x, v[0]); v[1] = fmaf(w, x.y, v[1]); v[2] = fmaf(w, x.z, v[2]); v[3] = fmaf(w, x.w, v[3]);
        v[4] = fmaf(w, y.x, v[4]); v[5] = fmaf(w, y.y, v[5]); v[6] = fmaf(w, y.z, v[6]); v[7] = fmaf(w, y.w, v[7]);
    }
    paged_finish8<BF16>(a, D, sp.q0 + tok, sp.head * a.G + (rr - t * a.G), col, m, l, v);
}

template <int D, bool BF16>
cudaError_t launch_tc_t(const PagedArgs &a, const PagedMaps &maps, int box_rows, cudaStream_t st) {
    using C = TcCfg<D>;
    static_assert(C::SMEM <= 227 * 1024, "shared memory of a CTA");
    auto kernel = paged_tc_kernel<D, BF16>;
    static OncePerDevice once;
    const cudaError_t e = once([&]() { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM); });
    if (e != cudaSuccess) return e;
    const unsigned ctas = (unsigned)(a.sms < TC_JOIN_PARTS ? a.sms : TC_JOIN_PARTS);
    const cudaError_t r = launch_pdl(kernel, dim3(ctas), dim3(TC_THREADS), C::SMEM, st, a, maps.k, maps.v, maps.q, box_rows);
    if (r != cudaSuccess) return r;
    return launch_pdl(paged_tc_join_kernel<D, BF16>, dim3(ctas, TC_ITEM_ROWS * D / 8 / TC_JOIN_THREADS), dim3(TC_JOIN_THREADS), 0, st, a);
}

}  // namespace

int64_t paged_tc_words(int sms) { return (int64_t)sms * (sizeof(TcSplit) / 4); }
int64_t paged_tc_part_floats(int d, int sms) { return (int64_t)2 * sms * TC_ITEM_ROWS * (d + 2); }

cudaError_t launch_paged_tc(const PagedArgs &a, int dt, int d, const PagedMaps &maps, int box_rows, cudaStream_t st) {
    if (d == 128) return dt == TTQ_DT_BF16 ? launch_tc_t<128, true>(a, maps, box_rows, st) : launch_tc_t<128, false>(a, maps, box_rows, st);
    return dt == TTQ_DT_BF16 ? launch_tc_t<64, true>(a, maps, box_rows, st) : launch_tc_t<64, false>(a, maps, box_rows, st);
}

}  // namespace ttq
