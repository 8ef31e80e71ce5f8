// Sampling: the next token of every row of logits from given random numbers, with temperature, top-k, top-p and min-p.
//
// All three cuts keep a head of the same order (logit descending, index ascending), so a row's result needs no sort: the logit at which
// the head ends, and how many tokens with exactly this logit still belong to it.  Weights are w = exp((x - max) / T), computed
// in 64 bits and summed as 2^-44 fixed point: integer sums are exact, do not depend on the order of the atomics, and their rounding
// (2^-45 a token, where the largest weight is 1) is far below the weight of any token that decides a cut.  In 32 bits a cut among 10^5
// tokens of similar weight falls on a neighbour of the right one about once in 400 rows.
//
// A cluster of CTAs holds a row in shared memory, so the logits are read once.  The cut is found by histograms of counts or weights:
// first over 2048 equal parts of the range that has weight (max - 32 T to max: evenly spread logits, few collisions).  The tokens of the
// part with the cut, a few hundred, go to the first CTA, which goes on alone: each against each, or, above 512, histograms over the
// order-preserving keys, 2048 at a time, until a bin is one key.  (Only where a part holds more than LIST tokens do all CTAs go on, adding into the first
// one's histogram.)  Bound: one reading of the logits; in practice the 64-bit exponentials (58 clocks per 32 weights and
// scheduler, 22 of them for eleven 64-bit instructions at half the 32-bit rate) for large batches, the chain of cluster barriers for small ones.
#include <cooperative_groups.h>

#include "ttq_internal.cuh"

namespace ttq {
namespace {

namespace cg = cooperative_groups;

constexpr int SAMPLE_THREADS = 512;
constexpr int SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int BINS = 2048, BINS_PER_THREAD = BINS / SAMPLE_THREADS;
constexpr int LIST = 2048;     // tokens that the first CTA takes over
constexpr int PAIRS = 512;     // of which so many are compared pair by pair (a thread each)
constexpr int MAX_CLUSTER = 8;
constexpr double FIXED_ONE = 17592186044416.0;  // 2^44
constexpr float FIXED_RANGE = 32.f;              // exp(-32 * 2047 / 2048) < 2^-46: no weight in the last part
typedef unsigned long long u64;

struct SampleArgs {
    const void *logits;
    int dt, V, slice;
    int64_t ld;
    ttq_sampling s;
    const float *u;
    int64_t *ids;
};

// Order-preserving: larger float, larger key.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Shared {
    uint32_t lo[BINS], hi[BINS];    // this CTA's histogram; the first CTA's becomes the row's
    u64 list_w[PAIRS + 1];          // and their counts or weights
    uint32_t list[LIST + 1];        // keys of the tokens that decide (first CTA)
    double table[512];              // 2^(j / 512)
    u64 warp_sum[SAMPLE_WARPS];
    // exchanged between the CTAs of a row
    u64 best, mass;
    uint32_t kmin, range_lo, range_hi;
    int ties;
    // a level's result (first CTA)
    u64 found_before, found_mass;
    int found_bin, list_n;
    // a descent's (first CTA)
    uint32_t cut_key;
    u64 cut_inside, cut_all;
    int cut_found;
};

template <class T>
__device__ __forceinline__ T warp_inclusive(T v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}
// Sum of v over lower-numbered threads; `all`: over every thread.
__device__ __forceinline__ u64 block_exclusive(u64 v, u64 *warp_sums, u64 &all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const u64 incl = warp_inclusive(v);
    __syncthreads();
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    const u64 w = lane < SAMPLE_WARPS ? warp_sums[lane] : 0, wi = warp_inclusive(w);
    all = __shfl_sync(0xffffffffu, wi, SAMPLE_WARPS - 1);
    return __shfl_sync(0xffffffffu, wi - w, warp) + incl - v;
}
__device__ __forceinline__ void add_u64(uint32_t *lo, uint32_t *hi, u64 v) {
    const uint32_t l = (uint32_t)v, old = atomicAdd(lo, l);
    const uint32_t h = (uint32_t)(v >> 32) + (old + l < old ? 1u : 0u);
    if (h) atomicAdd(hi, h);
}

// exp((x - max) / T) in 2^-44 fixed point.  2^y with y = 512ths + r: a table and the series of 2^r to r^3 (|r| <= 2^-10: 9e-15 of the
// weight).  64-bit instructions run at half the rate of 32-bit ones and conversions slower, so the
// logit is widened by integer instructions and the range is checked in 32 bits: beyond -46 the weight is zero either way.
constexpr int TABLE = 512;
struct Weigher {
    float xmax, scale32;
    double dmax, scale;  // log2(e) / T
    const double *table;
    __device__ __forceinline__ u64 operator()(float x) const {
        const uint32_t b = __float_as_uint(x);
        const double xd = __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(b << 29));  // (below 2^-126: below 2^-126)
        const double y = (xd - dmax) * scale;
        constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer in the low bits
        const double kd = fma(y, (double)TABLE, MAGIC);
        const int k = __double2loint(kd);
        const double r = fma(kd - MAGIC, -1.0 / TABLE, y);
        double p = fma(r, 5.5504108664821580e-2, 2.4022650695910072e-1);  // ln(2)^n / n!
        p = fma(p, r, 6.9314718055994531e-1);
        p = fma(p, r, 1.0) * table[k & (TABLE - 1)];
        const double v = __hiloint2double(__double2hiint(p) + (((k >> 9) + 44) << 20), __double2loint(p)) + 4503599627370496.0;  // + 2^52
        const u64 w = (u64)__double_as_longlong(v) & 0xfffffffffffffull;
        return x == xmax ? (u64)FIXED_ONE : ((x - xmax) * scale32 > -46.f ? w : 0);
    }
};

__global__ void __launch_bounds__(SAMPLE_THREADS, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Shared &sh = *reinterpret_cast<Shared *>(smem_raw);
    float *xs = reinterpret_cast<float *>(smem_raw + sizeof(Shared));
    cg::cluster_group cluster = cg::this_cluster();
    const int CS = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    Shared &first = *cluster.map_shared_rank(&sh, 0);
    auto cluster_sync = [&]() {
        if (CS == 1) __syncthreads();
        else cluster.sync();
    };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t row = blockIdx.x / CS;
    const int V = a.V, i_first = rank * a.slice, n = max(0, min(a.slice, V - i_first));
    static_assert(TABLE == SAMPLE_THREADS, "one entry per thread");
    sh.table[tid] = exp2((double)tid / TABLE);
    for (int i = tid; i < BINS; i += SAMPLE_THREADS) sh.lo[i] = sh.hi[i] = 0;
    if (tid == 0) {
        sh.best = 0;
        sh.kmin = 0xffffffffu;
        sh.list_n = 0;
    }
    grid_launch_dependents();
    grid_dependency_wait();
    const float temperature = a.s.temperature_dev ? a.s.temperature_dev[row] : a.s.temperature;
    const float top_p = a.s.top_p_dev ? a.s.top_p_dev[row] : a.s.top_p;
    const float min_p = a.s.min_p_dev ? a.s.min_p_dev[row] : a.s.min_p;
    int top_k = a.s.top_k_dev ? a.s.top_k_dev[row] : a.s.top_k;
    if (top_k <= 0 || top_k > V) top_k = V;

    // the row into shared memory (NaN as -inf, -0 as +0); its largest logit with the lowest index, and its smallest
    u64 best = 0;
    uint32_t kmin = 0xffffffffu;
    {
        auto take = [&](int i, float x) {
            x = x != x ? -INFINITY : x + 0.f;
            xs[i] = x;
            const uint32_t k = key_of(x);
            const u64 c = ((u64)k << 32) | (0xffffffffu - (uint32_t)(i_first + i));
            best = c > best ? c : best;
            if (x != -INFINITY) kmin = min(kmin, k);
        };
        // 16 bytes per load from the first aligned address on, all in flight together
        const int size = a.dt == TTQ_DT_F32 ? 4 : 2, per = 16 / size;
        const uint8_t *src = reinterpret_cast<const uint8_t *>(a.logits) + (row * a.ld + i_first) * size;
        const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / size), groups = (n - head) / per;
        if (tid < head) take(tid, load_as_float(src, a.dt, tid));
        if (tid < n - head - groups * per) take(head + groups * per + tid, load_as_float(src, a.dt, head + groups * per + tid));
        const uint4 *vec = reinterpret_cast<const uint4 *>(src + head * size);
        for (int g0 = tid; g0 < groups; g0 += 8 * SAMPLE_THREADS) {
            uint4 r[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (g0 + j * SAMPLE_THREADS < groups) r[j] = vec[g0 + j * SAMPLE_THREADS];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int g = g0 + j * SAMPLE_THREADS;
                if (g >= groups) break;
                if (size == 4) {
                    const uint32_t w[4] = {r[j].x, r[j].y, r[j].z, r[j].w};
#pragma unroll
                    for (int q = 0; q < 4; q++) take(head + 4 * g + q, __uint_as_float(w[q]));
                } else {
                    float f[8];
                    xh_unpack(r[j], a.dt, f);
#pragma unroll
                    for (int q = 0; q < 8; q++) take(head + 8 * g + q, f[q]);
                }
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 x = __shfl_xor_sync(0xffffffffu, best, o);
        best = x > best ? x : best;
    }
    kmin = __reduce_min_sync(0xffffffffu, kmin);
    __syncthreads();
    if (lane == 0) {
        atomicMax(&sh.best, best);
        atomicMin(&sh.kmin, kmin);
    }
    cluster_sync();
    {
        const Shared &o = *cluster.map_shared_rank(&sh, lane < CS ? lane : 0);
        best = o.best;
        kmin = __reduce_min_sync(0xffffffffu, o.kmin);
#pragma unroll
        for (int m = MAX_CLUSTER / 2; m > 0; m >>= 1) {
            const u64 x = __shfl_xor_sync(0xffffffffu, best, m);
            best = x > best ? x : best;
        }
        best = __shfl_sync(0xffffffffu, best, 0);
    }
    const uint32_t kmax = (uint32_t)(best >> 32);
    const float xmax = of_key(kmax);
    if (xmax == -INFINITY || !(temperature > 0.f)) {
        if (rank == 0 && tid == 0) a.ids[row] = xmax == -INFINITY ? -1 : (int)(0xffffffffu - (uint32_t)best);
        cluster_sync();  // (no CTA leaves while another may read its shared memory)
        return;
    }
    const double scale = 1.4426950408889634 / (double)temperature;
    const Weigher weight{xmax, (float)scale, (double)xmax, scale, sh.table};

    // Level 0: 2048 parts of the range from the largest logit down to the smallest, or to where weights vanish.  Monotone in x: a
    // difference, a product and a conversion, each rounded.  The last part also holds everything below.
    const float clip = FIXED_RANGE * temperature, range = fminf(clip, xmax - of_key(kmin)), per_part = fminf((float)BINS / range, 3e38f);
    auto place_of = [&](float x) { return x == xmax ? 0.f : (xmax - x) * per_part; };
    auto part_of = [&](float x) { return (int)fminf(place_of(x), (float)(BINS - 1)); };

    // every token of this CTA: f(logit, key), four at a time
    auto each_token = [&](auto &&f) {
        int i = tid;
        for (; i + 3 * SAMPLE_THREADS < n; i += 4 * SAMPLE_THREADS) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = xs[i + j * SAMPLE_THREADS];
#pragma unroll
            for (int j = 0; j < 4; j++) f(x[j], key_of(x[j]));
        }
        for (; i < n; i += SAMPLE_THREADS) f(xs[i], key_of(xs[i]));
    };
    // The first CTA: the bin of the row's histogram at which the running count or weight, from `before` on, reaches the target (-1:
    // none), and the histogram cleared.  `p` >= 0: the target is this part of the whole.
    auto scan = [&](bool by_mass, u64 before, u64 target_n, double &target, double p) {
        u64 v[BINS_PER_THREAD], mine = 0, all;
#pragma unroll
        for (int j = 0; j < BINS_PER_THREAD; j++) {
            const int b = BINS_PER_THREAD * tid + j;
            v[j] = ((u64)sh.hi[b] << 32) | sh.lo[b];
            sh.lo[b] = sh.hi[b] = 0;
            mine += v[j];
        }
        if (tid == 0) sh.found_bin = -1;
        u64 cum = before + block_exclusive(mine, sh.warp_sum, all);
        if (p >= 0.0) target = p * (double)all;
        auto reached = [&](u64 c) { return by_mass ? (double)c >= target : c >= target_n; };
#pragma unroll
        for (int j = 0; j < BINS_PER_THREAD; j++) {
            if (v[j] > 0 && reached(cum + v[j]) && !reached(cum)) {
                sh.found_bin = BINS_PER_THREAD * tid + j;
                sh.found_before = cum;
                sh.found_mass = v[j];
            }
            cum += v[j];
        }
        __syncthreads();
    };

    // One descent through the tokens with keys above `lim`, and `lim_n` of those equal to it: the key at which the running count
    // (by_mass false) or weight (true: p of the whole), from the top, reaches the target; how many tokens of this key are inside
    // and in all.  `few`: no more than LIST tokens are above `lim`.  False: the target is not reached before the weights vanish,
    // nothing is cut.
    auto descend = [&](bool by_mass, u64 target_n, double p, uint32_t lim, u64 lim_n, bool few, uint32_t &key, u64 &inside, u64 &in_all) -> bool {
        double target = 0.0;  // (the first CTA's)
        u64 before = 0;
        int part = -1;
        if (!few) {
            auto add = [&](float x, u64 copies) {
                const int bin = part_of(x);
                if (by_mass) add_u64(sh.lo + bin, sh.hi + bin, weight(x) * copies);
                else atomicAdd(sh.lo + bin, (uint32_t)copies);
            };
            each_token([&](float x, uint32_t k) {
                if (k > lim) add(x, 1);
            });
            if (lim_n > 0 && rank == 0 && tid == 0) add(of_key(lim), lim_n);
            __syncthreads();
            if (rank > 0)
                for (int i = tid; i < BINS; i += SAMPLE_THREADS) {
                    const uint32_t l = sh.lo[i], h = sh.hi[i];
                    if (l | h) {
                        add_u64(first.lo + i, first.hi + i, ((u64)h << 32) | l);
                        sh.lo[i] = sh.hi[i] = 0;
                    }
                }
            cluster_sync();
            if (rank == 0) scan(by_mass, 0, target_n, target, by_mass ? p : -1.0);
            cluster_sync();
            part = first.found_bin;
            before = first.found_before;
            if (part < 0 || (part == BINS - 1 && range == clip)) return false;
        }
        // the part's tokens to the first CTA
        const float from = part < 0 ? -1.f : (float)part, to = part < 0 || part == BINS - 1 ? INFINITY : (float)(part + 1);
        auto chosen = [&](float x, uint32_t k) {
            const float at = place_of(x);
            return k > lim && at >= from && !(at >= to && to < INFINITY);
        };
        each_token([&](float x, uint32_t k) {
            if (chosen(x, k)) {
                const int at = atomicAdd(&first.list_n, 1);
                if (at < LIST) first.list[at] = k;
            }
        });
        cluster_sync();
        const int listed = first.list_n;
        const bool alone = listed <= LIST, with_lim = lim_n > 0 && (part < 0 || part_of(of_key(lim)) == part);
        if (rank == 0 || !alone) {
            auto sync = [&]() {
                if (alone) __syncthreads();
                else cluster_sync();
            };
            if (alone && few && by_mass) {  // the whole has not been weighed yet
                u64 mine = 0, all;
                for (int i = tid; i < listed; i += SAMPLE_THREADS) mine += weight(of_key(sh.list[i]));
                if (tid == 0 && with_lim) mine += weight(of_key(lim)) * lim_n;
                block_exclusive(mine, sh.warp_sum, all);
                target = p * (double)all;
            }
            if (alone && listed <= PAIRS) {
                const int entries = listed + (with_lim ? 1 : 0);
                for (int i = tid; i < entries; i += SAMPLE_THREADS) {
                    const uint32_t k = i < listed ? sh.list[i] : lim;
                    const u64 copies = i < listed ? 1 : lim_n;
                    if (i == listed) sh.list[i] = lim;
                    sh.list_w[i] = by_mass ? weight(of_key(k)) * copies : copies;
                }
                if (tid == 0) sh.cut_found = 0;
                __syncthreads();
                for (int i = tid; i < entries; i += SAMPLE_THREADS) {
                    const uint32_t k = sh.list[i];
                    u64 above = before, same = 0;
                    int ties = 0;
#pragma unroll 4
                    for (int j = 0; j < entries; j++) {
                        const uint32_t kj = sh.list[j];
                        const u64 w = sh.list_w[j];
                        if (kj > k) above += w;
                        if (kj == k) same += w, ties++;
                    }
                    auto reached = [&](u64 c) { return by_mass ? (double)c >= target : c >= target_n; };
                    if (same > 0 && reached(above + same) && !reached(above)) {  // (one key; its ties write the same)
                        const u64 have = i < listed ? (u64)ties : lim_n;
                        sh.cut_key = k;
                        sh.cut_all = have;
                        if (by_mass) {
                            const double r = ceil((target - (double)above) / (double)(same / have));
                            sh.cut_inside = r < 1.0 ? 1 : (r > (double)have ? have : (u64)r);
                        } else {
                            sh.cut_inside = target_n - above;
                        }
                        sh.cut_found = 1;
                    }
                }
            } else {
            // keys in [bottom, top], 2048 bins of 2^shift keys at a time
            uint32_t klo = 0xffffffffu, khi = 0;
            auto tokens = [&](auto &&f) {
                if (alone)
                    for (int i = tid; i < listed; i += SAMPLE_THREADS) f(sh.list[i], (u64)1);
                else
                    each_token([&](float x, uint32_t k) {
                        if (chosen(x, k)) f(k, (u64)1);
                    });
                if (with_lim && rank == 0 && tid == 0) f(lim, lim_n);
            };
            tokens([&](uint32_t k, u64) {
                klo = min(klo, k);
                khi = max(khi, k);
            });
            if (rank == 0 && tid == 0) {
                sh.range_lo = 0xffffffffu;
                sh.range_hi = 0;
            }
            klo = __reduce_min_sync(0xffffffffu, klo);
            khi = __reduce_max_sync(0xffffffffu, khi);
            sync();
            if (lane == 0 && khi > 0) {
                atomicMin(&first.range_lo, klo);
                atomicMax(&first.range_hi, khi);
            }
            sync();
            uint32_t bottom = first.range_lo, top = first.range_hi;
            while (true) {
                int shift = 0;
                while (((top - bottom) >> shift) >= (uint32_t)BINS) shift++;
                tokens([&](uint32_t k, u64 copies) {
                    if (k > top || k < bottom) return;
                    const int bin = (int)((top - k) >> shift);
                    if (by_mass) add_u64(first.lo + bin, first.hi + bin, weight(of_key(k)) * copies);
                    else atomicAdd(first.lo + bin, (uint32_t)copies);
                });
                sync();
                if (rank == 0) scan(by_mass, before, target_n, target, -1.0);
                sync();
                const int bin = first.found_bin;
                if (bin >= 0) before = first.found_before;
                if (bin < 0 || shift == 0) {
                    if (rank == 0 && tid == 0) {
                        sh.cut_found = bin >= 0;
                        if (bin >= 0) {
                            const uint32_t k = top - (uint32_t)bin;
                            sh.cut_key = k;
                            if (by_mass) {
                                const u64 each = weight(of_key(k));  // (a bin with weight was found)
                                const u64 have = sh.found_mass / each;
                                const double r = ceil((target - (double)before) / (double)each);
                                sh.cut_all = have;
                                sh.cut_inside = r < 1.0 ? 1 : (r > (double)have ? have : (u64)r);
                            } else {
                                sh.cut_all = sh.found_mass;
                                sh.cut_inside = target_n - before;
                            }
                        }
                    }
                    break;
                }
                const uint32_t up = top - ((uint32_t)bin << shift), down = up - ((1u << shift) - 1u);
                bottom = down < bottom || down > up ? bottom : down;
                top = up;
                sync();  // (the result is written again)
            }
            }
        }
        cluster_sync();
        const bool found = first.cut_found != 0;
        key = first.cut_key;
        inside = first.cut_inside;
        in_all = first.cut_all;
        if (rank == 0 && tid == 0) sh.list_n = 0;
        cluster_sync();  // (the list and the result are written again)
        return found;
    };

    // cut: keys above cut_key and the first cut_n of the cut_all equal to it
    uint32_t cut_key = 0;
    u64 cut_n = 0, cut_all = 0;
    if (top_k < V && !descend(false, (u64)top_k, 0.0, 0, 0, false, cut_key, cut_n, cut_all)) cut_key = 0, cut_n = cut_all = 0;
    if (top_p < 1.f) {
        uint32_t key;
        u64 inside, in_all;
        if (top_p > 0.f) {
            if (descend(true, 0, (double)top_p, cut_key, cut_n, cut_n > 0 && top_k <= LIST, key, inside, in_all)) {
                cut_all = key == cut_key ? cut_all : in_all;  // (at the count's cut only its own copies were weighed)
                cut_key = key;
                cut_n = inside;
            }
        } else {  // one token: the largest logit, lowest index
            cut_key = kmax;
            cut_n = 1;
            cut_all = 2;  // ties are ranked below
        }
    }

    // what is left, in the order of the vocabulary: every warp a contiguous run of the slice
    const int run = (n + SAMPLE_WARPS - 1) / SAMPLE_WARPS, i0 = min(n, warp * run), i1 = min(n, i0 + run);
    u64 ties_before = 0;
    const bool rank_ties = cut_n < cut_all;
    if (rank_ties) {
        u64 ties = 0, all;
        for (int i = i0 + lane; i < i1; i += 32) ties += key_of(xs[i]) == cut_key;
        ties = (u64)__reduce_add_sync(0xffffffffu, (unsigned)ties);
        ties_before = __shfl_sync(0xffffffffu, block_exclusive(lane == 0 ? ties : 0, sh.warp_sum, all), 0);
        if (tid == 0) sh.ties = (int)all;
        cluster_sync();
        for (int c = 0; c < rank; c++) ties_before += (u64)cluster.map_shared_rank(&sh, c)->ties;
    }
    // (1 and more: nothing but the largest logit, whose weight a fixed-point one may equal by its rounding)
    const u64 floor_w = min_p >= 1.f ? (u64)FIXED_ONE + 1 : (min_p > 0.f ? (u64)ceil((double)min_p * FIXED_ONE) : 0);
    const float cut_x = cut_key > 0 ? of_key(cut_key) : -INFINITY;
    auto walk = [&](auto &&visit) {  // visit(i, kept weight) over this warp's run, 32 tokens at a time; false ends it
        u64 tie = ties_before;
        for (int i = i0; i < i1; i += 32) {
            const bool in = i + lane < i1;
            const float x = in ? xs[i + lane] : -INFINITY;
            const uint32_t k = key_of(x);
            bool keep = in && k >= cut_key;
            if (rank_ties) {
                const unsigned eq = __ballot_sync(0xffffffffu, in && k == cut_key);
                if (k == cut_key && tie + __popc(eq & ((1u << lane) - 1u)) >= cut_n) keep = false;
                tie += __popc(eq);
            }
            u64 w = 0;
            if (__any_sync(0xffffffffu, keep)) {
                if (keep) w = weight(x);
                if (w < floor_w && k != kmax) w = 0;
            }
            if (!visit(i + lane, w)) break;
        }
    };
    u64 mine = 0, here;
    if (rank_ties) {
        walk([&](int, u64 w) { mine += w; return true; });
    } else {
        // four tokens of a lane at a time: the weights' chain of 64-bit instructions is long
        auto sum = [&](auto &&x4, int m) {
            u64 w[4];
#pragma unroll
            for (int j = 0; j < m; j++) {
                const uint32_t k = key_of(x4[j]);
                w[j] = weight(x4[j]);
                mine += k < cut_key || (w[j] < floor_w && k != kmax) ? 0 : w[j];
            }
        };
        int i = i0 + lane;
        for (; i + 96 < i1; i += 128) {
            const float x4[4] = {xs[i], xs[i + 32], xs[i + 64], xs[i + 96]};
            if (x4[0] >= cut_x || x4[1] >= cut_x || x4[2] >= cut_x || x4[3] >= cut_x) sum(x4, 4);
        }
        for (; i < i1; i += 32) {
            const float x4[4] = {xs[i]};
            sum(x4, 1);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    u64 start = __shfl_sync(0xffffffffu, block_exclusive(lane == 0 ? mine : 0, sh.warp_sum, here), 0);
    if (tid == 0) sh.mass = here;
    cluster_sync();
    u64 total;
    {
        const u64 m = lane < CS ? cluster.map_shared_rank(&sh, lane)->mass : 0, incl = warp_inclusive(m);
        start += __shfl_sync(0xffffffffu, incl - m, rank);
        total = __shfl_sync(0xffffffffu, incl, 31);
    }
    cluster_sync();  // (no CTA leaves while another may read its shared memory)
    // first token whose cumulative weight exceeds the target
    // (at most the largest u below 1: above 2^53 a double does not tell total - 1 from total)
    const double target = (double)fminf(fmaxf(a.u[row], 0.f), 0x1.fffffep-1f) * (double)total;
    if (mine > 0 && (double)start <= target && target < (double)(start + mine)) {
        u64 cum = start;
        walk([&](int i, u64 w) {
            const u64 incl = warp_inclusive(w);
            const unsigned hit = __ballot_sync(0xffffffffu, (double)(cum + incl) > target);
            if (hit) {
                if (lane == __ffs(hit) - 1) a.ids[row] = i_first + i;
                return false;
            }
            cum += __shfl_sync(0xffffffffu, incl, 31);
            return true;
        });
    }
}

}  // namespace

cudaError_t launch_sample(const void *logits, int dt, int64_t M, int V, int64_t ld, const ttq_sampling &s, const float *u, int64_t *ids, int sms,
                          cudaStream_t st) {
    // CTAs per row: as many as it takes to fill the card with two CTAs per SM, at least so many that two fit there with their slices
    // (a row of 2^18 logits: 128 KB a CTA, one per SM)
    int cluster = 1;
    while (cluster < MAX_CLUSTER && ((int64_t)M * cluster * 2 <= 2 * (int64_t)sms || (V + cluster - 1) / cluster > 18432) && V / cluster > SAMPLE_THREADS) cluster *= 2;
    const int slice = (V + cluster - 1) / cluster;
    const size_t smem = sizeof(Shared) + (size_t)slice * sizeof(float);
    static OncePerDevice once;
    const cudaError_t e = once([&]() {
        return cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(Shared) + ((1 << 18) / MAX_CLUSTER) * sizeof(float)));
    });
    if (e != cudaSuccess) return e;
    static const bool pdl = env_flag("TTQ_PDL", true);
    const SampleArgs a{logits, dt, V, slice, ld, s, u, ids};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(M * cluster));
    cfg.blockDim = dim3(SAMPLE_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, sample_kernel, a);
}

}  // namespace ttq
