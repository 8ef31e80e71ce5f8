// Sampling: the next token of every row of logits from given random numbers, with temperature, top-k, top-p and min-p.
//
// All three cuts keep a head of the same order (logit descending, index ascending), so a row's result needs no sort: the logit t at
// which the head ends, and how many tokens with exactly this logit still belong to it.  t is found by descending through the
// 32 bits of an order-preserving key, 11, 11 and 10 bits at a time, with a histogram of counts and weights per step.
// Weights are w = exp((x - max) / T), computed in 64 bits and summed as 2^-44 fixed point: integer sums are exact, do not depend on the
// order of the atomics, and their rounding (2^-45 a token, where the largest weight is 1) is far below the weight of any token that
// decides a cut.  In 32 bits a cut among 10^5 tokens of similar weight falls on a neighbour of the right one about once in 400 rows.
#include "ttq_internal.cuh"

namespace ttq {
namespace {

constexpr int SAMPLE_THREADS = 1024;
constexpr int SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int BINS = 2048;
constexpr double FIXED_ONE = 17592186044416.0;  // 2^44

struct SampleArgs {
    const void *logits;
    int dt, V;
    int64_t ld;
    ttq_sampling s;
    const float *u;
    int64_t *ids;
};

// Order-preserving: larger float, larger key; -0 and +0 alike; NaN below everything (as -inf).
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Shared {
    uint32_t cnt[BINS], lo[BINS], hi[BINS];
    unsigned long long warp_sum[SAMPLE_WARPS];
    int warp_cnt[SAMPLE_WARPS];
    unsigned long long above_mass, found_mass;
    int above_cnt, found_bin, found_cnt;
    int result;
};

// Sum of v over lower-numbered threads; `all`: over every thread.
template <class T>
__device__ __forceinline__ T block_exclusive(T v, T *warp_sums, T &all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    T before = 0;
    all = 0;
    for (int w = 0; w < SAMPLE_WARPS; w++) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    return before + incl - v;
}

__global__ void __launch_bounds__(SAMPLE_THREADS) sample_kernel(const SampleArgs a) {
    __shared__ Shared sh;
    grid_launch_dependents();
    grid_dependency_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t row = blockIdx.x;
    const int V = a.V;
    const int64_t base = row * a.ld;
    const float temperature = a.s.temperature_dev ? a.s.temperature_dev[row] : a.s.temperature;
    const float top_p = a.s.top_p_dev ? a.s.top_p_dev[row] : a.s.top_p;
    const float min_p = a.s.min_p_dev ? a.s.min_p_dev[row] : a.s.min_p;
    int top_k = a.s.top_k_dev ? a.s.top_k_dev[row] : a.s.top_k;
    if (top_k <= 0 || top_k > V) top_k = V;

    // largest key and its lowest index
    unsigned long long best = 0;
    for (int i = tid; i < V; i += SAMPLE_THREADS) {
        const unsigned long long k = ((unsigned long long)key_of(load_as_float(a.logits, a.dt, base + i)) << 32) | (0xffffffffu - (uint32_t)i);
        best = k > best ? k : best;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long x = __shfl_xor_sync(0xffffffffu, best, o);
        best = x > best ? x : best;
    }
    if (lane == 0) sh.warp_sum[warp] = best;
    __syncthreads();
    for (int w = 0; w < SAMPLE_WARPS; w++) best = sh.warp_sum[w] > best ? sh.warp_sum[w] : best;
    const uint32_t kmax = (uint32_t)(best >> 32);
    const float xmax = of_key(kmax);
    const int argmax = (int)(0xffffffffu - (uint32_t)best);
    if (xmax == -INFINITY || !(temperature > 0.f)) {
        if (tid == 0) a.ids[row] = xmax == -INFINITY ? -1 : argmax;
        return;
    }
    const double dmax = xmax, dtemp = temperature;
    auto weight = [&](uint32_t k) -> double {
        return k == kmax ? 1.0 : exp(((double)of_key(k) - dmax) / dtemp);  // (an infinite maximum leaves weight to itself only)
    };
    auto fixed = [&](double w) { return (unsigned long long)__double2ull_rn(w * FIXED_ONE); };

    // One descent.  Elements: keys above `lim`, and `lim_n` of those equal to it.  Finds the key at which the running count
    // (by_mass false) or weight (true), from the top, reaches the target: key, copies of it inside, count and weight before it.
    auto descend = [&](bool by_mass, int target_cnt, double target_mass, uint32_t lim, int lim_n, uint32_t &key, int &copies,
                       unsigned long long &mass_before) {
        uint32_t prefix = 0;
        int cnt_before = 0;
        mass_before = 0;
        for (int level = 0; level < 3; level++) {
            const int shift = level == 0 ? 21 : (level == 1 ? 10 : 0), bits = level == 2 ? 10 : 11;
            __syncthreads();
            for (int i = tid; i < BINS; i += SAMPLE_THREADS) sh.cnt[i] = sh.lo[i] = sh.hi[i] = 0;
            __syncthreads();
            auto add = [&](uint32_t k, uint32_t n) {
                if (level > 0 && (k >> (shift + bits)) != prefix) return;
                const int bin = (k >> shift) & ((1 << bits) - 1);
                atomicAdd(&sh.cnt[bin], n);
                const unsigned long long f = fixed(weight(k)) * n;
                const uint32_t lo = (uint32_t)f, old = atomicAdd(&sh.lo[bin], lo);
                const uint32_t hi = (uint32_t)(f >> 32) + (old + lo < old ? 1u : 0u);
                if (hi) atomicAdd(&sh.hi[bin], hi);
            };
            for (int i = tid; i < V; i += SAMPLE_THREADS) {
                const uint32_t k = key_of(load_as_float(a.logits, a.dt, base + i));
                if (k > lim) add(k, 1);
            }
            if (tid == 0) add(lim, (uint32_t)lim_n);
            __syncthreads();
            // two bins per thread, the highest first
            const int b1 = BINS - 1 - 2 * tid, b0 = b1 - 1;
            const int n1 = (int)sh.cnt[b1], n0 = (int)sh.cnt[b0];
            const unsigned long long m1 = ((unsigned long long)sh.hi[b1] << 32) | sh.lo[b1], m0 = ((unsigned long long)sh.hi[b0] << 32) | sh.lo[b0];
            int all_n;
            unsigned long long all_m;
            int cn = cnt_before + block_exclusive(n1 + n0, sh.warp_cnt, all_n);
            unsigned long long cm = mass_before + block_exclusive(m1 + m0, sh.warp_sum, all_m);
            auto reached = [&](int n, unsigned long long m) { return by_mass ? (double)m >= target_mass : n >= target_cnt; };
            if (tid == 0) sh.found_bin = -1;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int n = j == 0 ? n1 : n0, bin = j == 0 ? b1 : b0;
                const unsigned long long m = j == 0 ? m1 : m0;
                if (n > 0 && reached(cn + n, cm + m) && !reached(cn, cm)) {
                    sh.found_bin = bin;
                    sh.above_cnt = cn;
                    sh.above_mass = cm;
                    sh.found_cnt = n;
                }
                cn += n;
                cm += m;
            }
            __syncthreads();
            const int bin = sh.found_bin;
            if (bin < 0) {  // (target within rounding of the whole: everything stays)
                key = lim;
                copies = lim_n;
                return;
            }
            cnt_before = sh.above_cnt;
            mass_before = sh.above_mass;
            prefix = (prefix << bits) | (uint32_t)bin;
        }
        key = prefix;
        const int have = sh.found_cnt;
        if (by_mass) {
            const double each = (double)fixed(weight(key));
            double r = each > 0.0 ? ceil((target_mass - (double)mass_before) / each) : 1.0;
            copies = r < 1.0 ? 1 : (r > have ? have : (int)r);
        } else {
            copies = target_cnt - cnt_before;
        }
    };

    // cut: keys above cut_key and the first cut_n of those equal to it
    uint32_t cut_key = 0;
    int cut_n = V;
    unsigned long long before;
    if (top_k < V) descend(false, top_k, 0.0, 0, 0, cut_key, cut_n, before);
    if (top_p < 1.f) {
        unsigned long long total;
        if (top_k < V) {
            total = before + fixed(weight(cut_key)) * (unsigned long long)cut_n;
        } else {
            unsigned long long mine = 0;
            for (int i = tid; i < V; i += SAMPLE_THREADS) mine += fixed(weight(key_of(load_as_float(a.logits, a.dt, base + i))));
            block_exclusive(mine, sh.warp_sum, total);
        }
        const double target = fmax((double)top_p, 0.0) * (double)total;
        const uint32_t lim = top_k < V ? cut_key : 0;
        const int lim_n = top_k < V ? cut_n : 0;
        if (target > 0.0) {
            descend(true, 0, target, lim, lim_n, cut_key, cut_n, before);
        } else {
            cut_key = kmax;
            cut_n = 1;
        }
    }

    // what is left, in the order of the vocabulary: every warp a contiguous run of it
    const int run = (V + SAMPLE_WARPS - 1) / SAMPLE_WARPS, i0 = warp * run, i1 = min(V, i0 + run);
    // first the tokens that tie with the cut
    int ties = 0;
    for (int i = i0 + lane; i < i1; i += 32) ties += key_of(load_as_float(a.logits, a.dt, base + i)) == cut_key;
    ties = __reduce_add_sync(0xffffffffu, ties);
    int all_ties;
    int ties_before = block_exclusive(lane == 0 ? ties : 0, sh.warp_cnt, all_ties);
    ties_before = __shfl_sync(0xffffffffu, ties_before, 0);
    // weight that token i keeps; `tie_rank`: ties before it
    auto kept = [&](uint32_t k, int tie_rank) -> unsigned long long {
        if (k < cut_key || (k == cut_key && tie_rank >= cut_n)) return 0;
        const double w = weight(k);
        return w >= (double)min_p || k == kmax ? fixed(w) : 0;
    };
    auto walk = [&](auto &&visit) {  // visit(i, kept weight, whole chunk) over this warp's run; false ends it
        int tie = ties_before;
        for (int i = i0; i < i1; i += 32) {
            const bool in = i + lane < i1;
            const uint32_t k = in ? key_of(load_as_float(a.logits, a.dt, base + i + lane)) : 0;
            const unsigned eq = __ballot_sync(0xffffffffu, in && k == cut_key);
            const unsigned long long w = in ? kept(k, tie + __popc(eq & ((1u << lane) - 1u))) : 0;
            tie += __popc(eq);
            if (!visit(i + lane, w)) break;
        }
    };
    unsigned long long mine = 0, total;
    walk([&](int, unsigned long long w) { mine += w; return true; });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    unsigned long long start = block_exclusive(lane == 0 ? mine : 0ull, sh.warp_sum, total);
    start = __shfl_sync(0xffffffffu, start, 0);
    // first token whose cumulative weight exceeds the target; the last one with weight if rounding leaves none
    double target = (double)fminf(fmaxf(a.u[row], 0.f), 1.f) * (double)total;
    if (target >= (double)total) target = (double)(total - 1);
    if (mine > 0 && (double)start <= target && target < (double)(start + mine)) {
        unsigned long long cum = start;
        walk([&](int i, unsigned long long w) {
            unsigned long long incl = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, (double)(cum + incl) > target);
            if (hit) {
                if (lane == __ffs(hit) - 1) a.ids[row] = i;
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
    (void)sms;
    const SampleArgs a{logits, dt, V, ld, s, u, ids};
    return launch_pdl(sample_kernel, dim3((unsigned)M), dim3(SAMPLE_THREADS), 0, st, a);
}

}  // namespace ttq
