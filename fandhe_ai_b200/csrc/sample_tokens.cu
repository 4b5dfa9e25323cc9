// Drawing the next token of every row of logits on the device.
//
// For a row x[0..V) with temperature T the weight of token i is w_i = e^((x_i - max x) / T); a logit of -inf has weight
// zero and is never kept.  Tokens are taken in the order "larger logit first, equal logits: lower index first":
//   S1 = the first top_k of them (all for top_k <= 0),
//   S2 = the shortest prefix of S1 whose weight reaches top_p * W(S1) (all of S1 for top_p >= 1),
//   S3 = the tokens of S2 with w_i >= min_p (the first token always),
// and the drawn token is the smallest index i of S3 at which the running sum over S3 in index order exceeds u * W(S3).
//
// Arithmetic.  A token stands next to a border of these sums in every row (neighbours in a flat row of 128k tokens are 1e-5 of
// the sum apart), so weights are computed in f64 and held as integers, w * 2^shift rounded (vocab * 2^shift <= 2^62, so
// no sum of a row overflows): integer sums do not depend on their order, whatever the cluster size or the scheduling.
// A weight below 2^-(shift + 1) is zero in the sums; min_p is compared with the f64 weight.
//
// One cluster of C thread blocks owns a row and keeps it in its shared memory, so that the logits are read from HBM once
// however many passes the filters take.  Selection needs no sort: tokens fall into 2048 bins of (max - x) / T (a monotone
// function, 1/32 of a doubling of the weight per bin), the bin a border falls into is found from the counts, and only the
// few tokens of that bin are ranked exactly.  Tokens that the counts already rule out are left behind: the others ("survivors",
// usually a few hundred) move to a list in index order, and what follows works on that.  A bin that holds more than kCandidates tokens (flat or heavily tied rows) is
// resolved by bisection over the ordered pair (logit, index) instead.
//
// Measured on a B200: one row of 128256 f32 logits 25 us, 128 such rows with every filter 107 us, 512 rows of 32000 bf16 logits 60 us,
// of 32768 62 us.  Bound by latency, not by HBM (whose share is 10 us of the 107): a row takes about 37 thousand clocks, of which 5 load it, 9 go
// into the bins and the f64 sum, 9 into cluster barriers and 4 each into leaving tokens behind and ranking the border's bin.
#include <cfloat>
#include <type_traits>

#include "kernels.cuh"
#include "launch.cuh"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kCandidates = 512;
constexpr int kSurvivors = 3584;
constexpr int kMaxCluster = 8;
constexpr int kMaxPerCta = 45056;      // f32 logits of a thread block: 176 KB, which leaves room for what else it keeps

// 2^(j / 64)
__constant__ double kRoots[64] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951};

struct Shared {
    double roots[64];                         // the table again, where threads may look up different entries
    uint64_t exchange[2][kMaxCluster][4];     // [phase][source rank][value], written by the peers
    uint64_t warp_sum[kWarps][4];
    uint32_t hist[kBins];
    uint32_t total[kBins];                    // the bins of the whole row
    uint64_t all_pair[kCandidates];           // the candidates of the whole row, written by the peers
    uint64_t all_w[kCandidates];
    uint32_t counts[kMaxCluster];
    uint32_t scan_count[kWarps];
    float scan_mass[kWarps];
    float list_x[kSurvivors];
    uint16_t list_i[kSurvivors];              // place in this block's share
    uint32_t n_cand;
    uint32_t found[6];
    unsigned long long best;
};

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, uint64_t v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int m) {
    return static_cast<uint64_t>(__shfl_xor_sync(0xffffffffu, static_cast<unsigned long long>(v), m));
}

// f32 -> u32 with the same order (-inf smallest); -0 is made +0 first so that equal logits have equal keys
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// larger = earlier in the order (larger logit, then lower index)
__device__ __forceinline__ uint64_t order_pair(float x, uint32_t i) {
    return (static_cast<uint64_t>(order_key(x)) << 32) | (0xFFFFFFFFu - i);
}

template <typename T>
__device__ __forceinline__ float logit_f32(T v);
template <>
__device__ __forceinline__ float logit_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float logit_f32<uint16_t>(uint16_t v) { return bf16_bits_to_f32(v); }

static_assert(sizeof(Shared) + 16 + kMaxPerCta * 4 <= 232448, "a thread block's shared memory");
static_assert((kMaxPerCta + kThreads - 1) / kThreads < 128, "a thread's run, in two words of bits");

struct Row {
    float max_x, bin_scale;
    double max_d, arg_scale;      // 64 log2(e) / T
    const double* roots;
    int shift, dead_bin;          // from this bin on a weight rounds to zero

    __device__ __forceinline__ int bin(float x) const {       // kBins for -inf
        const float d = max_x - x;
        const int b = d == 0.0f ? 0 : static_cast<int>(fminf(d * bin_scale, static_cast<float>(kBins - 1)));
        return x == -INFINITY ? kBins : b;
    }
    // 2^(y / 64), y = n + r, |r| <= 1/2: the table's 2^((n mod 64) / 64), the Taylor polynomial of 2^(r / 64) (its remainder is below
    // 2^-54), and n / 64 in the exponent.  About 2^-50 relative, as the f64 subtraction and quotient it starts from.
    __device__ __forceinline__ double scaled_weight(float x, int up) const {
        const double magic = 6755399441055744.0;      // 1.5 * 2^52: adding it rounds to an integer and leaves that in the low word
        const double y = (static_cast<double>(x) - max_d) * arg_scale;
        const double z = y + magic;
        const int n = __double2loint(z);
        const double r = y - (z - magic);
        double q = fma(r, 1.2417843701716925e-12, 5.732851688640402e-10);
        q = fma(q, r, 2.1173137155464776e-07);
        q = fma(q, r, 5.86490495505617e-05);
        q = fma(q, r, 0.010830424696249145);
        q = fma(q, r, 1.0);
        q *= roots[n & 63];
        return __hiloint2double(__double2hiint(q) + ((n >> 6) + up) * (1 << 20), __double2loint(q));
    }
    // the weight as an integer, 2^shift for the maximum
    __device__ __forceinline__ uint64_t weight(float x, int b) const {
        const double w = scaled_weight(b >= dead_bin ? max_x : x, shift) + 4503599627370496.0;      // 2^52: rounds, and the mantissa is the integer
        return b >= dead_bin ? 0 : static_cast<uint64_t>(__double_as_longlong(w)) & 0xFFFFFFFFFFFFFull;
    }
    // min_p asks for the weight itself: rounded, it would be zero or a small whole number there.  Beyond 2^-150 no f32 reaches.
    __device__ __forceinline__ bool reaches(float x, double least) const {
        return (max_x - x) * bin_scale < 4800.0f && scaled_weight(x, 0) >= least;
    }
};

// Sums (or with kMax: maxima) of N values over the cluster; `mine` receives nothing, `out` the totals, and
// sh.exchange[phase][rank] keeps the per-block values until the phase after next.
template <int N, bool kMax>
__device__ __forceinline__ void cluster_reduce(Shared& sh, int& phase, uint32_t rank, uint32_t nranks, const uint64_t (&v)[N],
                                               uint64_t (&out)[N]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t x[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        x[k] = v[k];
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) {
            const uint64_t o = shfl_xor_u64(x[k], m);
            x[k] = kMax ? (o > x[k] ? o : x[k]) : x[k] + o;
        }
        if (lane == 0) sh.warp_sum[warp][k] = x[k];
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            x[k] = lane < kWarps ? sh.warp_sum[lane][k] : 0;
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) {
                const uint64_t o = shfl_xor_u64(x[k], m);
                x[k] = kMax ? (o > x[k] ? o : x[k]) : x[k] + o;
            }
            if (static_cast<uint32_t>(lane) < nranks) st_cluster_u64(mapa_shared(smem_u32(&sh.exchange[phase][rank][k]), lane), x[k]);
        }
    }
    cluster_sync_all();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        out[k] = 0;
        for (uint32_t r = 0; r < nranks; ++r) {
            const uint64_t o = sh.exchange[phase][r][k];
            out[k] = kMax ? (o > out[k] ? o : out[k]) : out[k] + o;
        }
    }
    phase ^= 1;
}

struct Cut {                 // kept: bin < bin, or bin == bin and not after (x, i)
    int bin;
    uint64_t pair;
    __device__ __forceinline__ bool keeps(int b, float x, uint32_t i) const { return b < bin || (b == bin && order_pair(x, i) >= pair); }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_tokens_kernel(SampleShape p, const T* __restrict__ logits,
                                                                 const float* __restrict__ temperature, const int* __restrict__ top_k,
                                                                 const float* __restrict__ top_p, const float* __restrict__ min_p,
                                                                 const float* __restrict__ uniform, int* __restrict__ ids,
                                                                 float* __restrict__ prob, int* __restrict__ kept) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Shared& sh = *reinterpret_cast<Shared*>(smem_raw);
    T* xs = reinterpret_cast<T*>(smem_raw + (sizeof(Shared) + 15) / 16 * 16);      // in their own type
    const uint32_t nranks = p.cluster, rank = nranks > 1 ? cluster_ctarank() : 0;
    const int64_t row = blockIdx.x / nranks;
    if (p.active && p.active[row] == 0) return;      // the whole cluster, before its first barrier
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t first = int64_t(rank) * p.per_cta;
    const int64_t left = int64_t(p.vocab) - first;
    const int n = left <= 0 ? 0 : (left < p.per_cta ? int(left) : p.per_cta);
    const T* src = logits + row * p.row_stride + first;
    int phase = 0;

    // ---- the row into shared memory; its first maximum; is there a NaN or +inf?
    uint64_t best = 0, bad = 0;
    auto take = [&](int i, float x) {
        if (!(x < INFINITY)) bad = 1;
        const uint64_t pr = order_pair(x, uint32_t(first) + i);
        if (x != -INFINITY && pr > best) best = pr;
    };
    if (nranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    constexpr int kVec = 16 / sizeof(T);
    int done = 0;
    if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
        done = n / kVec * kVec;
#pragma unroll 4
        for (int g = tid; g < n / kVec; g += kThreads) {
            const uint4 raw = __ldcs(reinterpret_cast<const uint4*>(src) + g);
            const T* v = reinterpret_cast<const T*>(&raw);
            reinterpret_cast<uint4*>(xs)[g] = raw;
#pragma unroll
            for (int k = 0; k < kVec; ++k) take(g * kVec + k, logit_f32<T>(v[k]));
        }
    }
    for (int i = done + tid; i < n; i += kThreads) {
        xs[i] = src[i];
        take(i, logit_f32<T>(src[i]));
    }
    for (int b = tid; b < kBins; b += kThreads) sh.hist[b] = 0;
    if (tid < 64) sh.roots[tid] = kRoots[tid];
    if (tid == 0) sh.n_cand = 0;
    if (nranks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // the peers are running: their shared memory may be written
    const uint64_t best_bad[2] = {best, bad};
    uint64_t top[2];
    cluster_reduce<2, true>(sh, phase, rank, nranks, best_bad, top);

    const float t = temperature ? temperature[row] : 1.0f;
    const int k = top_k ? top_k[row] : 0;
    const float tp = top_p ? top_p[row] : 1.0f;
    const float mp = min_p ? min_p[row] : 0.0f;
    const float u = uniform[row];
    const bool valid = top[0] != 0 && top[1] == 0 && t >= 0.0f && t < INFINITY && tp == tp && mp == mp && u >= 0.0f && u < 1.0f;
    const uint32_t best_i = 0xFFFFFFFFu - static_cast<uint32_t>(top[0]);
    if (!valid || t == 0.0f || k == 1 || tp <= 0.0f) {      // nothing to draw from, or the first maximum is all that is kept
        if (rank == 0 && tid == 0) {
            ids[row] = valid ? int(best_i) : -1;
            if (prob) prob[row] = valid ? 1.0f : 0.0f;
            if (kept) kept[row] = valid ? 1 : 0;
        }
        return;
    }
    Row r;
    {
        const uint32_t key = static_cast<uint32_t>(top[0] >> 32);
        r.max_x = __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
        r.bin_scale = fminf(46.166241308f / t, FLT_MAX);      // 32 log2(e) / T
        r.max_d = static_cast<double>(r.max_x);
        r.arg_scale = 92.33248261893424 / static_cast<double>(t);      // 64 log2(e) / T
        r.roots = sh.roots;
        r.shift = p.shift;
        r.dead_bin = min(kBins - 1, 32 * (p.shift + 2));
    }
    const double unit = static_cast<double>(1ull << p.shift);
    const int run = p.run;
    int lo = tid * run, hi = min(n, lo + run);      // this thread's elements: of the block's share, or of the list
    bool listed = false;
    auto X = [&](int i) { return listed ? sh.list_x[i] : logit_f32<T>(xs[i]); };
    auto index = [&](int i) { return uint32_t(first) + (listed ? uint32_t(sh.list_i[i]) : uint32_t(i)); };

    // Every block hands the tokens of bin `b` to all blocks, as ordered pairs (0: not among `under`); returns how many places that
    // takes, which is known not to exceed kCandidates.
    auto gather = [&](int b, const Cut& under) -> int {
        if (uint32_t(tid) < nranks) sh.counts[tid] = nranks > 1 ? ld_cluster_u32(mapa_shared(smem_u32(&sh.hist[b]), tid)) : sh.hist[b];
        if (tid == 0) { sh.n_cand = 0; sh.best = ~0ull; }
        __syncthreads();
        int total = 0, at = 0;
        for (uint32_t q = 0; q < nranks; ++q) {
            if (q < rank) at += int(sh.counts[q]);
            total += int(sh.counts[q]);
        }
        for (int i = lo; i < hi; ++i) {
            const float x = X(i);
            if (r.bin(x) != b) continue;
            const uint64_t pair = under.keeps(b, x, index(i)) ? order_pair(x, index(i)) : 0;
            const int to = at + int(atomicAdd(&sh.n_cand, 1u));
            for (uint32_t q = 0; q < nranks; ++q) st_cluster_u64(mapa_shared(smem_u32(&sh.all_pair[to]), q), pair);
        }
        cluster_sync_all();
        return total;
    };
    auto logit_of = [&](uint64_t pair) {
        const uint32_t key = static_cast<uint32_t>(pair >> 32);
        return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
    };
    // The last pair of bin `b` (under `under`) that belongs to the prefix in which `enough` is not reached before it, by
    // bisection over the 64-bit order: `measure` gives a token's contribution, `base` what lies above the bin.
    auto bisect = [&](int b, const Cut& under, bool by_weight, uint64_t base, double enough) -> uint64_t {
        uint64_t a = 0, z = ~0ull;           // the largest pair P with measure(pairs >= P) >= enough
        while (a < z) {
            const uint64_t mid = a + ((z - a) >> 1) + 1;
            uint64_t s[1] = {0}, sum[1];
            for (int i = lo; i < hi; ++i) {
                const float x = X(i);
                if (r.bin(x) == b && order_pair(x, index(i)) >= mid && under.keeps(b, x, index(i))) s[0] += by_weight ? r.weight(x, b) : 1ull;
            }
            cluster_reduce<1, false>(sh, phase, rank, nranks, s, sum);
            if (static_cast<double>(base + sum[0]) >= enough) a = mid;
            else z = mid - 1;
        }
        return a;
    };

    // ---- the bins of the row; top-p over the whole row also wants the row's sum
    const bool limited = k > 0 && k < p.vocab;
    uint64_t row_sum = 0;
    auto bins = [&](auto weighed) {
        for (int i0 = lo; i0 < lo + run; i0 += 4) {      // four at a time, without branches around the arithmetic
            float x[4];
            int b[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                x[q] = i0 + q < hi ? logit_f32<T>(xs[i0 + q]) : -INFINITY;
                b[q] = r.bin(x[q]);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (b[q] < kBins) atomicAdd(&sh.hist[b[q]], 1u);
            if (decltype(weighed)::value) {
                uint64_t w[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) w[q] = r.weight(x[q], b[q]);
                row_sum += (w[0] + w[1]) + (w[2] + w[3]);
            }
        }
    };
    if (tp < 1.0f && !limited) bins(std::true_type());
    else bins(std::false_type());
    if (nranks > 1) {
        cluster_sync_all();
        const int slice = kBins / int(nranks);
        for (int b = int(rank) * slice + tid; b < int(rank + 1) * slice; b += kThreads) {
            uint32_t s = 0;
            for (uint32_t q = 0; q < nranks; ++q) s += ld_cluster_u32(mapa_shared(smem_u32(&sh.hist[b]), q));
            for (uint32_t q = 0; q < nranks; ++q) st_cluster_u32(mapa_shared(smem_u32(&sh.total[b]), q), s);
        }
        cluster_sync_all();
    } else {
        __syncthreads();
        for (int b = tid; b < kBins; b += kThreads) sh.total[b] = sh.hist[b];
        __syncthreads();
    }
    // prefix over the bins: each thread owns four of them
    constexpr int kPer = kBins / kThreads;
    uint32_t c4[kPer], count_before;
    float m4[kPer], mass_before;
    uint32_t all_count = 0;
    float all_mass = 0.0f;
    {
        uint32_t c = 0;
        float m = 0.0f;
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
            const int b = tid * kPer + q;
            c4[q] = sh.total[b];
            m4[q] = float(c4[q]) * exp2f(-(float(b) + 0.5f) * (1.0f / 32.0f));     // an estimate: only decides where to look
            c += c4[q];
            m += m4[q];
        }
        uint32_t cs = c;
        float ms = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t cu = __shfl_up_sync(0xffffffffu, cs, o);
            const float mu = __shfl_up_sync(0xffffffffu, ms, o);
            if (lane >= o) { cs += cu; ms += mu; }
        }
        if (lane == 31) { sh.scan_count[warp] = cs; sh.scan_mass[warp] = ms; }
        __syncthreads();
        uint32_t cb = 0;
        float mb = 0.0f;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) { cb += sh.scan_count[w]; mb += sh.scan_mass[w]; }
            all_count += sh.scan_count[w];
            all_mass += sh.scan_mass[w];
        }
        count_before = cb + cs - c;
        mass_before = mb + ms - m;
    }
    Cut cut{kBins, 0};

    // ---- where the borders lie by the counts: the bin of the k-th token, and the bin in which the estimated mass reaches top_p
    const bool cut_k = limited && uint32_t(k) < all_count;
    float k_mass = all_mass;
    if (tid == 0) sh.found[3] = uint32_t(kBins - 1);
    if (cut_k) {
        uint32_t cb = count_before;
        float mb = mass_before;
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
            if (cb < uint32_t(k) && uint32_t(k) <= cb + c4[q]) {
                sh.found[0] = tid * kPer + q;
                sh.found[1] = uint32_t(k) - cb;
                sh.found[2] = __float_as_uint(mb + m4[q] * (float(uint32_t(k) - cb) / float(c4[q])));
            }
            cb += c4[q];
            mb += m4[q];
        }
    }
    __syncthreads();
    const int bk = cut_k ? int(sh.found[0]) : kBins - 1;
    if (cut_k) k_mass = __uint_as_float(sh.found[2]);
    int bp = bk;
    if (tp < 1.0f) {
        const float est = tp * k_mass;
        float mb = mass_before;
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
            if (mb < est && est <= mb + m4[q]) atomicMin(&sh.found[3], uint32_t(tid * kPer + q));
            mb += m4[q];
        }
        __syncthreads();
        bp = min(int(sh.found[3]), bk);
    }
    // ---- the survivors: S1 lies in the bins up to bk; without top-k, S2 up to bp (give or take: should its border turn out to lie
    // further, the whole share is gone through again), and S3 up to where a weight falls below min_p
    int last_bin = kBins - 1;
    if (cut_k) last_bin = bk;
    else if (tp < 1.0f) last_bin = limited ? kBins - 1 : min(bp + 2, kBins - 1);      // (fewer tokens than top_k: their sum is still to come)
    else if (mp > 0.0f) last_bin = min(static_cast<int>(-32.0f * log2f(fminf(mp, 1.0f))) + 2, kBins - 1);
    if (last_bin < kBins - 1) {
        // a logit below this is in a later bin for certain (the bins themselves are asked for again below)
        const float least = r.max_x - (float(last_bin + 1) / r.bin_scale * 1.00001f + fabsf(r.max_x) * 1e-6f);
        uint64_t mine = 0, more = 0;      // of this thread's first 64 elements, and of the others
        for (int i0 = lo; i0 < lo + run; i0 += 8) {
            uint32_t some = 0;
#pragma unroll
            for (int q = 0; q < 8; ++q) some |= (i0 + q < hi && logit_f32<T>(xs[i0 + q]) >= least ? 1u : 0u) << q;
            (i0 - lo < 64 ? mine : more) |= uint64_t(some) << ((i0 - lo) & 63);
        }
        const int count = __popcll(mine) + __popcll(more);
        int upto = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += up;
        }
        if (lane == 31) sh.warp_sum[warp][0] = uint64_t(upto);
        __syncthreads();
        int total = 0, at = upto - count;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) at += int(sh.warp_sum[w][0]);
            total += int(sh.warp_sum[w][0]);
        }
        __syncthreads();
        if (total <= kSurvivors) {
            auto put = [&](uint64_t bits, int from) {
                while (bits) {
                    const int j = from + __ffsll(static_cast<long long>(bits)) - 1;
                    bits &= bits - 1;
                    sh.list_x[at] = logit_f32<T>(xs[j]);
                    sh.list_i[at++] = uint16_t(j);
                }
            };
            put(mine, lo);
            put(more, lo + 64);
            __syncthreads();
            listed = true;
            const int per = (total + kThreads - 1) / kThreads;
            lo = min(total, tid * per);
            hi = min(total, lo + per);
        }
    }
    auto unlist = [&]() {
        listed = false;
        lo = tid * run;
        hi = min(n, lo + run);
    };

    // ---- top-k: the k-th token's rank inside its bin
    if (cut_k) {
        const uint32_t want = sh.found[1];
        cut.bin = bk;
        if (sh.total[bk] <= kCandidates) {
            const int m = gather(bk, Cut{kBins, 0});
            for (int i = tid; i < m; i += kThreads) {
                const uint64_t mine = sh.all_pair[i];
                uint32_t ahead = 0;
#pragma unroll 4
                for (int j = 0; j < m; ++j) ahead += sh.all_pair[j] > mine;
                if (ahead == want - 1) sh.best = mine;
            }
            __syncthreads();
            cut.pair = sh.best;
        } else {
            cut.pair = bisect(bk, Cut{kBins, 0}, false, 0, double(want));
        }
    }

    // ---- top-p: exact sums around the estimated bin until the border lies inside it, then the border inside the bin
    if (tp < 1.0f) {
        int blo = 0, bhi = bk;
        const Cut k_cut = cut;
        // sums of the tokens of S1 in the bins [from, to), and in bin `to`
        auto sums = [&](int from, int to, uint64_t (&sum)[3]) {
            uint64_t s[3] = {0, 0, limited ? 0 : row_sum};
#pragma unroll 3
            for (int i = lo; i < hi; ++i) {
                const float x = X(i);
                const int b = r.bin(x);
                if (b < from || (limited ? b > k_cut.bin : b > to) || b == kBins) continue;
                if (limited && b == k_cut.bin && !k_cut.keeps(b, x, index(i))) continue;
                const uint64_t w = r.weight(x, b);
                if (limited) s[2] += w;
                if (b < to) s[0] += w;
                else if (b == to) s[1] += w;
            }
            cluster_reduce<3, false>(sh, phase, rank, nranks, s, sum);
        };
        uint64_t sum[3];
        sums(0, bp, sum);
        const double target = double(tp) * double(sum[2]);
        uint64_t above = sum[0], inside = sum[1];
        for (;;) {
            int next;
            if (double(above) >= target && bp > blo) {               // the border lies above this bin: towards it by the estimates
                bhi = bp - 1;
                float gap = float((double(above) - target) / unit);
                for (next = bhi; next > blo; --next) {
                    const float est_b = float(sh.total[next]) * exp2f(-(float(next) + 0.5f) * (1.0f / 32.0f));
                    if (gap < est_b) break;
                    gap -= est_b;
                }
                uint64_t more[3];
                sums(next, bp, more);                                 // what lies between comes off
                above -= more[0];
            } else if (double(above + inside) < target && bp < bhi) {  // ... below it
                blo = bp + 1;
                float gap = float((target - double(above + inside)) / unit);
                for (next = blo; next < bhi; ++next) {
                    const float est_b = float(sh.total[next]) * exp2f(-(float(next) + 0.5f) * (1.0f / 32.0f));
                    if (gap <= est_b) break;
                    gap -= est_b;
                }
                above += inside;
                if (listed && next > last_bin) unlist();
                uint64_t more[3];
                sums(bp + 1, next, more);
                above += more[0];
                inside = more[1];
                bp = next;
                continue;
            } else {
                break;
            }
            uint64_t more[3];
            sums(next, next, more);
            inside = more[1];
            bp = next;
        }
        cut.bin = bp;
        if (sh.total[bp] <= kCandidates) {
            const int m = gather(bp, k_cut);
            for (int i = tid; i < m; i += kThreads) sh.all_w[i] = sh.all_pair[i] ? r.weight(logit_of(sh.all_pair[i]), bp) : 0;
            __syncthreads();
            for (int i = tid; i < m; i += kThreads) {
                const uint64_t mine = sh.all_pair[i];
                uint64_t ahead = above;
#pragma unroll 4
                for (int j = 0; j < m; ++j) ahead += sh.all_pair[j] > mine ? sh.all_w[j] : 0;
                if (mine && double(ahead) < target) atomicMin(&sh.best, static_cast<unsigned long long>(mine));   // the last kept one
            }
            __syncthreads();
            cut.pair = sh.best;
        } else {
            cut.pair = bisect(bp, k_cut, true, above, target);
        }
    }

    // ---- the draw: sums of the kept weights in index order
    uint64_t s[2] = {0, 0}, sum[2];
    auto kept_weight = [&](int i, uint64_t* w) -> bool {
        const float x = X(i);
        const int b = r.bin(x);
        if (b > cut.bin || b == kBins || (b == cut.bin && !cut.keeps(b, x, index(i)))) return false;
        *w = r.weight(x, b);
        return !(mp > 0.0f) || index(i) == best_i || r.reaches(x, double(mp));
    };
    for (int i = lo; i < hi; ++i) {
        uint64_t w;
        if (kept_weight(i, &w)) { s[0] += w; s[1] += 1; }
    }
    const int ph = phase;
    cluster_reduce<2, false>(sh, phase, rank, nranks, s, sum);
    // u = 0 draws the first kept token however small its weight is, so the running sum there is that of the counts
    const int by = u == 0.0f ? 1 : 0;
    const double goal = double(u) * double(sum[0]);
    uint64_t before = 0;
    for (uint32_t q = 0; q < rank; ++q) before += sh.exchange[ph][q][by];
    const uint64_t own_sum = sh.exchange[ph][rank][by];
    if (double(before) <= goal && double(before + own_sum) > goal) {      // one block, and in it one thread, holds the token
        uint64_t c = s[by];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t up = static_cast<uint64_t>(__shfl_up_sync(0xffffffffu, static_cast<unsigned long long>(c), o));
            if (lane >= o) c += up;
        }
        if (lane == 31) sh.warp_sum[warp][3] = c;
        __syncthreads();
        for (int w = 0; w < warp; ++w) before += sh.warp_sum[w][3];
        before += c - s[by];
        if (double(before) <= goal && double(before + s[by]) > goal) {
            uint64_t w = 0;
            for (int i = lo; i < hi; ++i) {
                if (!kept_weight(i, &w)) continue;
                before += by ? 1 : w;
                if (double(before) > goal) {
                    ids[row] = int(index(i));
                    const bool dead = (r.max_x - X(i)) * r.bin_scale > 32000.0f;      // 2^-1000 of the maximum
                    if (prob) prob[row] = dead ? 0.0f : float(r.scaled_weight(X(i), 0) * unit / double(sum[0]));
                    if (kept) kept[row] = int(sum[1]);
                    break;
                }
            }
        }
    }
}

}  // namespace

cudaError_t sample_tokens(const SampleShape& want, const void* logits, int bf16, const float* temperature, const int* top_k,
                          const float* top_p, const float* min_p, const float* uniform, int* ids, float* prob, int* kept, int sm_count,
                          cudaStream_t s) {
    SampleShape p = want;
    if (p.rows == 0) return cudaSuccess;
    // Blocks per row: enough that 64 KB of logits are one block's share (so that two blocks share an SM; 512 rows of 32000 bf16 logits
    // take 89 us with two blocks to a row), and for few rows as many as there are idle SMs as long as each keeps 4096 logits.
    int c = 1;
    while (c < kMaxCluster && (p.vocab > int64_t(c) * (bf16 ? 32768 : 16384) || (p.rows * c * 2 <= sm_count && p.vocab >= c * 2 * 4096))) c *= 2;
    p.cluster = c;
    p.per_cta = (((p.vocab + c - 1) / c) + 7) / 8 * 8;
    if (p.per_cta > kMaxPerCta) return cudaErrorInvalidValue;
    p.run = ((p.per_cta + kThreads - 1) / kThreads) | 1;      // odd: the threads' runs start in different banks
    int bits = 12;                                              // weights below 2^52, see Row::weight
    while ((int64_t(1) << bits) < p.vocab) ++bits;
    p.shift = 62 - bits;
    const int smem = int((sizeof(Shared) + 15) / 16 * 16) + p.per_cta * (bf16 ? 2 : 4);
    static int configured[2][64] = {};
    const dim3 grid(static_cast<unsigned>(p.rows * c));
    if (bf16) {
        if (cudaError_t e = ensure_dynamic_smem(sample_tokens_kernel<uint16_t>, smem, configured[0])) return e;
        return launch_ex(sample_tokens_kernel<uint16_t>, grid, dim3(kThreads), smem, s, c, false, p, static_cast<const uint16_t*>(logits),
                         temperature, top_k, top_p, min_p, uniform, ids, prob, kept);
    }
    if (cudaError_t e = ensure_dynamic_smem(sample_tokens_kernel<float>, smem, configured[1])) return e;
    return launch_ex(sample_tokens_kernel<float>, grid, dim3(kThreads), smem, s, c, false, p, static_cast<const float*>(logits),
                     temperature, top_k, top_p, min_p, uniform, ids, prob, kept);
}

int64_t sample_tokens_max_vocab() { return int64_t(kMaxPerCta) * kMaxCluster; }

}  // namespace b200
