// Sampling of one token per row of logits: temperature, top-k, top-p and min-p from a given uniform number.
//
//   w_i = exp((l_i - max l) / T); order by (l descending, i ascending); keep the first k; of those the shortest prefix
//   whose weight reaches p * (their sum); drop w_i < min_p; draw the lowest index i with
//   sum of kept w_j, j <= i  >  u * (sum of kept w).
//
// All three filters keep a prefix of the same order, so nothing is sorted: only the token at which a prefix ends (its
// border) is looked for.  A row is spread over a thread-block cluster; every CTA keeps its slice of keys in shared
// memory, so one pass over the logits is all the memory traffic.  A histogram of counts over 2048 bins that are linear in
// the logit (bins of leading key bits would put a whole binade on one shared-memory address) gives the bin that holds
// the k-th token, and, each bin taken at the weight of its middle, the one in which the weight reaches p.  One more pass
// adds up the exact weights above that bin and lists its tokens, which the CTAs exchange and compare pairwise; the exact
// sums tell whether the guess was right.  Where everything down to the k-th token is a short list, the rest of the work is
// done on the list alone.  What this does not settle (a bin of more than 512 tokens: coarse 16-bit logits, large
// vocabularies, long tails; a wrong guess) goes to a radix descent over the ordered bit pattern with exact sums, ties at
// its end counted in index order.
//
// Weights are integers, 2^frac * 2^((l - max) log2(e) / T) rounded, plus 1, frac = min(51, 62 - ceil(log2 V)); 0 below
// e^-707: integer sums do not depend on their order, so a draw is the same for every cluster size, and the border of a
// top-p set moves by no more than V * 2^-frac of the row's largest weight (2^-30 at V = 49152).  The power of two is a
// table of 2^(i/512) times the exponential series to degree 3 in 64-bit floats (error 9e-15), nine 64-bit operations in a
// chain of seven.  (The library's exp2 took 2.8 times as long; 32 entries in 16 copies, free of bank conflicts, and degree
// 5, eleven operations, a tenth longer.)
//
// Bound by latency where rows are few: six cluster barriers, reads of the peers' shared memory, code run once; 49152 bf16
// logits take 4.6 us greedy, 8.5 us with a temperature, 13.9 us with top-k 50, 18.7 us with top-p 0.9 over a flat
// distribution.  Where rows are many, a CTA's phases one after another (bins cleared, table, load, two cluster barriers, in
// four waves of CTAs for 512 rows, with no load of a next row under them): 512 rows 37 us greedy (1.3 TB/s), 53 us with a
// temperature and min-p, which leaves few weights to work out; and the chain of the weights: 81 us with a temperature.
// (Times on the device, without a call's host work.)
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/prime_kernels_b200.h"
#include "pk_common.cuh"

namespace pk {
namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleMaxVocab = 1 << 18;

struct SampleParams {
    const void* logits;
    long long row_stride;      // elements
    int vocab, slice, frac;    // slice: keys per CTA
    const float *uniform, *temperature, *top_p, *min_p;
    const int* top_k;
    float temperature_v, top_p_v, min_p_v;
    int top_k_v;
    long long* ids;
    float* logprobs;
};

// ---- ordered keys (key_below, key_above: of the nearest value of the type at or below, above): key(a) < key(b) iff a < b; -0 and +0 share one key; NaN and -inf are key 0 ("never drawn")
template <int DT> struct KeyOf;
template <> struct KeyOf<0> {      // bf16
    using Key = uint16_t;
    using Raw = uint16_t;
    static __device__ __forceinline__ uint32_t key(uint32_t r) {
        if ((r & 0x7fffu) > 0x7f80u || r == 0xff80u) return 0;
        if (r == 0x8000u) r = 0;
        return (r & 0x8000u) ? (~r & 0xffffu) : (r | 0x8000u);
    }
    static __device__ __forceinline__ uint32_t key_below(float v) { return key(__bfloat16_as_ushort(__float2bfloat16_rd(v))); }
    static __device__ __forceinline__ uint32_t key_above(float v) { return key(__bfloat16_as_ushort(__float2bfloat16_ru(v))); }
    static __device__ __forceinline__ float value(uint32_t k) {
        return __uint_as_float(((k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu)) << 16);
    }
};
template <> struct KeyOf<1> {      // fp16
    using Key = uint16_t;
    using Raw = uint16_t;
    static __device__ __forceinline__ uint32_t key(uint32_t r) {
        if ((r & 0x7fffu) > 0x7c00u || r == 0xfc00u) return 0;
        if (r == 0x8000u) r = 0;
        return (r & 0x8000u) ? (~r & 0xffffu) : (r | 0x8000u);
    }
    static __device__ __forceinline__ uint32_t key_below(float v) { return key(__half_as_ushort(__float2half_rd(v))); }
    static __device__ __forceinline__ uint32_t key_above(float v) { return key(__half_as_ushort(__float2half_ru(v))); }
    static __device__ __forceinline__ float value(uint32_t k) {
        return __half2float(__ushort_as_half((unsigned short)((k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu))));
    }
};
template <> struct KeyOf<2> {      // fp32
    using Key = uint32_t;
    using Raw = uint32_t;
    static __device__ __forceinline__ uint32_t key(uint32_t r) {
        if ((r & 0x7fffffffu) > 0x7f800000u || r == 0xff800000u) return 0;
        if (r == 0x80000000u) r = 0;
        return (r & 0x80000000u) ? ~r : (r | 0x80000000u);
    }
    static __device__ __forceinline__ uint32_t key_below(float v) { return key(__float_as_uint(v)); }
    static __device__ __forceinline__ uint32_t key_above(float v) { return key(__float_as_uint(v)); }
    static __device__ __forceinline__ float value(uint32_t k) {
        return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
    }
};

constexpr int kBins = 2048, kCoarse = 64, kFine = kBins / kCoarse;
constexpr int kListMax = 512;      // tokens of a border bin that are compared pairwise
constexpr int kShortList = 256;    // tokens down to the k-th for which the list is all
constexpr int kMaxCluster = 8;
constexpr int kTableBits = 9, kTable = 1 << kTableBits;

struct SampleShared {
    // bin 0 holds the largest logits; lo: sum of offsets into a linear bin; hi:lo: sum of weights (radix descent)
    uint32_t cnt[kBins], lo[kBins], hi[kBins];
    __align__(16) unsigned long long coarse_w[kCoarse];// published: sums of 32 bins; the bits of a float estimate for linear bins
    uint32_t coarse_c[kCoarse];
    double table[kTable];                              // 2^(i/kTable)
    unsigned long long list[2][kListMax];              // published, by search: tokens of the border bins, key << 32 | ~index
    uint32_t list_n[2], list_at[kMaxCluster];          // list_at: running total of the CTAs' list_n
    ulonglong2 sums[2], all_sums;                      // published, by search: weight above the listed bins, below them
    unsigned long long all[kListMax], all_w[kListMax]; // the lists of the whole cluster
    unsigned long long warp_w[kSampleWarps], warp_x[kSampleWarps];
    uint32_t warp_c[kSampleWarps], warp_min[kSampleWarps];
    uint2 best;                                        // published: largest key, smallest drawable key - 1
    uint32_t first;                                    // published: lowest index of the largest key (greedy)
    unsigned long long pub_w;                          // published: kept weight of this CTA
    uint32_t pub_ties;                                 // published: tokens equal to the border key
    unsigned long long border;
    // result of find_bin
    uint32_t bin, last, above_c, eq_c, total_c;
    unsigned long long above_w;
};

__device__ __forceinline__ unsigned long long warp_sum_u64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    return v;
}
template <typename U> __device__ __forceinline__ U warp_scan(U v, int lane) {   // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const U n = __shfl_up_sync(kFullMask, v, o);
        if (lane >= o) v += n;
    }
    return v;
}
__device__ __forceinline__ unsigned long long token_of(uint32_t key, int index) {
    return ((unsigned long long)key << 32) | (uint32_t)~index;
}

// floor(part * whole) for 0 <= part < 1, exactly (a double holds 53 of the 62 bits of a sum of weights: among equal tokens the
// product would fall beside the running sum that it is equal to); `exact`: nothing was cut off
__device__ __forceinline__ unsigned long long part_of(float part, unsigned long long whole, bool& exact) {
    const uint32_t b = __float_as_uint(part), e = max(b >> 23, 1u), m = (b & 0x7fffffu) | (b >> 23 ? 0x800000u : 0u);
    const int shift = 150 - (int)e;                           // part = m * 2^-shift, shift 24..149
    const unsigned long long lo = m * whole, hi = __umul64hi(m, whole);
    if (shift < 64) {
        exact = (lo & ((1ull << shift) - 1)) == 0;
        return (hi << (64 - shift)) | (lo >> shift);
    }
    const int s = min(shift - 64, 63);                        // hi < 2^23
    exact = lo == 0 && (hi & ((1ull << s) - 1)) == 0;
    return hi >> s;
}

// double(v) by integer operations (a conversion costs as much as four 64-bit products); subnormals come out wrong by
// less than 2^-126 and infinity as 2^128
__device__ __forceinline__ double widen(float v) {
    const uint32_t b = __float_as_uint(v);
    return __hiloint2double((int)((((b & 0x7fffffffu) >> 3) + 0x38000000u) | (b & 0x80000000u)), (int)(b << 29));
}
struct Weigher {
    double max, scale, unit;    // scale = kTable log2(e) / T, unit = 2^frac
    int frac;
    float cut;                  // logits below it weigh nothing; the caller leaves them out
    const double* table;
    __device__ Weigher(float largest, float T, int frac, const double* table) : frac(frac), table(table) {
        max = widen(largest);
        scale = kTable * 1.4426950408889634 / (double)T;
        unit = (double)(1ull << frac);
        // e^-707 > 2^-1021, rounded up: what passes has a normal 2^t; +inf where the largest logit is +inf
        cut = __fadd_ru(largest, __fmul_ru(-707.f, T));
    }
    // unit * exp((v - max) / T) rounded, plus 1: u = 0 draws the first kept token whatever it weighs.  Not for logits below
    // the cut (a mask of the type's lowest value, anything below a largest logit of +inf): they weigh 0, are never drawn.
    __device__ __forceinline__ unsigned long long operator()(float v) const {
        constexpr double kRound = 6755399441055744.0;             // 1.5 * 2^52: adding it rounds to an integer
        constexpr double kLn = 0.6931471805599453 / kTable;
        const double d = widen(v) - max;
        const double nd = fma(d, scale, kRound);
        const int n = __double2loint(nd);
        const double r = fma(d, scale, kRound - nd);
        const double p = fma(r * r, fma(r, kLn * kLn * kLn / 6.0, kLn * kLn / 2.0), fma(r, kLn, 1.0));
        const double t = table[n & (kTable - 1)];
        const double scaled = __hiloint2double(__double2hiint(t) + (((n >> kTableBits) + frac) << 20), __double2loint(t));
        // scaled * p <= 2^51: adding 2^52 leaves the rounded integer in the mantissa
        return (unsigned long long)__double_as_longlong(fma(scaled, p, 4503599627370497.0)) & 0xfffffffffffffull;
    }
    // log of a token's share of the kept weight z, not through its rounded weight
    __device__ __forceinline__ float log_share(float v, unsigned long long z) const {
        return (float)((widen(v) - max) * scale * (0.6931471805599453 / kTable) - log((double)z / unit));
    }
    // smallest weight that passes min_p
    __device__ __forceinline__ unsigned long long least(float min_p) const {
        return min_p > 0.f ? __double2ull_rn(fmin((double)min_p, 1.0) * unit) + 1 : 1;
    }
};

// Estimated weight of the n tokens of a linear bin, relative to the row's largest: all at their mean offset into the bin
// (off, a sum of 64ths); `step` binades per bin.
__device__ __forceinline__ float bin_weight(int bin, uint32_t n, uint32_t off, float step) {
    return n ? (float)n * exp2f(-((float)bin + ((float)off + 0.5f * (float)n) / (64.f * (float)n)) * step) : 0.f;
}

__device__ __forceinline__ void clear_bins(SampleShared& sh) {
    uint4* p = reinterpret_cast<uint4*>(sh.cnt);
    for (int i = threadIdx.x; i < 3 * kBins / 4; i += kSampleThreads) p[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
}
// Sums of 32 bins each, then the histogram is readable by the whole cluster.
template <bool kExact> __device__ __forceinline__ void publish_bins(SampleShared& sh, float step, cg::cluster_group& cluster) {
    __syncthreads();
    static_assert(kBins == 4 * kSampleThreads && kFine == 32, "four bins a thread, eight threads a coarse bin");
    const int tid = threadIdx.x;
    const uint4 n = reinterpret_cast<const uint4*>(sh.cnt)[tid];
    uint32_t c = n.x + n.y + n.z + n.w;
    unsigned long long w = 0;
    float e = 0.f;
    if (kExact) {
        const uint4 l = reinterpret_cast<const uint4*>(sh.lo)[tid], h = reinterpret_cast<const uint4*>(sh.hi)[tid];
        w = ((unsigned long long)(h.x + h.y + h.z + h.w) << 32) + ((unsigned long long)l.x + l.y + l.z + l.w);
    } else {
        const uint4 f = reinterpret_cast<const uint4*>(sh.lo)[tid];
        e = bin_weight(4 * tid, n.x, f.x, step) + bin_weight(4 * tid + 1, n.y, f.y, step) +
            bin_weight(4 * tid + 2, n.z, f.z, step) + bin_weight(4 * tid + 3, n.w, f.w, step);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        c += __shfl_xor_sync(kFullMask, c, o);
        if (kExact) w += __shfl_xor_sync(kFullMask, w, o);
        else e += __shfl_xor_sync(kFullMask, e, o);
    }
    if ((tid & 7) == 0) {
        sh.coarse_c[tid >> 3] = c;
        sh.coarse_w[tid >> 3] = kExact ? w : (unsigned long long)__float_as_uint(e);
    }
    cluster.sync();
}
// Where a search of the histogram ends: by count, or by weight (exact, or the estimate for linear bins).
//
// By count: the bin, from the largest logits down, in which the running count reaches `target`, what lies above being
// above_c and above_w.  By exact weight: the same for the running weight.  By estimate: the bin in which the estimated
// weight reaches `share` of the total (`total` where that is > 0), and its neighbour where the goal is within the estimate's
// error of the border (the spread inside a bin: (step ln 2)^2 / 24, 1.6e-5 for bins down to 40 T; where they are wider
// the exact sums show a miss, and the bits of the keys are searched).
template <bool kExact>
__device__ __forceinline__ void find_bin(SampleShared& sh, bool by_count, unsigned long long target, uint32_t above_c,
                                         unsigned long long above_w, float share, float total, float step,
                                         cg::cluster_group& cluster) {
    const int tid = threadIdx.x, lane = tid & 31, C = (int)cluster.num_blocks();
    uint32_t* part_c = reinterpret_cast<uint32_t*>(sh.all);                  // scratch: [CTA][64], then [CTA][32]
    unsigned long long* part_w = sh.all_w;
    static_assert(kSampleThreads == kMaxCluster * kCoarse && kListMax >= kSampleThreads, "one thread per CTA and coarse bin");
    __syncthreads();                                   // the last result, and the scratch, have been read
    if ((tid >> 6) < C) {
        const SampleShared* o = cluster.map_shared_rank(&sh, tid >> 6);
        part_c[tid] = o->coarse_c[tid & 63];
        part_w[tid] = o->coarse_w[tid & 63];
    }
    __syncthreads();
    uint32_t uc = 0;
    unsigned long long uw = 0;
    float ue = 0.f, goal = 0.f, near = 0.f;
    uint32_t all_c = 0;
    if (tid < 32) {
        uint32_t c0 = 0, c1 = 0;
        unsigned long long w0 = 0, w1 = 0;
        float e0 = 0.f, e1 = 0.f;
#pragma unroll 1
        for (int r = 0; r < C; ++r) {
            const uint2 n = *reinterpret_cast<const uint2*>(&part_c[r * kCoarse + 2 * lane]);
            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&part_w[r * kCoarse + 2 * lane]);
            c0 += n.x;
            c1 += n.y;
            if (kExact) {
                w0 += x.x;
                w1 += x.y;
            } else {
                e0 += __uint_as_float((uint32_t)x.x);
                e1 += __uint_as_float((uint32_t)x.y);
            }
        }
        const uint32_t ic = above_c + warp_scan(c0 + c1, lane);
        all_c = __shfl_sync(kFullMask, ic, 31);
        uc = ic - c0 - c1;                             // above this lane's bins
        bool reached, second;
        if (kExact) {
            const unsigned long long iw = above_w + warp_scan(w0 + w1, lane);
            uw = iw - w0 - w1;
            reached = (by_count ? ic : iw) >= target;
            second = (by_count ? uc + c0 : uw + w0) < target;
        } else {
            const float ie = warp_scan(e0 + e1, lane);
            if (!(total > 0.f)) total = __shfl_sync(kFullMask, ie, 31);
            goal = share * total;
            near = 4e-5f * total;
            ue = ie - e0 - e1;
            reached = by_count ? ic >= target : ie >= goal;
            second = by_count ? uc + c0 < target : ue + e0 < goal;
        }
        const unsigned hit = __ballot_sync(kFullMask, reached);
        const int owner = hit ? __ffs(hit) - 1 : 31;
        uc = __shfl_sync(kFullMask, uc + (second ? c0 : 0), owner);
        if (kExact) uw = __shfl_sync(kFullMask, uw + (second ? w0 : 0), owner);
        else ue = __shfl_sync(kFullMask, ue + (second ? e0 : 0.f), owner);
        if (lane == owner) sh.bin = 2 * lane + (second ? 1 : 0);
    }
    __syncthreads();
    const int b = (int)sh.bin * kFine + lane;
    if ((tid >> 5) < C) {
        const SampleShared* o = cluster.map_shared_rank(&sh, tid >> 5);
        part_c[tid] = o->cnt[b];
        part_w[tid] = kExact ? ((unsigned long long)o->hi[b] << 32) + o->lo[b] : o->lo[b];
    }
    __syncthreads();
    if (tid < 32) {
        uint32_t n = 0;
        unsigned long long x = 0;
#pragma unroll 1
        for (int r = 0; r < C; ++r) {
            n += part_c[r * 32 + lane];
            x += part_w[r * 32 + lane];
        }
        const uint32_t jc = uc + warp_scan(n, lane);
        unsigned long long jw = 0;
        float e = 0.f, je = 0.f;
        bool reached;
        if (kExact) {
            jw = uw + warp_scan(x, lane);
            reached = (by_count ? jc : jw) >= target;
        } else {
            e = bin_weight(b, n, (uint32_t)x, step);
            je = ue + warp_scan(e, lane);
            reached = by_count ? jc >= target : je >= goal;
        }
        const unsigned hit = __ballot_sync(kFullMask, reached);
        if (lane == (hit ? __ffs(hit) - 1 : 31)) {
            sh.bin = kExact || by_count || je - e < goal - near ? b : max(b - 1, 0);
            sh.last = kExact || by_count || je > goal + near ? b : b + 1;
            sh.above_c = jc - n;
            sh.eq_c = n;
            sh.total_c = all_c;
            sh.above_w = jw - x;
        }
    }
    __syncthreads();
}

// Radix descent over the key, 11 bits a level (digits inverted: bin 0 holds the largest), with exact sums: the border
// token at which the count or the weight reaches the target, and the weight kept.  The way for rows that the linear bins do
// not settle; keys[0..n) is this CTA's slice, which starts at token `begin`.
template <int DT>
__device__ __noinline__ void radix_border(SampleShared& sh, const typename KeyOf<DT>::Key* keys, int n, int begin, const Weigher& weight,
                                          bool by_count, unsigned long long target, unsigned long long& border,
                                          unsigned long long& kept) {
    using K = KeyOf<DT>;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t cut_key = max(K::key_above(weight.cut), 1u);
    auto weight_of = [&](uint32_t k) -> unsigned long long { return k >= cut_key ? weight(K::value(k)) : 0; };
    uint32_t prefix = 0, above_c = 0;
    unsigned long long above = 0;
    for (int top = 8 * sizeof(typename K::Key); top > 0;) {
        const int shift = max(top - 11, 0);
        cluster.sync();                                // peers may still be reading the last histogram
        clear_bins(sh);
        for (int i = tid; i < n; i += kSampleThreads) {
            const uint32_t k = keys[i];
            if (k == 0 || (uint32_t)((unsigned long long)k >> top) != prefix) continue;
            const uint32_t bin = kBins - 1 - ((k >> shift) & ((1u << (top - shift)) - 1));
            const unsigned long long w = weight_of(k);
            const uint32_t lo = (uint32_t)w, old = atomicAdd(&sh.lo[bin], lo);       // two sums, the carry passed on
            const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
            atomicAdd(&sh.cnt[bin], 1u);
            if (hi) atomicAdd(&sh.hi[bin], hi);
        }
        publish_bins<true>(sh, 0.f, cluster);
        find_bin<true>(sh, by_count, target, above_c, above, 0.f, 0.f, 0.f, cluster);
        prefix = (prefix << (top - shift)) | (kBins - 1 - sh.bin);
        above_c = sh.above_c;
        above = sh.above_w;
        top = shift;
    }
    const unsigned long long one = weight_of(prefix);
    const uint32_t ties = sh.eq_c;
    unsigned long long keep = by_count ? target - above_c : (one ? (target - above + one - 1) / one : 1);
    keep = min(keep, (unsigned long long)ties);
    kept = above + keep * one;
    border = (unsigned long long)prefix << 32;
    if (keep == ties) return;
    // the keep-th of the ties in index order: warp w counts a contiguous run
    const int run = ((n + kSampleWarps - 1) / kSampleWarps + 31) / 32 * 32;
    const int r0 = min(warp * run, n), r1 = min(r0 + run, n);
    uint32_t c = 0;
    for (int i = r0 + lane; i < r1; i += 32) c += keys[i] == prefix;
    c = __reduce_add_sync(kFullMask, c);
    if (lane == 0) sh.warp_c[warp] = c;
    __syncthreads();
    uint32_t before = 0, mine = 0;
    for (int i = 0; i < kSampleWarps; ++i) {
        if (i < warp) before += sh.warp_c[i];
        mine += sh.warp_c[i];
    }
    if (tid == 0) sh.pub_ties = mine;
    cluster.sync();
    for (int r = 0; r < rank; ++r) before += cluster.map_shared_rank(&sh, r)->pub_ties;
    if (before < keep && keep <= before + c) {
        for (int i0 = r0; i0 < r1; i0 += 32) {
            const int i = i0 + lane;
            const unsigned eq = __ballot_sync(kFullMask, i < r1 && keys[i] == prefix);
            if (before + __popc(eq) >= keep) {
                const int at = begin + i0 + __fns(eq, 0, (int)(keep - before));
                if (lane < C) cluster.map_shared_rank(&sh, lane)->border = token_of(prefix, at);
                break;
            }
            before += __popc(eq);
        }
    }
    cluster.sync();
    border = sh.border;
}

constexpr size_t kSampleShared = (sizeof(SampleShared) + 15) / 16 * 16;
constexpr int kSampleMost = 227 * 1024;                    // a block's shared memory
static_assert(kSampleShared + (size_t)kSampleMaxVocab / kMaxCluster * 4 <= kSampleMost, "the largest slice fits");

template <int DT>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(SampleParams p) {
    using K = KeyOf<DT>;
    using Key = typename K::Key;
    using Raw = typename K::Raw;
    constexpr int kVec = 16 / sizeof(Raw);             // logits per 16-byte load
    extern __shared__ __align__(16) unsigned char smem[];
    SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
    Key* keys = reinterpret_cast<Key*>(smem + kSampleShared);
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int begin = min(rank * p.slice, p.vocab), n = min(p.vocab - begin, p.slice);

    // ---- keys of this slice (filled up with key 0 to whole 16-byte vectors), the largest and the smallest drawable one
    const Raw* src = static_cast<const Raw*>(p.logits) + (long long)row * p.row_stride + begin;
    uint32_t largest = 0, least = 0xffffffffu;         // per 16-bit half for 16-bit keys; least - 1, so that key 0 is last
    auto seen_word = [&](uint32_t o) {
        largest = sizeof(Raw) == 2 ? __vmaxu2(largest, o) : max(largest, o);
        least = sizeof(Raw) == 2 ? __vminu2(least, __vsub2(o, 0x00010001u)) : min(least, o - 1);
    };
    auto key_word = [&](uint32_t r) { return sizeof(Raw) == 2 ? K::key(r & 0xffffu) | (K::key(r >> 16) << 16) : K::key(r); };
    const int vectors = (n + kVec - 1) / kVec;
    uint4* keys4 = reinterpret_cast<uint4*>(keys);
    const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
    const int nv = vec ? n / kVec : 0;
    constexpr int kAhead = 4;
#pragma unroll
    for (int a = 0; a < kAhead; ++a)                   // on their way while the tables are set up
        if (tid + a * kSampleThreads < nv)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(src + (tid + a * kSampleThreads) * kVec));
    static_assert(kTable <= kSampleThreads, "an entry a thread");
    if (tid < kTable) sh.table[tid] = exp2((double)tid / kTable);
    if (tid < 2) sh.list_n[tid] = 0;
    clear_bins(sh);
    for (int i0 = tid; i0 < nv; i0 += kAhead * kSampleThreads) {
        uint4 q[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (i0 + a * kSampleThreads < nv) q[a] = ld_stream_16(src + (i0 + a * kSampleThreads) * kVec);
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int i = i0 + a * kSampleThreads;
            if (i < nv) {
                const uint4 o = make_uint4(key_word(q[a].x), key_word(q[a].y), key_word(q[a].z), key_word(q[a].w));
                seen_word(o.x); seen_word(o.y); seen_word(o.z); seen_word(o.w);
                keys4[i] = o;
            }
        }
    }
    for (int i = nv * kVec + tid; i < vectors * kVec; i += kSampleThreads) {
        const uint32_t k = i < n ? K::key(src[i]) : 0;
        keys[i] = (Key)k;
        seen_word(sizeof(Raw) == 2 ? k | (k << 16) : k);
    }
    if (sizeof(Raw) == 2) {
        largest = max(largest & 0xffffu, largest >> 16);
        least = min(least & 0xffffu, least >> 16);
    }
    largest = __reduce_max_sync(kFullMask, largest);
    least = __reduce_min_sync(kFullMask, least);
    if (lane == 0) {
        sh.warp_c[warp] = largest;
        sh.warp_min[warp] = least;
    }
    __syncthreads();
    if (warp == 0) {
        largest = __reduce_max_sync(kFullMask, lane < kSampleWarps ? sh.warp_c[lane] : 0);
        least = __reduce_min_sync(kFullMask, lane < kSampleWarps ? sh.warp_min[lane] : 0xffffffffu);
        if (lane == 0) sh.best = make_uint2(largest, least);
    }
    cluster.sync();
    uint32_t kmax = 0;
    least = 0xffffffffu;
    if (lane < C) {
        const uint2 x = cluster.map_shared_rank(&sh, lane)->best;
        kmax = x.x;
        least = x.y;
    }
    kmax = __reduce_max_sync(kFullMask, kmax);
    least = __reduce_min_sync(kFullMask, least);
    least += 1;                                        // wraps to 0 where nothing is drawable

    // f(key, index in the slice) for the four keys of quad i
    const int quads = (n + 3) / 4;
    auto each_key = [&](int i, auto&& f) {
        if (sizeof(Raw) == 2) {
            const uint2 q = reinterpret_cast<const uint2*>(keys)[i];
            f(q.x & 0xffffu, i * 4);
            f(q.x >> 16, i * 4 + 1);
            f(q.y & 0xffffu, i * 4 + 2);
            f(q.y >> 16, i * 4 + 3);
        } else {
            const uint4 q = keys4[i];
            f(q.x, i * 4);
            f(q.y, i * 4 + 1);
            f(q.z, i * 4 + 2);
            f(q.w, i * 4 + 3);
        }
    };

    const float given_T = p.temperature ? p.temperature[row] : p.temperature_v, T = given_T > 1e35f ? 1e35f : given_T;
    if (kmax == 0 || !(T > 0.f)) {                     // nothing to draw, or greedy (T <= 0, NaN): the lowest index
        uint32_t first = 0xffffffffu;
        if (kmax != 0)
            for (int i = tid; i < quads; i += kSampleThreads)
                each_key(i, [&](uint32_t k, int at) {
                    if (k == kmax) first = min(first, (uint32_t)(begin + at));
                });
        first = __reduce_min_sync(kFullMask, first);
        if (lane == 0) sh.warp_min[warp] = first;
        __syncthreads();
        if (warp == 0) {
            first = __reduce_min_sync(kFullMask, lane < kSampleWarps ? sh.warp_min[lane] : 0xffffffffu);
            if (lane == 0) sh.first = first;
        }
        cluster.sync();
        if (rank == 0 && warp == 0) first = __reduce_min_sync(kFullMask, lane < C ? cluster.map_shared_rank(&sh, lane)->first : 0xffffffffu);
        if (rank == 0 && tid == 0) {
            p.ids[row] = kmax == 0 ? 0 : (long long)first;
            if (p.logprobs) p.logprobs[row] = kmax == 0 ? __int_as_float(0x7fc00000) : 0.f;
        }
        cluster.sync();                                // rank 0 has read its peers
        return;
    }
    const float vmax = K::value(kmax);
    const Weigher weight(vmax, T, p.frac, sh.table);
    const uint32_t cut_key = max(K::key_above(weight.cut), 1u);              // keys below it weigh nothing
    auto weight_of = [&](uint32_t k) -> unsigned long long { return k >= cut_key ? weight(K::value(k)) : 0; };

    const int top_k = p.top_k ? p.top_k[row] : p.top_k_v;
    const float given_p = p.top_p ? p.top_p[row] : p.top_p_v, top_p = fmaxf(given_p, 0.f);
    const float min_p = p.min_p ? p.min_p[row] : p.min_p_v;
    const float u = fmaxf(p.uniform[row], 0.f);                              // NaN: 0
    const bool by_k = top_k > 0 && top_k < p.vocab, by_p = given_p < 1.f;                   // NaN: off
    auto least_target = [](float part, unsigned long long whole) {           // smallest integer >= part * whole, 1..whole; part < 1
        bool exact;
        const unsigned long long t = part_of(part, whole, exact);
        return max(t + (exact ? 0 : 1), 1ull);
    };
    auto draw_target = [&](unsigned long long whole) {
        bool exact;
        return u >= 1.f ? whole - 1 : part_of(u, whole, exact);
    };
    const unsigned long long least_w = weight.least(min_p);

    // index order: warp w of the CTA owns a contiguous run of the slice
    const int run_quads = (quads + kSampleWarps - 1) / kSampleWarps, run = run_quads * 4;
    const int q0 = min(warp * run_quads, quads), q1 = min(q0 + run_quads, quads);
    const int r0 = min(warp * run, n), r1 = min(r0 + run, n);

    unsigned long long border = 1ull << 32;            // tokens (key, index) at or above it stay; here any drawable key
    unsigned long long run_above = 0;                  // weight of this warp's run above the listed bins
    uint32_t listed = 0;                               // with run_above: the tokens of sh.all at or above the border
    bool have_runs = false;
    if (by_k || by_p) {
        // bins of equal width down to 40 T below the maximum (e^-40 of its weight), the rest in the last bin; monotone in
        // the logit whatever the rounding.  Where the top k are counted, to 40 at least: their number does not depend on
        // T (64 rows of deviation 3, T 0.1, top-k 50: 21.2 us, 46.7 with bins down to 40 T)
        const float vref = fminf(vmax, 3.4028235e38f), range = fminf(vref - K::value(least), 40.f * (by_k ? fmaxf(T, 1.f) : T));
        const float per = range > 0.f ? fminf((float)(kBins - 1) / range, 1e30f) : 0.f;
        const float step = per > 0.f ? fminf(1.4426950408889634f / (T * per), 1e30f) : 0.f;
        auto place = [&](uint32_t k) { return fminf(fmaxf((vref - K::value(k)) * per, 0.f), (float)(kBins - 1)); };
        auto linear = [&](uint32_t k) -> uint32_t { return (uint32_t)place(k); };   // of +inf: bin 0
        uint32_t rest = 0;                             // the last bin may hold most of a row: counted a warp at a time
        for (int i = tid; i < quads; i += kSampleThreads)
            each_key(i, [&](uint32_t k, int) {
                if (k == 0) return;
                const float at = place(k);
                const uint32_t bin = (uint32_t)at;
                if (bin == kBins - 1) {                // at == bin: nothing for sh.lo
                    ++rest;
                    return;
                }
                atomicAdd(&sh.cnt[bin], 1u);
                if (by_p) atomicAdd(&sh.lo[bin], (uint32_t)((at - (float)bin) * 64.f));
            });
        rest = __reduce_add_sync(kFullMask, rest);
        if (lane == 0 && rest) atomicAdd(&sh.cnt[kBins - 1], rest);
        publish_bins<false>(sh, step, cluster);
        unsigned long long z = 0;                      // weight of what the filters so far keep; 0: not known yet

        // Smallest key whose linear bin is at most `limit` (a 32-way search by the lanes of a warp; bins fall as keys grow):
        // the passes below compare keys instead of computing bins.
        auto lowest_key = [&](int limit) -> uint32_t {
            if (limit < 0) return kmax + 1;
            uint32_t lo = least - 1, hi = kmax;
#pragma unroll 1
            while (hi - lo > 1) {
                const uint32_t by = (hi - lo + 31) / 32, at = min(lo + by * (lane + 1), hi);
                const int f = __ffs(__ballot_sync(kFullMask, (int)linear(at) <= limit)) - 1;   // the last lane passes
                hi = __shfl_sync(kFullMask, at, f);
                lo += by * f;
            }
            return hi;
        };
        // Lists the tokens of bins first..last, adds up the weight above them (into run_above for this warp's run) and,
        // where asked, below them; then the cluster's lists are in sh.all / sh.all_w.  Returns the number listed, which
        // may exceed kListMax (then nothing is in sh.all).
        unsigned long long above_w = 0, below_w = 0;
        auto scan = [&](int search, int first, int last, bool below) -> uint32_t {
            const uint32_t above_key = lowest_key(first - 1), list_key = lowest_key(last);
            unsigned long long a = 0, b = 0;
            for (int i = q0 + lane; i < q1; i += 32) {
                bool some = false, heavy = below;
                each_key(i, [&](uint32_t k, int) {
                    some |= k >= list_key && k < above_key;
                    heavy |= k >= above_key;
                });
                if (heavy)
                    each_key(i, [&](uint32_t k, int) {
                        const unsigned long long w = weight(K::value(k));
                        if (k >= above_key && k >= cut_key) a += w;
                        if (k < list_key && k >= cut_key) b += w;
                    });
                if (some)
                    each_key(i, [&](uint32_t k, int at) {
                        if (k >= list_key && k < above_key) {
                            const uint32_t slot = atomicAdd(&sh.list_n[search], 1u);
                            if (slot < kListMax) sh.list[search][slot] = token_of(k, begin + at);
                        }
                    });
            }
            run_above = a = warp_sum_u64(a);
            b = below ? warp_sum_u64(b) : 0;
            __syncthreads();                           // the last use of warp_w, warp_x
            if (lane == 0) {
                sh.warp_w[warp] = a;
                sh.warp_x[warp] = b;
            }
            __syncthreads();
            if (warp == 0) {
                a = warp_sum_u64(lane < kSampleWarps ? sh.warp_w[lane] : 0);
                b = warp_sum_u64(lane < kSampleWarps ? sh.warp_x[lane] : 0);
                if (lane == 0) sh.sums[search] = make_ulonglong2(a, b);
            }
            cluster.sync();
            if (warp == 0) {                           // lane r asks CTA r
                uint32_t c = 0;
                ulonglong2 x = make_ulonglong2(0, 0);
                if (lane < C) {
                    const SampleShared* o = cluster.map_shared_rank(&sh, lane);
                    c = o->list_n[search];
                    x = o->sums[search];
                }
                const uint32_t at = warp_scan(c, lane);
                if (lane < kMaxCluster) sh.list_at[lane] = at;
                x.x = warp_sum_u64(x.x);
                x.y = warp_sum_u64(x.y);
                if (lane == 0) sh.all_sums = x;
            }
            __syncthreads();
            uint32_t from = 0, peer = 0;               // thread i takes token i: which CTA holds it, and where
            const uint32_t end = sh.list_at[kMaxCluster - 1];
            above_w = sh.all_sums.x;
            below_w = sh.all_sums.y;
#pragma unroll 1
            for (int r = 0; r < C - 1; ++r)
                if ((uint32_t)tid >= sh.list_at[r]) {
                    from = sh.list_at[r];
                    peer = r + 1;
                }
            if ((uint32_t)tid < end && end <= kListMax) {
                const unsigned long long x = cluster.map_shared_rank(&sh, (int)peer)->list[search][tid - from];
                const uint32_t k = (uint32_t)(x >> 32);
                sh.all[tid] = x;
                sh.all_w[tid] = weight_of(k);
            }
            __syncthreads();
            return end;
        };
        // Per listed token (a power-of-two group of lanes shares one): how many tokens of the list precede it, and their
        // weight; by size, or by index.
        auto compare = [&](uint32_t m, uint32_t& e, uint32_t& sub, uint32_t& c, unsigned long long& w, bool by_index) {
            int lanes = 1;
            while (lanes < 32 && (uint32_t)(kSampleThreads / (lanes * 2)) >= m) lanes *= 2;
            e = tid / lanes;
            sub = tid & (lanes - 1);
            c = 0;
            w = 0;
            if (e < m) {
                const unsigned long long mask = by_index ? 0xffffffffull : ~0ull, x = sh.all[e] & mask;
#pragma unroll 2
                for (uint32_t j = sub; j < m; j += lanes) {
                    const bool before = (sh.all[j] & mask) > x;
                    const unsigned long long y = sh.all_w[j];
                    c += before;
                    w += before ? y : 0;
                }
            }
            __syncwarp();
            for (int o = 1; o < lanes; o *= 2) {
                c += __shfl_xor_sync(kFullMask, c, o);
                w += __shfl_xor_sync(kFullMask, w, o);
            }
        };
        auto block_sum = [&](unsigned long long v) {
            v = warp_sum_u64(v);
            __syncthreads();
            if (lane == 0) sh.warp_w[warp] = v;
            __syncthreads();
            return warp_sum_u64(lane < kSampleWarps ? sh.warp_w[lane] : 0);
        };
        auto block_min = [&](unsigned long long v) {
            // the smallest of 64 bits: of the high words, then of the low words that go with it
            auto warp_min = [](unsigned long long x) {
                const uint32_t hi = __reduce_min_sync(kFullMask, (uint32_t)(x >> 32));
                return ((unsigned long long)hi << 32) | __reduce_min_sync(kFullMask, (uint32_t)(x >> 32) == hi ? (uint32_t)x : 0xffffffffu);
            };
            v = warp_min(v);
            __syncthreads();
            if (lane == 0) sh.warp_w[warp] = v;
            __syncthreads();
            return warp_min(lane < kSampleWarps ? sh.warp_w[lane] : ~0ull);
        };
        bool linear_bins = true;                       // the histogram in shared memory is the one over linear bins
#pragma unroll 1
        for (int pass = 0; pass < 2; ++pass) {
            const bool by_count = pass == 0;
            if (!(by_count ? by_k : by_p)) continue;
            unsigned long long target = (unsigned long long)top_k;
            bool settled = false;
            if (linear_bins) {
                find_bin<false>(sh, by_count, target, 0, 0, top_p, (float)((double)z / weight.unit), step, cluster);
                if (by_count && (uint32_t)top_k >= sh.total_c) continue;     // everything drawable stays
                const uint32_t above_c = sh.above_c;
                const bool is_short = by_count && above_c + sh.eq_c <= kShortList;
                if (!by_count || sh.eq_c <= kListMax) {
                    const uint32_t m = scan(pass, is_short ? 0 : (int)sh.bin, (int)sh.last, !by_count && z == 0);
                    if (is_short && rank != 0) {
                        cluster.sync();
                        return;
                    }
                    if (m <= kListMax) {
                        uint32_t e, sub, c;
                        unsigned long long w;
                        if (!by_count) {
                            const unsigned long long in_list = block_sum((uint32_t)tid < m && sh.all[tid] >= border ? sh.all_w[tid] : 0);
                            if (z == 0) z = above_w + in_list + below_w;
                            target = least_target(top_p, z);
                            settled = above_w < target && target <= above_w + in_list;
                        } else {
                            settled = true;
                        }
                        if (settled) {
                            compare(m, e, sub, c, w, false);
                            const bool stays = e < m && (by_count ? (unsigned long long)((is_short ? 0 : above_c) + c) : above_w + w) < target;
                            const unsigned long long kept = block_sum(stays && sub == 0 ? sh.all_w[e] : 0);
                            if (is_short) {
                                // ---- everything down to the k-th token is on the list: the rest happens there, in one CTA
                                const bool in_p = stays && (!by_p || w < least_target(top_p, kept));
                                const unsigned long long mine = in_p && sh.all_w[e] >= least_w ? sh.all_w[e] : 0;
                                z = block_sum(sub == 0 ? mine : 0);
                                if (e < m && sub == 0) sh.all_w[e] = mine;    // block_sum's barriers: the old ones have been read
                                __syncthreads();
                                compare(m, e, sub, c, w, true);
                                const unsigned long long t = draw_target(z);
                                if (e < m && sub == 0 && w <= t && t < w + mine) {
                                    p.ids[row] = (long long)(uint32_t)~(uint32_t)sh.all[e];
                                    if (p.logprobs) p.logprobs[row] = weight.log_share(K::value((uint32_t)(sh.all[e] >> 32)), z);
                                }
                                cluster.sync();        // the lists have been read
                                return;
                            }
                            border = block_min(stays ? sh.all[e] : ~0ull);
                            if (by_count) z = above_w + kept;
                            listed = m;
                            have_runs = true;
                        }
                    }
                }
            }
            if (!settled) {
                if (!by_count && z == 0) {             // the weight of all, exactly
                    unsigned long long a = 0;
                    for (int i = tid; i < n; i += kSampleThreads) a += keys[i] ? weight_of(keys[i]) : 0;
                    a = block_sum(a);
                    if (tid == 0) sh.pub_w = a;
                    cluster.sync();
                    z = warp_sum_u64(lane < C ? cluster.map_shared_rank(&sh, lane)->pub_w : 0);
                }
                radix_border<DT>(sh, keys, n, begin, weight, by_count, by_count ? target : least_target(top_p, z), border, z);
                linear_bins = have_runs = false;
            }
        }
    }
    // ---- kept weight of each run in index order, and the draw
    // no key below `lowest` is kept: the border's, and what min_p leaves with a margin for rounding (next to nothing of a
    // vocabulary, as a rule: most weights are never computed)
    const uint32_t border_key = (uint32_t)(border >> 32), border_index = (uint32_t)border;
    uint32_t lowest = max(border_key, cut_key);
    if (min_p > 0.f)
        lowest = max(lowest, min(kmax, K::key_below(vmax + T * (logf(fminf(min_p, 1.f)) - 1e-3f) - 1e-6f * fabsf(vmax))));
    auto kept_weight = [&](uint32_t k, int i) -> unsigned long long {
        if (k < lowest || (k == border_key && (uint32_t)~(begin + i) < border_index)) return 0;
        const unsigned long long w = weight(K::value(k));
        return w >= least_w ? w : 0;
    };
    unsigned long long sum = 0;
    if (have_runs && !(min_p > 0.f)) {                 // known but for the listed tokens
        for (uint32_t j = lane; j < listed; j += 32) {
            const unsigned long long x = sh.all[j];
            const int at = (int)~(uint32_t)x - begin;
            if (x >= border && at >= r0 && at < r1) sum += sh.all_w[j];
        }
        sum = warp_sum_u64(sum) + run_above;
    } else {
        for (int i = q0 + lane; i < q1; i += 32) {
            bool some = false;
            each_key(i, [&](uint32_t k, int) { some |= k >= lowest; });
            if (some)
                each_key(i, [&](uint32_t k, int at) {
                    const unsigned long long w = weight(K::value(k));
                    if (k >= lowest && w >= least_w && (k != border_key || (uint32_t)~(begin + at) >= border_index)) sum += w;
                });
        }
        sum = warp_sum_u64(sum);
    }
    __syncthreads();                                   // warp_w of the border search has been read
    if (lane == 0) sh.warp_w[warp] = sum;
    __syncthreads();
    const unsigned long long mine = warp_sum_u64(lane < kSampleWarps ? sh.warp_w[lane] : 0);
    if (tid == 0) sh.pub_w = mine;
    cluster.sync();
    const unsigned long long theirs = lane < C ? cluster.map_shared_rank(&sh, lane)->pub_w : 0;
    const unsigned long long z = warp_sum_u64(theirs);
    unsigned long long base = warp_sum_u64(lane < rank ? theirs : 0);
    const unsigned long long target = draw_target(z);
    if (base <= target && target < base + mine) {      // one CTA of the cluster owns the draw
        int owner = 0;                                 // and one of its runs
        while (base + sh.warp_w[owner] <= target) base += sh.warp_w[owner++];
        const int b0 = min(owner * run, n), b1 = min(b0 + run, n);
        const int each = (run + kSampleThreads - 1) / kSampleThreads;
        const int i0 = min(b0 + tid * each, b1), i1 = min(i0 + each, b1);
        unsigned long long w = 0;
        for (int i = i0; i < i1; ++i) w += kept_weight(keys[i], i);
        const unsigned long long inc = warp_scan(w, lane);
        if (lane == 31) sh.warp_x[warp] = inc;
        __syncthreads();
        unsigned long long before = base + inc - w;
        for (int i = 0; i < warp; ++i) before += sh.warp_x[i];
        if (before <= target && target < before + w) {
            for (int i = i0; i < i1; ++i) {
                const unsigned long long x = kept_weight(keys[i], i);
                if (target < before + x) {
                    p.ids[row] = begin + i;
                    if (p.logprobs) p.logprobs[row] = weight.log_share(K::value(keys[i]), z);
                    break;
                }
                before += x;
            }
        }
    }
    cluster.sync();                                    // peers may still be reading this CTA's published sums
}

template <int DT>
int launch_sample(const SampleParams& p, int rows, int cluster, size_t smem, cudaStream_t st) {
    // the dynamic shared memory a launch may have, set once per device to the most one can need
    static std::atomic<unsigned long long> ready{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (!(ready.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(sample_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSampleMost);
        if (e != cudaSuccess) return (int)e;
        ready.fetch_or(bit, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * cluster));
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, sample_kernel<DT>, p);
}

}  // namespace pk

extern "C" int pk_sample(const PkSampleArgs* a) {
    using namespace pk;
    if (!a) return kErrNull;
    if (a->rows < 0 || a->rows > (1 << 24) || a->vocab <= 0 || a->vocab > kSampleMaxVocab || a->dtype < 0 || a->dtype > 2)
        return kErrShape;
    if (a->rows == 0) return kOk;
    if (!a->logits || !a->uniform || !a->ids) return kErrNull;
    const int es = a->dtype == 2 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(a->logits) % es || reinterpret_cast<uintptr_t>(a->ids) % 8) return kErrAlign;
    for (const void* x : {a->uniform, a->temperature, a->top_k, a->top_p, a->min_p, static_cast<const void*>(a->logprobs)})
        if (reinterpret_cast<uintptr_t>(x) % 4) return kErrAlign;
    // CTAs per row: as many as there are SMs for while rows are few (two or four for 64 rows make no difference: 31.6 us
    // and 31.1 with top-p), and enough for a slice of 64 KB, two of which fit an SM beside the 48 KB of tables.
    int cluster = 1;
    while (cluster < kMaxCluster && (long long)a->rows * cluster * 2 <= 148) cluster *= 2;
    while (cluster < kMaxCluster && (a->vocab + cluster - 1) / cluster > 64 * 1024 / es) cluster *= 2;
    SampleParams p{};
    p.logits = a->logits;
    p.row_stride = a->row_stride;
    p.vocab = a->vocab;
    p.slice = ((a->vocab + cluster - 1) / cluster + 7) / 8 * 8;
    int lg = 0;
    while ((1 << lg) < a->vocab) ++lg;
    p.frac = 62 - lg < 51 ? 62 - lg : 51;
    p.uniform = static_cast<const float*>(a->uniform);
    p.temperature = static_cast<const float*>(a->temperature);
    p.top_k = static_cast<const int*>(a->top_k);
    p.top_p = static_cast<const float*>(a->top_p);
    p.min_p = static_cast<const float*>(a->min_p);
    p.temperature_v = a->temperature_value;
    p.top_k_v = a->top_k_value;
    p.top_p_v = a->top_p_value;
    p.min_p_v = a->min_p_value;
    p.ids = static_cast<long long*>(a->ids);
    p.logprobs = static_cast<float*>(a->logprobs);
    const size_t smem = kSampleShared + (size_t)p.slice * es;
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    return a->dtype == 0 ? launch_sample<0>(p, a->rows, cluster, smem, st)
                         : (a->dtype == 1 ? launch_sample<1>(p, a->rows, cluster, smem, st)
                                          : launch_sample<2>(p, a->rows, cluster, smem, st));
}
