// Sampling of one token per row of logits: temperature, top-k, top-p and min-p from a given uniform number.
//
//   w_i = exp((l_i - max l) / T); order by (l descending, i ascending); keep the first k; of those the shortest prefix
//   whose weight reaches p * (their sum); drop w_i < min_p; draw the lowest index i with
//   sum of kept w_j, j <= i  >  u * (sum of kept w).
//
// All three filters keep a prefix of the same order, so no sort is needed: a radix descent over the ordered bit
// pattern of the logits (8 bits a level, a histogram of counts and weights) finds the key at which a prefix ends
// and how many of the tokens equal to it stay (lowest indices first).  A row is spread over a thread-block cluster:
// every CTA keeps its slice of keys in shared memory, histograms are merged through distributed shared memory, and
// one pass over the logits is all the memory traffic.
//
// Weights are integers, round(exp2(t) * 2^frac) computed in 64 bits with frac = min(52, 62 - ceil(log2 V)) and at
// least 1 (0 where the weight underflows a double): integer sums do not depend on their order, so a draw is the same for every cluster size and the border of
// a top-p set moves by no more than V * 2^-frac of the row's largest weight (2^-30 at V = 49152).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

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

// ---- ordered keys: key(a) < key(b) iff a < b; -0 and +0 share one key; NaN and -inf are key 0 ("never drawn")
template <int DT> struct KeyOf;
template <> struct KeyOf<0> {      // bf16
    using Key = uint16_t;
    using Raw = uint16_t;
    static __device__ __forceinline__ uint32_t key(uint32_t r) {
        if ((r & 0x7fffu) > 0x7f80u || r == 0xff80u) return 0;
        if (r == 0x8000u) r = 0;
        return (r & 0x8000u) ? (~r & 0xffffu) : (r | 0x8000u);
    }
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
    static __device__ __forceinline__ float value(uint32_t k) {
        return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
    }
};

struct Hist {
    uint32_t cnt[256], lo[256], hi[256];   // hi:lo = sum of weights
};
struct SampleShared {
    Hist hist[2];
    Hist first;                            // merged level-0 histogram
    Hist merged;
    unsigned long long warp_w[kSampleWarps];
    uint32_t warp_c[kSampleWarps];
    unsigned long long best;               // published: (key << 32 | ~index) of this CTA's largest key
    unsigned long long pub_w;              // published: kept weight of this CTA
    uint32_t pub_ties;                     // published: tokens equal to the border key
    // result of a descent step
    uint32_t digit, above_c, eq_c;
    unsigned long long above_w, eq_w;
};

__device__ __forceinline__ unsigned long long shfl_down_u64(unsigned long long v, int d) {
    return __shfl_down_sync(kFullMask, v, d);
}
__device__ __forceinline__ unsigned long long warp_sum_u64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    return v;
}
__device__ __forceinline__ unsigned long long warp_scan_u64(unsigned long long v, int lane) {   // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long n = __shfl_up_sync(kFullMask, v, o);
        if (lane >= o) v += n;
    }
    return v;
}

// exp((value(key) - max) / T) as a double; key != 0
struct Weigher {
    double max, scale;      // scale = log2(e) / T
    uint32_t kmax;
    double two_frac;
    __device__ __forceinline__ double relative(float v, uint32_t key) const {
        if (key == kmax) return 1.0;
        const double d = (double)v - max;
        return isinf(d) ? 0.0 : exp2(d * scale);
    }
    // at least 1, so that u = 0 draws the first kept token whatever it weighs; 0 where the weight underflows a double
    // (a mask of the type's lowest value, anything below a largest logit of +inf): such a token is never drawn
    __device__ __forceinline__ unsigned long long fixed(float v, uint32_t key) const {
        if (key == kmax) return __double2ull_rn(two_frac);
        const double d = (double)v - max;
        if (isinf(d)) return 0;
        const double e = exp2(d * scale);
        const unsigned long long w = __double2ull_rn(e * two_frac);
        return w > 1 ? w : (e > 0.0 ? 1 : 0);
    }
};

// One level of the descent: histogram of the keys whose bits above `shift + 8` are `prefix`, merged over the cluster.
template <int DT>
__device__ void histogram(const typename KeyOf<DT>::Key* keys, int n, int shift, uint32_t prefix, const Weigher& wt, Hist* mine,
                          Hist* merged, cg::cluster_group& cluster) {
    const int tid = threadIdx.x;
    for (int i = tid; i < 256; i += kSampleThreads) mine->cnt[i] = mine->lo[i] = mine->hi[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSampleThreads) {
        const uint32_t k = keys[i];
        if (k != 0 && (uint32_t)((unsigned long long)k >> (shift + 8)) == prefix) {
            const uint32_t b = (k >> shift) & 255u;
            const unsigned long long w = wt.fixed(KeyOf<DT>::value(k), k);
            atomicAdd(&mine->cnt[b], 1u);
            const uint32_t lo = (uint32_t)w, old = atomicAdd(&mine->lo[b], lo);
            const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old ? 1u : 0u);
            if (hi) atomicAdd(&mine->hi[b], hi);
        }
    }
    cluster.sync();
    const int c = (int)cluster.num_blocks();
    for (int i = tid; i < 256; i += kSampleThreads) {
        uint32_t cnt = 0;
        unsigned long long w = 0;
        for (int r = 0; r < c; ++r) {
            const Hist* h = cluster.map_shared_rank(mine, r);
            cnt += h->cnt[i];
            w += ((unsigned long long)h->hi[i] << 32) | h->lo[i];
        }
        merged->cnt[i] = cnt;
        merged->lo[i] = (uint32_t)w;
        merged->hi[i] = (uint32_t)(w >> 32);
    }
    __syncthreads();
}

// The bin, from the top, in which the running count (or weight) reaches the target; warp 0 of the CTA.
__device__ void find_bin(const Hist* h, bool by_count, unsigned long long target, uint32_t above_c, unsigned long long above_w,
                         SampleShared& sh) {
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        // lane owns bins 255 - 8 lane ... 248 - 8 lane
        unsigned long long c = 0, w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int b = 255 - 8 * lane - j;
            c += h->cnt[b];
            w += ((unsigned long long)h->hi[b] << 32) | h->lo[b];
        }
        const unsigned long long ic = warp_scan_u64(c, lane), iw = warp_scan_u64(w, lane);
        unsigned long long uc = above_c + ic - c, uw = above_w + iw - w;       // above this lane's bins
        const bool reached = (by_count ? above_c + ic : above_w + iw) >= target;
        const unsigned ballot = __ballot_sync(kFullMask, reached);
        const int owner = ballot ? __ffs(ballot) - 1 : 31;
        if (lane == owner) {
            for (int j = 0; j < 8; ++j) {
                const int b = 255 - 8 * lane - j;
                const uint32_t bc = h->cnt[b];
                const unsigned long long bw = ((unsigned long long)h->hi[b] << 32) | h->lo[b];
                if ((by_count ? uc + bc : uw + bw) >= target || j == 7) {
                    sh.digit = b; sh.above_c = (uint32_t)uc; sh.above_w = uw; sh.eq_c = bc; sh.eq_w = bw;
                    break;
                }
                uc += bc;
                uw += bw;
            }
        }
    }
    __syncthreads();
}

template <int DT>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleParams p) {
    using K = KeyOf<DT>;
    using Key = typename K::Key;
    using Raw = typename K::Raw;
    constexpr int kBits = 8 * sizeof(Key);
    constexpr int kVec = 16 / sizeof(Raw);
    extern __shared__ __align__(16) unsigned char smem[];
    Key* keys = reinterpret_cast<Key*>(smem);
    __shared__ SampleShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int begin = min(rank * p.slice, p.vocab), n = min(p.vocab - begin, p.slice);

    // ---- keys of this slice, its largest one (lowest index among equals)
    const Raw* src = static_cast<const Raw*>(p.logits) + (long long)row * p.row_stride + begin;
    unsigned long long best = 0;
    const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
    const int nv = vec ? n / kVec : 0;
    for (int i = tid; i < nv; i += kSampleThreads) {
        const uint4 q = ld_stream_16(src + i * kVec);
        const uint32_t r[4] = {q.x, q.y, q.z, q.w};
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (sizeof(Raw) == 2) {
                const uint32_t a = K::key(r[j] & 0xffffu), b = K::key(r[j] >> 16);
                o[j] = a | (b << 16);
                const int at = begin + i * kVec + 2 * j;
                best = max(best, ((unsigned long long)a << 32) | (uint32_t)~at);
                best = max(best, ((unsigned long long)b << 32) | (uint32_t)~(at + 1));
            } else {
                o[j] = K::key(r[j]);
                best = max(best, ((unsigned long long)o[j] << 32) | (uint32_t)~(begin + i * kVec + j));
            }
        }
        reinterpret_cast<uint4*>(keys)[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
    for (int i = nv * kVec + tid; i < n; i += kSampleThreads) {
        const uint32_t k = K::key(src[i]);
        keys[i] = (Key)k;
        best = max(best, ((unsigned long long)k << 32) | (uint32_t)~(begin + i));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(kFullMask, best, o));
    if (lane == 0) sh.warp_w[warp] = best;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < kSampleWarps; ++i) best = max(best, sh.warp_w[i]);
        sh.best = max(best, sh.warp_w[0]);
    }
    cluster.sync();
    best = 0;
    for (int r = 0; r < C; ++r) best = max(best, *cluster.map_shared_rank(&sh.best, r));
    const uint32_t kmax = (uint32_t)(best >> 32);

    const float T = p.temperature ? p.temperature[row] : p.temperature_v;
    if (kmax == 0 || !(T > 0.f)) {                     // nothing to draw, or greedy (T <= 0, NaN)
        if (rank == 0 && tid == 0) {
            p.ids[row] = kmax == 0 ? 0 : (long long)(uint32_t)~(uint32_t)best;
            if (p.logprobs) p.logprobs[row] = kmax == 0 ? __int_as_float(0x7fc00000) : 0.f;
        }
        cluster.sync();                                // peers may still be reading sh.best
        return;
    }
    Weigher wt;
    wt.max = (double)K::value(kmax);
    wt.scale = 1.4426950408889634 / (double)T;
    wt.kmax = kmax;
    wt.two_frac = (double)(1ull << p.frac);

    // ---- where the kept prefix ends: keys above `border` stay, of those equal to it the `keep` lowest indices
    const int top_k = p.top_k ? p.top_k[row] : p.top_k_v;
    const float top_p = p.top_p ? p.top_p[row] : p.top_p_v;
    const float min_p = p.min_p ? p.min_p[row] : p.min_p_v;
    const bool by_k = top_k > 0 && top_k < p.vocab, by_p = top_p < 1.f;
    uint32_t border = 1, keep = 0xffffffffu, ties = 0;
    if (by_k || by_p) {
        int buf = 0;
        histogram<DT>(keys, n, kBits - 8, 0, wt, &sh.hist[buf], &sh.first, cluster);
        buf ^= 1;
        uint32_t drawable = 0;
        unsigned long long all = 0;
        for (int b = 0; b < 256; ++b) {
            drawable += sh.first.cnt[b];
            all += ((unsigned long long)sh.first.hi[b] << 32) | sh.first.lo[b];
        }
        unsigned long long z = all;
        for (int pass = 0; pass < 2; ++pass) {
            unsigned long long target;
            if (pass == 0) {
                if (!by_k || (uint32_t)top_k >= drawable) continue;
                target = (unsigned long long)top_k;
            } else {
                if (!by_p) continue;
                const double t = ceil((double)fmaxf(top_p, 0.f) * (double)z);
                target = t < 1.0 ? 1ull : (unsigned long long)t;
                if (target > z) target = z;
            }
            uint32_t prefix = 0, above_c = 0;
            unsigned long long above_w = 0;
            const Hist* h = &sh.first;
            for (int shift = kBits - 8;; shift -= 8) {
                find_bin(h, pass == 0, target, above_c, above_w, sh);
                prefix = (prefix << 8) | sh.digit;
                above_c = sh.above_c;
                above_w = sh.above_w;
                if (shift == 0) break;
                __syncthreads();
                histogram<DT>(keys, n, shift - 8, prefix, wt, &sh.hist[buf], &sh.merged, cluster);
                buf ^= 1;
                h = &sh.merged;
            }
            border = prefix;
            ties = sh.eq_c;
            const unsigned long long w1 = wt.fixed(K::value(border), border);
            if (pass == 0) {
                keep = (uint32_t)target - above_c;
                z = above_w + (unsigned long long)keep * w1;
            } else {
                const unsigned long long m = w1 ? (target - above_w + w1 - 1) / w1 : 1;
                keep = (uint32_t)min(m, (unsigned long long)sh.eq_c);
            }
            __syncthreads();
        }
    }
    // ---- index order from here on: warp w of the CTA owns a contiguous run of the slice
    const int run = ((n + kSampleWarps - 1) / kSampleWarps + 31) / 32 * 32;
    const int r0 = min(warp * run, n), r1 = min(r0 + run, n);
    uint32_t tie_base = 0;
    const bool ranked = keep < ties;
    if (ranked) {
        uint32_t c = 0;
        for (int i = r0 + lane; i < r1; i += 32) c += keys[i] == border;
        c = __reduce_add_sync(kFullMask, c);
        if (lane == 0) sh.warp_c[warp] = c;
        __syncthreads();
        if (tid == 0) {
            uint32_t s = 0;
            for (int i = 0; i < kSampleWarps; ++i) {
                const uint32_t x = sh.warp_c[i];
                sh.warp_c[i] = s;
                s += x;
            }
            sh.pub_ties = s;
        }
        cluster.sync();
        tie_base = sh.warp_c[warp];
        for (int r = 0; r < rank; ++r) tie_base += *cluster.map_shared_rank(&sh.pub_ties, r);
    }
    const double min_rel = (double)min_p;
    auto kept_weight = [&](uint32_t k, uint32_t rank_of_tie) -> unsigned long long {
        if (k < border || (ranked && k == border && rank_of_tie >= keep)) return 0;
        const float v = K::value(k);
        if (min_p > 0.f && k != kmax && wt.relative(v, k) < min_rel) return 0;
        return wt.fixed(v, k);
    };
    unsigned long long sum = 0;
    uint32_t seen = tie_base;
    for (int i0 = r0; i0 < r1; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t k = i < r1 ? keys[i] : 0;
        uint32_t rk = 0;
        if (ranked) {
            const unsigned eq = __ballot_sync(kFullMask, k == border);
            rk = seen + __popc(eq & ((1u << lane) - 1));
            seen += __popc(eq);
        }
        sum += kept_weight(k, rk);
    }
    sum = warp_sum_u64(sum);
    if (lane == 0) sh.warp_w[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        unsigned long long s = 0;
        for (int i = 0; i < kSampleWarps; ++i) {
            const unsigned long long x = sh.warp_w[i];
            sh.warp_w[i] = s;
            s += x;
        }
        sh.pub_w = s;
    }
    cluster.sync();
    unsigned long long base = sh.warp_w[warp], z = 0;
    for (int r = 0; r < C; ++r) {
        const unsigned long long x = *cluster.map_shared_rank(&sh.pub_w, r);
        if (r < rank) base += x;
        z += x;
    }
    const float u = fmaxf(p.uniform[row], 0.f);          // NaN: 0
    const double want = (double)u * (double)z;
    unsigned long long target = u >= 1.f ? z - 1 : (unsigned long long)want;
    if (target >= z) target = z - 1;
    if (base <= target && target < base + sum) {         // one warp of the cluster owns the draw
        seen = tie_base;
        for (int i0 = r0; i0 < r1; i0 += 32) {
            const int i = i0 + lane;
            const uint32_t k = i < r1 ? keys[i] : 0;
            uint32_t rk = 0;
            if (ranked) {
                const unsigned eq = __ballot_sync(kFullMask, k == border);
                rk = seen + __popc(eq & ((1u << lane) - 1));
                seen += __popc(eq);
            }
            const unsigned long long w = kept_weight(k, rk);
            const unsigned long long inc = base + warp_scan_u64(w, lane);
            const unsigned hit = __ballot_sync(kFullMask, inc > target);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    p.ids[row] = begin + i;
                    if (p.logprobs) p.logprobs[row] = (float)log((double)w / (double)z);
                }
                break;
            }
            base = __shfl_sync(kFullMask, inc, 31);
        }
    }
    cluster.sync();                                      // peers may still be reading this CTA's published sums
}

template <int DT>
int launch_sample(const SampleParams& p, int rows, int cluster, size_t smem, cudaStream_t st) {
    cudaError_t e = cudaFuncSetAttribute(sample_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
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
    // CTAs per row: enough to fill the 148 SMs while rows are few, and enough for the slice to fit shared memory
    int cluster = 1;
    while (cluster < 8 && (long long)a->rows * cluster * 2 <= 148) cluster *= 2;
    const int max_slice = 200 * 1024 / es;
    while (cluster < 8 && (a->vocab + cluster - 1) / cluster > max_slice) cluster *= 2;
    SampleParams p{};
    p.logits = a->logits;
    p.row_stride = a->row_stride;
    p.vocab = a->vocab;
    p.slice = ((a->vocab + cluster - 1) / cluster + 7) / 8 * 8;
    int lg = 0;
    while ((1 << lg) < a->vocab) ++lg;
    p.frac = 62 - lg < 52 ? 62 - lg : 52;
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
    const size_t smem = (size_t)p.slice * es;
    cudaStream_t st = static_cast<cudaStream_t>(a->stream);
    return a->dtype == 0 ? launch_sample<0>(p, a->rows, cluster, smem, st)
                         : (a->dtype == 1 ? launch_sample<1>(p, a->rows, cluster, smem, st)
                                          : launch_sample<2>(p, a->rows, cluster, smem, st));
}
