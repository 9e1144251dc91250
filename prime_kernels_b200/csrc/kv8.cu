// Paged KV cache held in 8 bits, and attention over it (head dim 64).
//
// Values are e4m3; every (page, kv head) has one E8M0 scale for its K and one for its V tokens: x = v8 * 2^(e - 127).
// The scale follows the round-up rule of the other quantisers of this library (2^ceil(log2(amax / 448))), so a value
// never saturates, and a scale that grows moves the values already held by a power of two.  Two layouts, the ones
// the decode step reads in bf16: [pages, kv heads, page size, 128] (K in 0..63, V in 64..127) and
// [2, pages, page size, kv heads, 64]; both are described by byte strides.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/prime_kernels_b200.h"
#include "pk_common.cuh"

namespace pk {
namespace cg = cooperative_groups;

constexpr int kHeadDim = 64;

struct Kv8Params {
    uint8_t* cache;
    uint8_t* scales;                                   // [pages, kv heads, 2]
    long long k_off, v_off, page_stride, token_stride, head_stride;     // bytes
    int pages, page_shift, kv_heads;
    const int* block_table;
    long long bt_stride;
    int bt_cols;
    const int* seq_lens;
    const int* cu;                                     // [batch + 1], null: one token per request
    int batch, tokens;
};

__device__ __forceinline__ float exp2_biased(uint32_t e) {              // 2^(e - 127), e 0..254
    return __uint_as_float(e ? (e << 23) : 0x00400000u);
}
__device__ __forceinline__ uint32_t e8m0_roundup(float x) {
    uint16_t r;
    asm("cvt.rp.satfinite.ue8m0x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(x));
    return r & 0xffu;
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// four e4m3 values to two f16x2 words; exact
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(lo), "=r"(hi) : "r"(four));
}

// request of token t (last r with cu[r] <= t) and its token range, clamped to the rows there are; false: no request
__device__ __forceinline__ bool request_of(const Kv8Params& p, int t, int& r, int& first, int& count) {
    if (!p.cu) {
        r = first = t;
        count = 1;
        return t < p.batch;
    }
    int lo = 0, hi = p.batch;                          // cu[lo] <= t < cu[hi] once found
    if (t < p.cu[0] || t >= p.cu[p.batch]) return false;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.cu[mid] <= t) lo = mid; else hi = mid;
    }
    r = lo;
    first = max(p.cu[lo], 0);
    count = min(p.cu[hi], p.tokens) - first;
    return true;
}

// ---------------------------------------------------------------- append
// One warp per (16 consecutive rows, kv head), or per (request, kv head) with one token each.  Among its rows the warp
// looks for the first new token of a page, which leads: it stores all new tokens of that page, K and V, whether or not
// they lie among the warp's rows.  16 of them are kept in registers between the maximum and the values; more (pages of 32
// slots and up) are read again, from L2.  17.4 k tokens x 32 heads out of fused projection rows, 214 MB, take 43 us on the
// device (0.76 of the measured copy bandwidth; 42 us with pages of 16 slots, 56 and 64 us with 128 and 256): bytes, and what
// a warp leaves unused of them, as it loads a page only when the one before is stored.  A warp per row, all but the leaders
// of which left at once, took 134 us.
struct AppendParams {
    Kv8Params c;
    const uint16_t *k, *v;
    long long k_token, k_head, v_token, v_head;        // elements
};

// Largest finite magnitude of bf16 values, as its 15 bits: magnitudes are ordered like their bits, two to a word.
__device__ __forceinline__ uint32_t amax_two(const uint4 q) {             // of eight, in two halves
    return __vmaxu2(__vmaxu2(q.x & 0x7fff7fffu, q.y & 0x7fff7fffu), __vmaxu2(q.z & 0x7fff7fffu, q.w & 0x7fff7fffu));
}
template <int kQ> __device__ __forceinline__ uint32_t amax_bits(const uint4 (&q)[kQ]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kQ; ++i) m = __vmaxu2(m, amax_two(q[i]));
    m = max(m & 0xffffu, m >> 16);
    if (m >= 0x7f80u) {                                // NaN and Inf do not count
        m = 0;
        for (int i = 0; i < kQ; ++i) {
            const uint32_t w[4] = {q[i].x & 0x7fff7fffu, q[i].y & 0x7fff7fffu, q[i].z & 0x7fff7fffu, q[i].w & 0x7fff7fffu};
            for (int j = 0; j < 4; ++j) {
                if ((w[j] & 0xffffu) < 0x7f80u) m = max(m, w[j] & 0xffffu);
                if ((w[j] >> 16) < 0x7f80u) m = max(m, w[j] >> 16);
            }
        }
    }
    return m;
}

__device__ __forceinline__ uint2 to_e4m3x8(const uint4 q, float inv) {
    return make_uint2(e4m3x2(bf16_lo(q.x) * inv, bf16_hi(q.x) * inv) | (e4m3x2(bf16_lo(q.y) * inv, bf16_hi(q.y) * inv) << 16),
                      e4m3x2(bf16_lo(q.z) * inv, bf16_hi(q.z) * inv) | (e4m3x2(bf16_lo(q.w) * inv, bf16_hi(q.w) * inv) << 16));
}
// The tokens of a page that are held already, after its scale grew: times f, a power of two.
__device__ void rescale_page(uint8_t* dst, long long token_stride, int slots, float f, int lane) {
    for (int i = lane >> 2; i < slots; i += 8) {
        uint4* q = reinterpret_cast<uint4*>(dst + (long long)i * token_stride + (lane & 3) * 16);
        uint4 a = *q;
        uint32_t* w = reinterpret_cast<uint32_t*>(&a);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t lo, hi;
            e4m3x4_to_f16(w[j], lo, hi);
            const float2 fl = __half22float2(*reinterpret_cast<const __half2*>(&lo));
            const float2 fh = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            w[j] = e4m3x2(fl.x * f, fl.y * f) | (e4m3x2(fh.x * f, fh.y * f) << 16);
        }
        *q = a;
    }
}

template <int kGroup>
__global__ void __launch_bounds__(256, kGroup == 1 ? 2 : 3) kv8_append_kernel(AppendParams p) {
    const Kv8Params& c = p.c;
    const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const long long group = item / c.kv_heads;
    const int h = (int)(item - group * c.kv_heads), size = 1 << c.page_shift;
    if (group * kGroup >= c.tokens) return;
    // ---- lane i looks at row i of the group
    const int mine = (int)group * kGroup + lane;
    int slot = 0, m = 0, page = -1;
    if (lane < kGroup && mine < c.tokens) {
        int r, first, count;
        if (request_of(c, mine, r, first, count)) {
            const long long pos = (long long)c.seq_lens[r] - count + (mine - first);
            slot = (int)(pos & (size - 1));
            if (pos >= 0 && (slot == 0 || mine == first) && (pos >> c.page_shift) < c.bt_cols) {
                page = c.block_table[r * c.bt_stride + (pos >> c.page_shift)];
                m = min(size - slot, first + count - mine);
                if (page >= c.pages) page = -1;
            }
        }
    }
    for (unsigned leaders = __ballot_sync(kFullMask, page >= 0); leaders; leaders &= leaders - 1) {
        const int who = __ffs(leaders) - 1;
        const int t = (int)group * kGroup + who, s = __shfl_sync(kFullMask, slot, who), n = __shfl_sync(kFullMask, m, who);
        const long long pg = __shfl_sync(kFullMask, page, who);
        uint8_t* base = c.cache + pg * c.page_stride + (long long)h * c.head_stride;
        uint8_t* scale = c.scales + (pg * c.kv_heads + h) * 2;
        const uint16_t* k = p.k + (long long)t * p.k_token + (long long)h * p.k_head + (lane & 7) * 8;
        const uint16_t* v = p.v + (long long)t * p.v_token + (long long)h * p.v_head + (lane & 7) * 8;
        const int row = lane >> 3;                                           // of every four
        constexpr int kQ = kGroup == 1 ? 1 : 4;                              // 16 tokens, a quarter of them a lane; or one
        uint4 kq[kQ], vq[kQ];
        auto load = [&](int from) {
            const uint16_t *ka = k + (from + row) * p.k_token, *va = v + (from + row) * p.v_token;
#pragma unroll
            for (int i = 0; i < kQ; ++i, ka += 4 * p.k_token, va += 4 * p.v_token) {
                const bool on = from + row + 4 * i < n;
                kq[i] = on ? *reinterpret_cast<const uint4*>(ka) : make_uint4(0, 0, 0, 0);
                vq[i] = on ? *reinterpret_cast<const uint4*>(va) : make_uint4(0, 0, 0, 0);
            }
        };
        uint32_t ka = 0, va = 0;
        const int last = (n - 1) & ~15;
        for (int from = 0; from <= last; from += 16) {
            load(from);
            ka = max(ka, amax_bits(kq));
            va = max(va, amax_bits(vq));
        }
        auto scale_of = [](uint32_t bits) { return e8m0_roundup(__fmul_rn(__uint_as_float(__reduce_max_sync(kFullMask, bits) << 16), 1.f / 448.f)); };
        uint32_t ek = scale_of(ka), ev = scale_of(va);
        if (s) {                                                             // tokens are held: the scale may only grow
            const uint32_t ok = min((uint32_t)scale[0], 254u), ov = min((uint32_t)scale[1], 254u);
            if (ek > ok) rescale_page(base + c.k_off, c.token_stride, s, exp2_biased(127u - min(ek - ok, 126u)), lane);
            if (ev > ov) rescale_page(base + c.v_off, c.token_stride, s, exp2_biased(127u - min(ev - ov, 126u)), lane);
            ek = max(ek, ok);
            ev = max(ev, ov);
            __syncwarp();                                                    // the old scales have been read
        }
        const float ki = exp2_biased(254u - ek), vi = exp2_biased(254u - ev);
        uint8_t* to = base + (long long)s * c.token_stride + (lane & 7) * 8;
        for (int from = last; from >= 0; from -= 16) {                       // the last 16 are still in registers
            if (from != last) load(from);
            uint8_t* at = to + (from + row) * c.token_stride;
#pragma unroll
            for (int i = 0; i < kQ; ++i, at += 4 * c.token_stride)
                if (from + row + 4 * i < n) {
                    *reinterpret_cast<uint2*>(at + c.k_off) = to_e4m3x8(kq[i], ki);
                    *reinterpret_cast<uint2*>(at + c.v_off) = to_e4m3x8(vq[i], vi);
                }
        }
        if (lane == 0) *reinterpret_cast<uint16_t*>(scale) = (uint16_t)(ek | (ev << 8));
    }
}

// ---------------------------------------------------------------- attention
// Rows of one (request, kv head): (token, query head of the group), row = token * G + head; tiles of 8 or 16 rows.  A
// tile's keys are dealt to the CTAs of a cluster and, in steps of 32 keys, to the warps of a CTA; every warp keeps a
// running softmax of its own (one pass over the cache), merged at the end in shared memory and then through
// distributed shared memory.  Products run on m16n8k16 f16 with fp32 accumulation: e4m3 converts to f16 exactly, and
// q is divided by a power of two per row so that its bf16 bits fit f16 (elements 2^-22 below the row's largest lose
// bits).  The cache reaches the operand registers by way of a ring of its own for every warp (asynchronous 16-byte
// copies, no barrier but the warp's): a lane's 16 bytes of a K row are its dims of all four k-steps, and pairs of V rows
// are interleaved by byte permutation.
//
// V scales differ from page to page, so weights enter the second product as 2^(s + eV - top) with a running maximum
// `top` of s + eV of their own, apart from the running maximum of s that the sum uses: a page's scale can neither overflow
// them nor push all of them below f16.  What they lose: a weight is off by 2^-11 of itself or by 2^-25 of the row's largest
// product of weight and V scale, whichever is more, which is below the rounding of a bf16 output unless the heavier tokens
// hold next to nothing in a dim.  So with equal scores a page keeps its full precision in every dim down to a V scale
// of 2^-13 of the largest, loses bits below that, and from 2^-25 on adds nothing.  (bf16 would reach further with 2^-9 of
// each weight; weights apart from scales would take an accumulator for each page.)  Sums and maxima are fp32, exponentials
// ex2.approx (2^-22).
//
// A key that only later tokens of a tile see has weight 0 for the others, and 0 * NaN is NaN: where rows of a tile differ
// in what they see, NaN among the V values is taken for 0 in the product and put into the rows that see it at the end
// (the prompt kernel computes rows that it spoiled once more).
//
// Bound by the bytes of the cache where there are many and lengths are alike, by the longest item where they differ (the
// split is one number for a launch), by the chain of dependent reads at the start (length, page, page's data) and the
// merge where there are few.  64 requests of 2144 to 8192 tokens, 15/5 heads: 45 us on the device, 4.7 TB/s, 0.72 of the
// measured copy bandwidth; one CTA an item, the longest of which has 1.47 times the mean place's keys.  Steps of 16 keys read ahead in registers took 60 us (295 instructions a step, two thirds of
// them not products), with a ring 52 us; 32 keys share the page lookups, maxima and rescaling (only where a maximum
// moved).
struct AttendParams {
    Kv8Params c;
    const uint16_t* q;
    long long q_token, q_head;                         // elements
    uint16_t* out;
    long long o_token, o_head;
    float* lse;                                        // [tokens, q heads] or null
    int q_heads, group, tiles;
    unsigned wait_limit;                               // polls of a wait of the prompt kernel
    float scale;                                       // softmax scale * log2(e)
};

constexpr int kAttWarps = 8;
constexpr int kKeyRow = 64, kValueRow = 80;            // bytes: free of bank conflicts as the lanes read them
constexpr int kStageBytes = 32 * (kKeyRow + kValueRow), kStages = 2;
constexpr float kNegInf = -__builtin_huge_valf();

struct __align__(16) AttendShared {
    float o[16][kHeadDim + 4];
    float m[16], top[16], l[16];                       // running maxima (log2) and sum
    int nan_seen;
};

static_assert(sizeof(AttendShared) <= kStages * kStageBytes, "the merge reuses the rings");
constexpr int kAttShared = kAttWarps * kStages * kStageBytes;

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool valid) {
    const uint32_t n = valid ? 16u : 0u;               // 0: the 16 bytes are zero-filled
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// two fp32 operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\n"
        "fma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// NaN of e4m3 (0x7f, 0xff) among four values: 0x80 in each such byte
__device__ __forceinline__ uint32_t e4m3_nan(uint32_t four) { return ((four & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// the four values with 0 for NaN; `seen` collects
__device__ __forceinline__ uint32_t without_nan(uint32_t four, uint32_t& seen) {
    const uint32_t nan = e4m3_nan(four);
    seen |= nan;
    return four & ~((nan >> 7) * 0xffu);
}
// Output dims of a row that are NaN because a V value among the keys from..len - 1, all of which it sees, is: dims
// d0..d0 + n - 1 of `to`.
__device__ __noinline__ void put_nan(const Kv8Params& c, const int* table, int h, int from, int len, uint16_t* to, int d0, int n) {
    for (int key = from; key < len; ++key) {
        const int page = table[key >> c.page_shift];
        if (page < 0 || page >= c.pages) continue;
        const uint8_t* v = c.cache + (long long)page * c.page_stride + (long long)h * c.head_stride + c.v_off +
                           (long long)(key & ((1 << c.page_shift) - 1)) * c.token_stride;
        for (int d = d0; d < d0 + n; ++d)
            if ((v[d] & 0x7f) == 0x7f) to[d] = 0x7fff;
    }
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(kFullMask, v, 1));
    return fmaxf(v, __shfl_xor_sync(kFullMask, v, 2));
}

// 2^x / l in two factors, f and g: x is the exponent of the largest weight, -127 where all V of a row lie in pages of the
// lowest scale, and 2^-127 alone would come out 0.  g is 1 but for those.
__device__ __forceinline__ float unscale(float x, float l, float& g) {
    const bool low = x < -96.f;
    g = low ? exp2_biased(127 - 96) : 1.f;
    return ex2(low ? x + 96.f : x) / l;
}

// 16 dims (16t .. 16t + 15) of one q row as eight f16x2 registers, divided by 2^ex so that the largest |q| of the row
// lies in [2^7, 2^8); ex is returned.  All four lanes of the row's quad take part.
__device__ __forceinline__ int load_q(const uint16_t* row, int t, uint32_t (&f)[8]) {
    uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (row) {
        const uint4 a = *reinterpret_cast<const uint4*>(row + 16 * t), b = *reinterpret_cast<const uint4*>(row + 16 * t + 8);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(w[i])), fabsf(bf16_hi(w[i]))));
    amax = quad_max(amax);
    const int biased = (int)(__float_as_uint(amax) >> 23);
    int ex = biased - 134;                             // 2^(biased - 127) -> 2^7
    ex = max(min(ex, 126), -126);
    const float f2 = exp2_biased(127 - ex);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = pack_f16x2(bf16_lo(w[i]) * f2, bf16_hi(w[i]) * f2);
    return ex;
}

// The running softmaxes of n parts, `kPer` dims of one row, in the order of the parts.
template <int kPer> struct Merged {
    float m, top, l, acc[kPer];
    template <typename F> __device__ __forceinline__ void take(int n, int row, int d0, F&& part) {
        m = top = kNegInf;
        l = 0.f;
        for (int i = 0; i < n; ++i) {
            m = fmaxf(m, part(i)->m[row]);
            top = fmaxf(top, part(i)->top[row]);
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
        for (int i = 0; i < n; ++i) {
            const AttendShared* x = part(i);
            if (x->l[row] == 0.f) continue;
            l += x->l[row] * ex2(x->m[row] - m);
            const float f = ex2(x->top[row] - top);
#pragma unroll
            for (int k = 0; k < kPer; ++k) acc[k] += x->o[row][d0 + k] * f;
        }
    }
};

// kHalf: tiles of 8 rows (a decode step of up to 8 query heads per kv head): the lower half of the 16-row operand is
// empty and its softmax is left out.
template <bool kHalf>
__global__ void __launch_bounds__(kAttWarps * 32, 16 / kAttWarps) kv8_attend_kernel(const __grid_constant__ AttendParams p) {
    constexpr int kRows = kHalf ? 8 : 16, kR = kHalf ? 1 : 2;              // rows of a tile, of a lane
    const Kv8Params& c = p.c;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    extern __shared__ __align__(128) unsigned char smem[];
    AttendShared* sh = reinterpret_cast<AttendShared*>(smem);              // after the loop, over the rings
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int h = blockIdx.y, r = blockIdx.z;
    int first = r, count = 1;
    if (c.cu) {
        first = max(c.cu[r], 0);
        count = min(c.cu[r + 1], c.tokens) - first;
    }
    const int rows = count * p.group;
    const int seq = max(c.seq_lens[r], 0);
    const long long capacity = (long long)c.bt_cols << c.page_shift;
    const int* table = c.block_table + r * c.bt_stride;
    for (int tile = blockIdx.x / C; tile * kRows < rows; tile += p.tiles) {
        // ---- keys: steps of 32 keys, a contiguous share per CTA, dealt to its warps
        const int last = (min(tile * kRows + kRows, rows) - 1) / p.group, lead = tile * kRows / p.group;
        const int len_max = (int)min((long long)max(seq - count + last + 1, 0), capacity);
        const int len_min = (int)min((long long)max(seq - count + lead + 1, 0), capacity);
        const int steps = (len_max + 31) / 32, share = (steps + C - 1) / C;
        const int s_end = min((rank + 1) * share, steps);
        // the pages of the halves of this warp's next 16 steps and their scales, one half per lane; kStages - 1 steps are
        // on their way to shared memory while one is used
        int pages = -1, old_pages = -1;
        uint32_t scale2 = 0, old_scale2 = 0;                                 // E8M0 of K, of V
        unsigned char* ring = smem + warp * kStages * kStageBytes;
        long long lane_off = (lane >> 2) * c.token_stride + 16 * (lane & 3);
        const uint8_t* k_lane = c.cache + (long long)h * c.head_stride + c.k_off + lane_off;
        const long long v_from_k = c.v_off - c.k_off, eight = 8 * c.token_stride;
        unsigned char* to_k = ring + (lane >> 2) * kKeyRow + 16 * (lane & 3);
        unsigned char* to_v = ring + 32 * kKeyRow + (lane >> 2) * kValueRow + 16 * (lane & 3);
        auto fetch = [&](int i) {                                            // this warp's i-th step
            const int s = rank * share + warp + i * kAttWarps;
            if ((i & 15) == 0) {
                const int unit = 2 * (s + (lane >> 1) * kAttWarps) + (lane & 1);
                old_pages = pages;
                old_scale2 = scale2;
                pages = unit < 2 * s_end && unit * 16 < len_max ? table[(unit * 16) >> c.page_shift] : -1;
                if (pages >= c.pages || pages < 0) pages = -1;
                scale2 = pages < 0 ? 0u : *reinterpret_cast<const uint16_t*>(c.scales + ((long long)pages * c.kv_heads + h) * 2);
            }
            const int page0 = __shfl_sync(kFullMask, pages, 2 * (i & 15)), page1 = __shfl_sync(kFullMask, pages, 2 * (i & 15) + 1);
            if (s < s_end) {
                const int at = (i % kStages) * kStageBytes;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int page = u ? page1 : page0, key0 = s * 32 + u * 16, left = page < 0 ? 0 : len_max - key0;
                    const uint8_t* from = k_lane + (long long)max(page, 0) * c.page_stride +
                                          (long long)(key0 & ((1 << c.page_shift) - 1)) * c.token_stride;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const bool on = (lane >> 2) + 8 * j < left;
                        const uint8_t* src = on ? from + (j ? eight : 0) : k_lane - lane_off;
                        cp_async16(to_k + at + (16 * u + 8 * j) * kKeyRow, src, on);
                        cp_async16(to_v + at + (16 * u + 8 * j) * kValueRow, src + v_from_k, on);
                    }
                }
            }
            cp_async_commit();
        };
#pragma unroll 1
        for (int i = 0; i < kStages - 1; ++i) fetch(i);
        // ---- the rows of this lane
        int len[kR], ex[kR];
        uint32_t qa[2][8] = {};
#pragma unroll
        for (int i = 0; i < kR; ++i) {
            const int row = tile * kRows + g + 8 * i;
            const int tok = row / p.group;
            const bool on = row < rows;
            len[i] = on ? (int)min((long long)max(seq - count + tok + 1, 0), capacity) : len_max;
            ex[i] = load_q(on ? p.q + (long long)(first + tok) * p.q_token + (long long)(h * p.group + row - tok * p.group) * p.q_head
                              : nullptr, t, qa[i]);
        }
        float qs[kR];
#pragma unroll
        for (int i = 0; i < kR; ++i) qs[i] = p.scale * exp2_biased(127 + ex[i]);
        float o[8][4], m[kR], top[kR], l[kR];
        uint32_t nan_seen = 0;
#pragma unroll
        for (int i = 0; i < kR; ++i) {
            m[i] = top[i] = kNegInf;
            l[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        for (int i = 0, st = rank * share + warp; st < s_end; ++i, st += kAttWarps) {
            __syncwarp();                                                    // the stage that is refilled has been read
            fetch(i + kStages - 1);
            // the step's scales; the lanes may already hold the next 16 steps
            const bool older = ((i + kStages - 1) & ~15) != (i & ~15);
            const int mine_pages = older ? old_pages : pages;
            const uint32_t mine_scale2 = older ? old_scale2 : scale2;
            const bool valid[2] = {__shfl_sync(kFullMask, mine_pages, 2 * (i & 15)) >= 0,
                                   __shfl_sync(kFullMask, mine_pages, 2 * (i & 15) + 1) >= 0};
            const uint32_t sc[2] = {__shfl_sync(kFullMask, mine_scale2, 2 * (i & 15)),
                                    __shfl_sync(kFullMask, mine_scale2, 2 * (i & 15) + 1)};
            cp_async_wait<kStages - 1>();
            __syncwarp();
            const unsigned char* from = ring + (i % kStages) * kStageBytes;
            float s[4][4] = {};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint4 kw = *reinterpret_cast<const uint4*>(from + (g + 8 * j) * kKeyRow + 16 * t);
                const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t lo, hi;
                    e4m3x4_to_f16(w[k], lo, hi);
                    mma_f16(s[j], qa[0][2 * k], qa[1][2 * k], qa[0][2 * k + 1], qa[1][2 * k + 1], lo, hi);
                }
            }
            const bool edge = st * 32 + 32 > len_min || !valid[0] || !valid[1];
            const float ev[2] = {(float)(int)(sc[0] >> 8) - 127.f, (float)(int)(sc[1] >> 8) - 127.f};
            const float ks[2] = {exp2_biased(sc[0] & 0xffu), exp2_biased(sc[1] & 0xffu)};
            float pw[4][4] = {}, turn[kR];
            bool turned = false;
#pragma unroll
            for (int i2 = 0; i2 < kR; ++i2) {
                float mx[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float f0 = ks[u] * qs[i2];
#pragma unroll
                    for (int j = 2 * u; j < 2 * u + 2; ++j)
#pragma unroll
                        for (int k = 2 * i2; k < 2 * i2 + 2; ++k) s[j][k] *= f0;
                    if (edge) {
                        const int limit = valid[u] ? len[i2] - st * 32 - 2 * t : 0;      // keys from here on are masked
#pragma unroll
                        for (int j = 2 * u; j < 2 * u + 2; ++j)
#pragma unroll
                            for (int k = 0; k < 2; ++k)
                                if (8 * j + k >= limit || !valid[u]) s[j][2 * i2 + k] = kNegInf;
                    }
                    mx[u] = quad_max(fmaxf(fmaxf(s[2 * u][2 * i2], s[2 * u][2 * i2 + 1]), fmaxf(s[2 * u + 1][2 * i2], s[2 * u + 1][2 * i2 + 1])));
                }
                const float m1 = fmaxf(m[i2], fmaxf(mx[0], mx[1])), t1 = fmaxf(top[i2], fmaxf(mx[0] + ev[0], mx[1] + ev[1]));
                const float mu = m1 == kNegInf ? 0.f : m1, tu = t1 == kNegInf ? 0.f : t1;
                l[i2] *= ex2(m[i2] - mu);
                turn[i2] = ex2(top[i2] - tu);
                turned |= t1 > top[i2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float f = ex2(fminf(mu + ev[u] - tu, 127.f));      // 2^(s - m) -> 2^(s + ev - top)
#pragma unroll
                    for (int j = 2 * u; j < 2 * u + 2; ++j)
#pragma unroll
                        for (int k = 2 * i2; k < 2 * i2 + 2; ++k) {
                            const float e = ex2(s[j][k] - mu);
                            l[i2] += e;
                            pw[j][k] = e * f;
                        }
                }
                m[i2] = m1;
                top[i2] = t1;
            }
            if (__any_sync(kFullMask, turned)) {
#pragma unroll
                for (int d = 0; d < 8; ++d)
#pragma unroll
                    for (int i2 = 0; i2 < kR; ++i2) {
                        o[d][2 * i2] *= turn[i2];
                        o[d][2 * i2 + 1] *= turn[i2];
                    }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint2 vw[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    vw[j] = *reinterpret_cast<const uint2*>(from + 32 * kKeyRow + (16 * u + 2 * t + (j & 1) + 8 * (j >> 1)) * kValueRow + 8 * g);
                if (st * 32 + 32 > len_min && len_min < len_max) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) vw[j] = make_uint2(without_nan(vw[j].x, nan_seen), without_nan(vw[j].y, nan_seen));
                }
                const uint32_t a0 = pack_f16x2(pw[2 * u][0], pw[2 * u][1]), a1 = kHalf ? 0u : pack_f16x2(pw[2 * u][2], pw[2 * u][3]);
                const uint32_t a2 = pack_f16x2(pw[2 * u + 1][0], pw[2 * u + 1][1]),
                               a3 = kHalf ? 0u : pack_f16x2(pw[2 * u + 1][2], pw[2 * u + 1][3]);
#pragma unroll
                for (int d = 0; d < 4; ++d) {                                // dims 8g + 2d, 8g + 2d + 1
                    const uint32_t sel = (d & 1) ? 0x7362u : 0x5140u;
                    const uint32_t lo = __byte_perm(d < 2 ? vw[0].x : vw[0].y, d < 2 ? vw[1].x : vw[1].y, sel);
                    const uint32_t hi = __byte_perm(d < 2 ? vw[2].x : vw[2].y, d < 2 ? vw[3].x : vw[3].y, sel);
                    uint32_t b00, b01, b10, b11;
                    e4m3x4_to_f16(lo, b00, b10);
                    e4m3x4_to_f16(hi, b01, b11);
                    mma_f16(o[2 * d], a0, a1, a2, a3, b00, b01);
                    mma_f16(o[2 * d + 1], a0, a1, a2, a3, b10, b11);
                }
            }
        }
        // ---- merge the warps, then the CTAs
        cp_async_wait<0>();
        __syncthreads();                                                     // the rings are read: their memory is the merge's now
#pragma unroll
        for (int i = 0; i < kR; ++i) {
            l[i] += __shfl_xor_sync(kFullMask, l[i], 1);
            l[i] += __shfl_xor_sync(kFullMask, l[i], 2);
            const int row = g + 8 * i;
            if (t == 0) {
                sh[warp].m[row] = m[i];
                sh[warp].top[row] = top[i];
                sh[warp].l[row] = l[i];
            }
#pragma unroll
            for (int d = 0; d < 8; ++d) {                                    // columns 2t, 2t + 1 of tile d: dims 16t + d, 16t + 8 + d
                sh[warp].o[row][16 * t + d] = o[d][2 * i];
                sh[warp].o[row][16 * t + 8 + d] = o[d][2 * i + 1];
            }
        }
        bool nan_v = __syncthreads_or((int)nan_seen);
        constexpr int kPer = kRows * kHeadDim / (kAttWarps * 32);            // dims of one row that a thread merges: 2, 4 or 8
        const int row = (int)threadIdx.x / (kHeadDim / kPer), d0 = (int)threadIdx.x % (kHeadDim / kPer) * kPer;
        Merged<kPer> a;
        a.take(kAttWarps, row, d0, [&](int i) { return &sh[i]; });
        if (C > 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kPer; ++k) sh[0].o[row][d0 + k] = a.acc[k];
            if (d0 == 0) {
                sh[0].m[row] = a.m;
                sh[0].top[row] = a.top;
                sh[0].l[row] = a.l;
            }
            if (threadIdx.x == 0) sh[0].nan_seen = nan_v;
            cluster.sync();
            if (rank == 0) {
                a.take(C, row, d0, [&](int i) { return cluster.map_shared_rank(&sh[0], i); });
                if (len_min < len_max)
                    for (int i = 0; i < C; ++i) nan_v |= cluster.map_shared_rank(&sh[0], i)->nan_seen != 0;
            }
        }
        const int at = tile * kRows + row;
        if (rank == 0 && at < rows) {
            const int tok = at / p.group, head = h * p.group + at - tok * p.group;
            float g = 1.f;
            const float f = a.l == 0.f ? 0.f : unscale(a.top - a.m, a.l, g);
            uint32_t* to = reinterpret_cast<uint32_t*>(p.out + (long long)(first + tok) * p.o_token + (long long)head * p.o_head + d0);
#pragma unroll
            for (int k = 0; k < kPer; k += 2) to[k / 2] = pack_bf16x2(a.acc[k] * f * g, a.acc[k + 1] * f * g);
            if (__builtin_expect(nan_v, 0))
                put_nan(c, table, h, len_min & ~31, (int)min((long long)max(seq - count + tok + 1, 0), capacity),
                        p.out + (long long)(first + tok) * p.o_token + (long long)head * p.o_head, d0, kPer);
            if (p.lse && d0 == 0)
                p.lse[(long long)(first + tok) * p.q_heads + head] = a.l == 0.f ? kNegInf : (a.m + log2f(a.l)) * 0.6931471805599453f;
        }
        if (C > 1) cluster.sync(); else __syncthreads();                     // the parts are read before they are written again
    }
}

// ---------------------------------------------------------------- attention of many query tokens (prompt chunks)
// The same rows and the same arithmetic with 128 rows a tile, on tcgen05: S = Q K^T (M 128, N 64, both operands K-major
// in shared memory) and O += P V (P from tensor memory, V as it lies: [key][dim], MN-major), accumulators in tensor
// memory.  One CTA holds one tile; warps 0-3 own a row a thread (softmax), warps 4-7 turn e4m3 pages into swizzled f16
// tiles of 64 keys, and a thread of warp 7 issues the products: eight warps, two on each scheduler, 128 registers a thread.
// (Two warps with all of the pages made the softmax warps beside them the slowest; sparing warp 7 its share made the other
// three so: 259, 263 and 269 us where this took 252.)  S is double-buffered, so the next scores are computed
// while the softmax works, and two CTAs share an SM (256 columns of tensor memory each), so one's products run under
// the other's exponentials.
//
// The exponentials are the floor (16 a clock and SM against 64 x 4 flops each, a quarter of the tensor peak at head dim 64:
// 81 us for four chunks of up to 2048 tokens behind up to 6144, 15/5 heads).  Bound by the chain of a step, scores ->
// maximum -> exponentials -> weights, with two CTAs on an SM to hide it: 246 us on the device there, 2750 clocks a step at
// 1965 MHz for the place with most of them (176, the mean is 153); no unit is busy.  96 bytes of registers are spilled.
// `top` is raised only where a row's maximum has grown by 2^8, so that the accumulator is rarely rescaled; f16 holds 2^8
// times the weights.
constexpr int kTileRows = 128, kTileKeys = 64, kPromptStages = 4;
constexpr int kRawStages = 3, kRawBytes = kTileKeys * 128;              // e4m3 on its way
constexpr int kPromptThreads = 256, kProducers = 128;
constexpr uint32_t kPromptCols = 256, kColP = 128, kColO = 192;            // S in columns 0..127, P in 128..191, two of each
constexpr float kLazy = 8.f;
constexpr unsigned kWaitLimit = 1u << 20;

struct PromptShared {
    uint64_t full[kPromptStages], empty[kPromptStages], q_full, s_full[2], p_full[2], pv_done[2], drain;
    __align__(16) float ks[kPromptStages][4], ev[kPromptStages][4], bias[kPromptStages][4];   // per 16 keys; bias -inf: no page
    uint32_t tmem;
    volatile int abort, nan_out;                       // nan_out: an output was NaN
};
constexpr int kPromptBytes = kTileRows * 128 + kPromptStages * 2 * kTileKeys * 128 + kRawStages * kRawBytes + (int)sizeof(PromptShared);

__device__ unsigned int g_kv8_wait_timeouts;

// Bounded waits: false once `limit` polls are over, or as soon as another thread of the CTA has given up.
// Whoever gets false touches nothing that the wait guards and leaves its loop: the parts that depend on it run out in turn,
// the softmax warps agree on it at the end of the tile, and their rows become NaN.
__device__ __forceinline__ void gave_up(PromptShared& sh) {
    if (!sh.abort) {
        sh.abort = 1;
        atomicAdd(&g_kv8_wait_timeouts, 1u);
    }
}
__device__ __forceinline__ bool prompt_poll(PromptShared& sh, uint64_t* bar, uint32_t parity, unsigned limit) {
    for (uint32_t n = 0; n < limit; ++n) {
        if (mbar_test(bar, parity & 1u)) return true;
        if ((n & 63) == 63 && sh.abort) return false;
    }
    gave_up(sh);
    return false;
}
__device__ __forceinline__ bool prompt_wait(PromptShared& sh, uint64_t* bar, uint32_t parity, unsigned limit) {
    return __builtin_expect(mbar_test(bar, parity & 1u), 1) || prompt_poll(sh, bar, parity, limit);
}
// The same for a whole warp whose next instruction is a warp-wide one: lanes may leave the polling loop apart.
__device__ __forceinline__ bool warp_wait(PromptShared& sh, uint64_t* bar, uint32_t parity, unsigned limit) {
    return __all_sync(kFullMask, prompt_wait(sh, bar, parity, limit));
}
__device__ __forceinline__ bool any_of_softmax(bool mine) {                 // of the 128 threads of warps 0-3
    uint32_t r;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbarrier.cta.red.or.pred q, 1, 128, p;\nselp.u32 %0, 1, 0, q;\n}"
                 : "=r"(r) : "r"((uint32_t)mine) : "memory");
    return r != 0;
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 128-byte swizzle, rows of 128 bytes, 1024 bytes from one group of eight rows to the next, descriptor version 1; the same
// for a K-major operand (row = M or N index) and an MN-major one of 64 elements (row = K index)
__device__ __forceinline__ uint64_t tile_desc(const void* p) {
    return (((uint64_t)smem_u32(p) >> 4) & 0x3fffull) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// f16 x f16 -> f32, M 128, N 64; bit 16: B is MN-major
constexpr uint32_t kIdescQK = (1u << 4) | ((uint32_t)(kTileKeys >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
constexpr uint32_t kIdescPV = (1u << 4) | (1u << 16) | ((uint32_t)(kHeadDim >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t at, float* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const float* v) {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(v);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
        ::"r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
        "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]),
        "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]),
        "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31]), "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* u) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        ::"r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
        "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Rows that are NaN because a V value of a key they do not see is (weight 0 times NaN): those dims once more, one row a
// thread and without the products of the tensor cores, which takes milliseconds.  Everything is read anew, so that the
// loop keeps nothing in registers for it; 0 in place of NaN on the way to the tiles made every
// call 3 % slower.
__device__ __noinline__ void rows_apart(const AttendParams& p) {
    const Kv8Params& c = p.c;
    const int h = blockIdx.y, r = blockIdx.z, first = c.cu ? max(c.cu[r], 0) : r;
    const int count = c.cu ? min(c.cu[r + 1], c.tokens) - first : 1, rows = count * p.group, seq = max(c.seq_lens[r], 0);
    const long long capacity = (long long)c.bt_cols << c.page_shift;
    const int* table = c.block_table + r * c.bt_stride;
    auto at = [&](int key, int& page) -> const uint8_t* {                  // K of a key, null: no page
        page = table[key >> c.page_shift];
        if (page < 0 || page >= c.pages) return nullptr;
        return c.cache + (long long)page * c.page_stride + (long long)h * c.head_stride + c.k_off +
               (long long)(key & ((1 << c.page_shift) - 1)) * c.token_stride;
    };
    auto value = [](uint8_t b) {
        uint32_t lo, hi;
        e4m3x4_to_f16(b, lo, hi);
        return __half2float(__low2half(*reinterpret_cast<const __half2*>(&lo)));
    };
    for (int tile = p.tiles - 1 - (int)blockIdx.x; tile * kTileRows < rows; tile += p.tiles) {
        const int row = tile * kTileRows + (int)threadIdx.x, tok = row / p.group, last = (min(tile * kTileRows + kTileRows, rows) - 1) / p.group;
        if (row >= rows) break;
        const int len = (int)min((long long)max(seq - count + tok + 1, 0), capacity);
        const int len_max = (int)min((long long)max(seq - count + last + 1, 0), capacity);
        const int head = h * p.group + row - tok * p.group;
        unsigned long long dims = 0;
#pragma unroll 1
        for (int key = len, page; key < len_max; ++key)
            if (const uint8_t* k = at(key, page))
#pragma unroll 1
                for (int d = 0; d < kHeadDim; ++d) dims |= (unsigned long long)((k[c.v_off - c.k_off + d] & 0x7f) == 0x7f) << d;
        if (!dims) continue;
        const uint16_t* q = p.q + (long long)(first + tok) * p.q_token + (long long)head * p.q_head;
        float m = kNegInf;
        double l = 0., acc[kHeadDim];
#pragma unroll 1
        for (int d = 0; d < kHeadDim; ++d) acc[d] = 0.;
#pragma unroll 1
        for (int key = 0, page; key < len; ++key) {
            const uint8_t* k = at(key, page);
            if (!k) continue;
            const uint8_t* scales = c.scales + ((long long)page * c.kv_heads + h) * 2;
            double dot = 0.;
#pragma unroll 1
            for (int d = 0; d < kHeadDim; ++d) dot += (double)__uint_as_float((uint32_t)q[d] << 16) * value(k[d]);
            const float x = (float)(dot * p.scale * exp2_biased(scales[0])), m1 = fmaxf(m, x);
            const double turn = m == m1 ? 1. : exp2((double)m - m1), w = x == kNegInf ? 0. : exp2((double)x - m1), ev = w * exp2((double)scales[1] - 127.);
            m = m1;
            l = l * turn + w;
#pragma unroll 1
            for (int d = 0; d < kHeadDim; ++d)
                if (dims >> d & 1) acc[d] = acc[d] * turn + ev * value(k[c.v_off - c.k_off + d]);
        }
        uint16_t* to = p.out + (long long)(first + tok) * p.o_token + (long long)head * p.o_head;
#pragma unroll 1
        for (int d = 0; d < kHeadDim; ++d)
            if (dims >> d & 1) to[d] = (uint16_t)pack_bf16x2(l == 0. ? 0.f : (float)(acc[d] / l), 0.f);
    }
}

// The CTA gave up a wait in this tile: its rows, and those of the tiles it would have taken after it.
__device__ __noinline__ void rows_given_up(const AttendParams& p, int tile) {
    const Kv8Params& c = p.c;
    const int h = blockIdx.y, r = blockIdx.z, first = c.cu ? max(c.cu[r], 0) : r;
    const int rows = (c.cu ? min(c.cu[r + 1], c.tokens) - first : 1) * p.group;
    for (; tile * kTileRows < rows; tile += p.tiles) {
        const int row = tile * kTileRows + (int)threadIdx.x, tok = row / p.group, head = h * p.group + row - tok * p.group;
        if (row >= rows) break;
        uint4* to = reinterpret_cast<uint4*>(p.out + (long long)(first + tok) * p.o_token + (long long)head * p.o_head);
        for (int i = 0; i < 8; ++i) to[i] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
        if (p.lse) p.lse[(long long)(first + tok) * p.q_heads + head] = __int_as_float(0x7fffffff);
    }
}

__global__ void __launch_bounds__(kPromptThreads, 2) kv8_prompt_kernel(const __grid_constant__ AttendParams p) {
    const Kv8Params& c = p.c;
    // aligned by its declaration: addresses known when it is compiled take no registers (260 us with a base rounded up)
    extern __shared__ __align__(1024) unsigned char q_tile[];
    unsigned char* kv_tiles = q_tile + kTileRows * 128;                    // per stage: K, V
    unsigned char* raw_ring = kv_tiles + kPromptStages * 2 * kTileKeys * 128;
    PromptShared& sh = *reinterpret_cast<PromptShared*>(raw_ring + kRawStages * kRawBytes);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.y, r = blockIdx.z;
    int first = r, count = 1;
    if (c.cu) {
        first = max(c.cu[r], 0);
        count = min(c.cu[r + 1], c.tokens) - first;
    }
    const int rows = count * p.group;
    const int tile0 = p.tiles - 1 - (int)blockIdx.x;                       // later tiles see more keys: they start first
    if (tile0 * kTileRows >= rows) return;                                 // the whole CTA
    const int seq = max(c.seq_lens[r], 0);
    const long long capacity = (long long)c.bt_cols << c.page_shift;
    const int* table = c.block_table + r * c.bt_stride;

    if (tid == 0) {
        for (int i = 0; i < kPromptStages; ++i) {
            mbar_init(&sh.full[i], kProducers);
            mbar_init(&sh.empty[i], 1);
        }
        mbar_init(&sh.q_full, 128);
        mbar_init(&sh.s_full[0], 2);                                       // the products, and the thread that saw the scales
        mbar_init(&sh.s_full[1], 2);
        mbar_init(&sh.p_full[0], 128);
        mbar_init(&sh.p_full[1], 128);
        mbar_init(&sh.pv_done[0], 1);
        mbar_init(&sh.pv_done[1], 1);
        mbar_init(&sh.drain, 1);
        sh.abort = sh.nan_out = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 7) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(kPromptCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;

    uint32_t n = 0, tiles_done = 0;                                        // steps and tiles before this tile: barrier parities
    for (int tile = tile0; tile * kTileRows < rows; tile += p.tiles, ++tiles_done) {
        const int last = (min(tile * kTileRows + kTileRows, rows) - 1) / p.group, lead = tile * kTileRows / p.group;
        const int len_max = (int)min((long long)max(seq - count + last + 1, 0), capacity);
        const int len_min = (int)min((long long)max(seq - count + lead + 1, 0), capacity);
        const int steps = (len_max + kTileKeys - 1) / kTileKeys;
        if (warp < 4) {
            // ---------------- softmax: one row a thread
            asm volatile("bar.sync 1, 128;" ::: "memory");                // no warp is a tile ahead of another
            float qs;
            int len;
            {
                const int row = tile * kTileRows + tid, tok = row / p.group, head = h * p.group + row - tok * p.group;
                const bool on = row < rows;
                len = on ? (int)min((long long)max(seq - count + tok + 1, 0), capacity) : len_max;
                uint4 w[8];
                const uint4* src = reinterpret_cast<const uint4*>(p.q + (long long)(first + tok) * p.q_token + (long long)head * p.q_head);
                float amax = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    w[i] = on ? src[i] : make_uint4(0, 0, 0, 0);
                    const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(u[j])), fabsf(bf16_hi(u[j]))));
                }
                const int ex = max(min((int)(__float_as_uint(amax) >> 23) - 134, 126), -126);
                const float f2 = copysignf(exp2_biased(127 - ex), p.scale);
                qs = fabsf(p.scale) * exp2_biased(127 + ex);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                    uint32_t f[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) f[j] = pack_f16x2(bf16_lo(u[j]) * f2, bf16_hi(u[j]) * f2);
                    *reinterpret_cast<uint4*>(q_tile + tid * 128 + ((i ^ (tid & 7)) * 16)) = make_uint4(f[0], f[1], f[2], f[3]);
                }
                fence_async_smem();
                mbar_arrive(&sh.q_full);
            }
            const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
            float m = kNegInf, top = kNegInf, l = 0.f;
            int i = 0;                                                     // short of `steps` where a wait gave up
            for (; i < steps; ++i) {
                const uint32_t at = n + i, stage = at % kPromptStages;
                if (!warp_wait(sh, &sh.s_full[at & 1], at >> 1, p.wait_limit)) break;
                tc_fence_after();
                float s[kTileKeys];
                tmem_ld32(lanes + (at & 1) * kTileKeys, s);
                tmem_ld32(lanes + (at & 1) * kTileKeys + 32, s + 32);
                const float4 ks4 = *reinterpret_cast<const float4*>(sh.ks[stage]), ev4 = *reinterpret_cast<const float4*>(sh.ev[stage]),
                             bias4 = *reinterpret_cast<const float4*>(sh.bias[stage]);
                const float ks[4] = {ks4.x, ks4.y, ks4.z, ks4.w}, ev[4] = {ev4.x, ev4.y, ev4.z, ev4.w},
                            bias[4] = {bias4.x, bias4.y, bias4.z, bias4.w};
                tmem_ld_wait();
                if (__builtin_expect(i * kTileKeys + kTileKeys > len_min, 0)) {
                    const int left = len - i * kTileKeys;                  // scores from here on are masked
#pragma unroll
                    for (int k = 0; k < kTileKeys; ++k)
                        if (k >= left) s[k] = kNegInf;
                }
                float ck[4], m1 = m, t1 = top;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float mx[3];
#pragma unroll
                    for (int k = 0; k < 3; ++k) mx[k] = max3(s[16 * u + 5 * k], s[16 * u + 5 * k + 1], s[16 * u + 5 * k + 2]);
#pragma unroll
                    for (int k = 0; k < 3; ++k) mx[k] = max3(mx[k], s[16 * u + 5 * k + 3], s[16 * u + 5 * k + 4]);
                    mx[0] = fmaxf(max3(mx[0], mx[1], mx[2]), s[16 * u + 15]);
                    ck[u] = fmaxf(ks[u] * qs, 1e-37f);           // never 0: a masked score times it stays -inf
                    const float x = fmaf(mx[0], ck[u], bias[u]);
                    m1 = fmaxf(m1, x);
                    t1 = fmaxf(t1, x + ev[u]);
                }
                const float mu = m1 == kNegInf ? 0.f : m1;
                l *= ex2(m - mu);
                m = m1;
                float turn = 1.f;
                if (t1 > top + kLazy) {                                    // top = -inf: any finite maximum
                    turn = ex2(top - t1);
                    top = t1;
                }
                const float tu = top == kNegInf ? 0.f : top;
                // weights straight as 2^(s + ev - top), their sum put back to 2^(s - m); a page whose V scale is so small that
                // its weights vanish (a page of zeros) still counts in the sum: in two steps there
                // all arguments, the exponentials of the first half, those of the second between the first's uses: the
                // exponential unit is what the others wait for
                float f[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) f[u] = ex2(fminf(mu + ev[u] - tu, 127.f));       // 2^(s - m) -> 2^(s + ev - top)
#pragma unroll
                for (int k = 0; k < kTileKeys; k += 2) {
                    const float to_m = bias[k / 16] - mu;
                    const float2 x = fma2(make_float2(s[k], s[k + 1]), make_float2(ck[k / 16], ck[k / 16]), make_float2(to_m, to_m));
                    s[k] = x.x;
                    s[k + 1] = x.y;
                }
#pragma unroll
                for (int k = 0; k < 32; ++k) s[k] = ex2(s[k]);
                float2 sum[4] = {};
                uint32_t pk[16];
                auto use = [&](int k) {                                    // keys k, k + 1
                    const float2 e = make_float2(s[k], s[k + 1]);
                    sum[k / 16] = add2(sum[k / 16], e);
                    const float2 w = mul2(e, make_float2(f[k / 16], f[k / 16]));
                    pk[k / 2 % 16] = pack_f16x2(w.x, w.y);
                };
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    s[32 + k] = ex2(s[32 + k]);
                    s[33 + k] = ex2(s[33 + k]);
                    use(k);
                }
                if (i > 1) {                                               // this P has been read
                    if (!warp_wait(sh, &sh.pv_done[at & 1], (at - 2) >> 1, p.wait_limit)) break;
                    tc_fence_after();
                }
                tmem_st16(lanes + kColP + (at & 1) * 32, pk);
#pragma unroll
                for (int k = 32; k < kTileKeys; k += 2) use(k);
                tmem_st16(lanes + kColP + (at & 1) * 32 + 16, pk);
#pragma unroll
                for (int u = 0; u < 4; ++u) l += sum[u].x + sum[u].y;
                if (__builtin_expect(i > 0 && __any_sync(kFullMask, turn != 1.f), 0)) {
                    if (!warp_wait(sh, &sh.pv_done[(at - 1) & 1], (at - 1) >> 1, p.wait_limit)) break;
                    tc_fence_after();
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        tmem_ld32(lanes + kColO + 32 * d, s);
                        tmem_ld_wait();
#pragma unroll
                        for (int k = 0; k < 32; ++k) s[k] *= turn;
                        tmem_st32(lanes + kColO + 32 * d, s);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&sh.p_full[at & 1]);                           // two: a warp may be a step ahead of another
            }
            if (any_of_softmax(i < steps || (steps > 0 && !warp_wait(sh, &sh.pv_done[(n + steps - 1) & 1], (n + steps - 1) >> 1, p.wait_limit)))) {
                tmem_st_wait();                                            // on its way when the loop was left
                tc_fence_before();
                rows_given_up(p, tile);
                break;
            }
            float f = 0.f, g = 1.f;
            if (steps > 0) {
                tc_fence_after();
                f = unscale(top - m, l, g);
            }
            int again = tid;                                               // worked out once more: not kept in registers over the loop
            asm volatile("" : "+r"(again));
            const int row = tile * kTileRows + again, tok = row / p.group, head = h * p.group + row - tok * p.group;
            const bool on = row < rows;
            uint4* to = reinterpret_cast<uint4*>(p.out + (long long)(first + tok) * p.o_token + (long long)head * p.o_head);
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                float o[32];
                if (steps > 0) {
                    tmem_ld32(lanes + kColO + 32 * d, o);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = l == 0.f ? 0.f : o[k] * f * g;  // l = 0: sees no key
                float any = o[0];
#pragma unroll
                for (int k = 1; k < 32; ++k) any = fmaf(o[k], 0.f, any);   // NaN if one is (or an infinity)
                if (any != any) sh.nan_out = 1;
                if (on) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        to[4 * d + k] = make_uint4(pack_bf16x2(o[8 * k], o[8 * k + 1]), pack_bf16x2(o[8 * k + 2], o[8 * k + 3]),
                                                   pack_bf16x2(o[8 * k + 4], o[8 * k + 5]), pack_bf16x2(o[8 * k + 6], o[8 * k + 7]));
                }
            }
            if (on && p.lse) p.lse[(long long)(first + tok) * p.q_heads + head] = l == 0.f ? kNegInf : (m + log2f(l)) * 0.6931471805599453f;
            tc_fence_before();                                             // the accumulator is read: the next tile may write it
        } else {
            // ---------------- e4m3 pages to f16 tiles: a warp carries 16 keys of each step, a lane 16 bytes of two K rows and
            // of two V rows; the pages of the warp's next 32 steps and their scales are held one a lane.  The last warp issues
            // the products as well.
            const int unit = warp - 4, key = lane >> 2, part = lane & 3;
            static_assert(kProducers == 128 && kTileKeys == 64, "four warps, a quarter of a tile each");
            const uint8_t* from = c.cache + (long long)h * c.head_stride + c.k_off + key * c.token_stride + 16 * part;
            const long long v_from_k = c.v_off - c.k_off, eight = 8 * c.token_stride;
            const int in_page = (1 << c.page_shift) - 1;
            unsigned char* mine = raw_ring + (tid - 128) * 16;             // two K rows, two V rows; read back by their writer
            const uint32_t lo_at = (16 * unit + key) * 128 + ((2 * part) ^ key) * 16, hi_at = (16 * unit + key) * 128 + ((2 * part + 1) ^ key) * 16;
            int pages = -1, used_pages = -1;                               // of the steps being fetched, being converted
            uint32_t scale2 = 0, used_scale2 = 0;
            auto fetch = [&](int i) {
                const int at = i * kTileKeys + 16 * unit;
                if ((i & 31) == 0) {
                    const int first_key = at + lane * kTileKeys;
                    used_pages = pages;
                    used_scale2 = scale2;
                    pages = first_key < len_max ? table[first_key >> c.page_shift] : -1;
                    if (pages >= c.pages || pages < 0) pages = -1;
                    scale2 = pages < 0 ? 0u : *reinterpret_cast<const uint16_t*>(c.scales + ((long long)pages * c.kv_heads + h) * 2);
                }
                const int page = __shfl_sync(kFullMask, pages, i & 31);
                const int left = page < 0 ? 0 : len_max - at;
                const uint8_t* src = from + (page < 0 ? 0 : (long long)page * c.page_stride + (long long)(at & in_page) * c.token_stride);
                unsigned char* to = mine + (i % kRawStages) * kRawBytes;
                const bool on0 = key < left, on1 = key + 8 < left;
                const uint8_t *src0 = on0 ? src : from, *src1 = on1 ? src + eight : from;
                cp_async16(to, src0, on0);
                cp_async16(to + kProducers * 16, src1, on1);
                cp_async16(to + 2 * kProducers * 16, src0 + v_from_k, on0);
                cp_async16(to + 3 * kProducers * 16, src1 + v_from_k, on1);
                cp_async_commit();
            };
            auto produce = [&](int i) -> bool {
                const uint32_t at = n + i, stage = at % kPromptStages;
                fetch(i + kRawStages - 1);                                 // steps past the last fetch zeros
                cp_async_wait<kRawStages - 1>();
                if (at >= kPromptStages && !warp_wait(sh, &sh.empty[stage], at / kPromptStages - 1, p.wait_limit)) return false;
                unsigned char* k_tile = kv_tiles + stage * 2 * kTileKeys * 128;
                const unsigned char* raw16 = mine + (i % kRawStages) * kRawBytes;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint4 v = *reinterpret_cast<const uint4*>(raw16 + j * kProducers * 16);
                    unsigned char* to = k_tile + (j >> 1) * kTileKeys * 128 + (j & 1) * 8 * 128;
                    uint4 lo, hi;
                    e4m3x4_to_f16(v.x, lo.x, lo.y);
                    e4m3x4_to_f16(v.y, lo.z, lo.w);
                    e4m3x4_to_f16(v.z, hi.x, hi.y);
                    e4m3x4_to_f16(v.w, hi.z, hi.w);
                    *reinterpret_cast<uint4*>(to + lo_at) = lo;
                    *reinterpret_cast<uint4*>(to + hi_at) = hi;
                }
                const bool older = ((i + kRawStages - 1) & ~31) != (i & ~31);
                if (lane == (i & 31)) {
                    const bool none = (older ? used_pages : pages) < 0;
                    const uint32_t two = older ? used_scale2 : scale2;
                    sh.ks[stage][unit] = exp2_biased(two & 0xffu);
                    sh.ev[stage][unit] = (float)(int)(two >> 8) - 127.f;
                    sh.bias[stage][unit] = none ? kNegInf : 0.f;
                }
                fence_async_smem();
                mbar_arrive(&sh.full[stage]);
                return true;
            };
            for (int i = 0; i < kRawStages - 1; ++i) fetch(i);
            bool fed = true, ok = true;                                    // no wait of the warp for a stage, of this lane for products, gave up
            if (warp < 7) {
                for (int i = 0; fed && i < steps; ++i) fed = produce(i);
            } else {
                const uint64_t dq = tile_desc(q_tile);
                auto scores = [&](int i) -> bool {
                    const uint32_t at = n + i, stage = at % kPromptStages;
                    if (!prompt_wait(sh, &sh.full[stage], at / kPromptStages, p.wait_limit)) return false;
                    tc_fence_after();
                    const uint64_t dk = tile_desc(kv_tiles + stage * 2 * kTileKeys * 128);
#pragma unroll
                    for (int k = 0; k < 4; ++k)                            // 16 dims = 32 bytes a product
                        mma_ss(tmem + (at & 1) * kTileKeys, dq + 2 * k, dk + 2 * k, kIdescQK, k > 0);
                    mma_commit(&sh.s_full[at & 1]);
                    mbar_arrive(&sh.s_full[at & 1]);                       // hands on the scales that came with the tile
                    return true;
                };
                // two tiles ahead of the products: a tile's stage is free once the products of four steps before are done
                for (int i = 0; fed && i < min(2, steps); ++i) fed = produce(i);
                if (lane == 0) ok = prompt_wait(sh, &sh.q_full, tiles_done, p.wait_limit) && (steps == 0 || scores(0));
                __syncwarp();
                for (int i = 0; i < steps; ++i) {
                    if (lane == 0 && ok && i + 1 < steps) ok = scores(i + 1);
                    __syncwarp();
                    if (fed && i + 2 < steps) fed = produce(i + 2);
                    if (lane == 0 && ok) {
                        const uint32_t at = n + i, stage = at % kPromptStages;
                        ok = prompt_wait(sh, &sh.p_full[at & 1], at >> 1, p.wait_limit);
                        if (ok) {
                            tc_fence_after();
                            const uint64_t dv = tile_desc(kv_tiles + stage * 2 * kTileKeys * 128 + kTileKeys * 128);
#pragma unroll
                            for (int k = 0; k < 4; ++k)                    // 16 keys = 2048 bytes of V, 8 columns of P
                                mma_ts(tmem + kColO, tmem + kColP + (at & 1) * 32 + 8 * k, dv + 128 * k, kIdescPV, i > 0 || k > 0);
                            mma_commit(&sh.empty[stage]);
                            mma_commit(&sh.pv_done[at & 1]);
                        }
                    }
                    __syncwarp();
                }
            }
            cp_async_wait<0>();                                            // the next tile's copies go to the same places
            if (!__all_sync(kFullMask, fed && ok)) break;
        }
        n += (uint32_t)steps;
    }
    if (warp == 7) {
        if (lane == 0) {                                                   // nothing is in flight when the memory goes
            mma_commit(&sh.drain);                                         // also after a wait that gave up: whoever did
            unsigned polls = 0;
            while (!mbar_test(&sh.drain, 0) && ++polls < kWaitLimit) {}
            if (polls == kWaitLimit) gave_up(sh);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 7) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kPromptCols) : "memory");
    if (__builtin_expect(sh.nan_out && warp < 4, 0) && !sh.abort) rows_apart(p);
}

// ---------------------------------------------------------------- host
// The dynamic shared memory a kernel may have is set once per device, not before every launch.
template <typename K> cudaError_t allow_shared(K kernel, int bytes, std::atomic<unsigned long long>& done) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}
std::atomic<unsigned long long> g_prompt_ready{0}, g_attend_ready[2];
std::atomic<unsigned> g_wait_limit{kWaitLimit};

int kv8_params(const PkKv8Cache* a, int tokens, Kv8Params& c) {
    if (!a) return kErrNull;
    if (a->batch < 0 || a->batch > 65535 || tokens < 0 || a->kv_heads <= 0 || a->kv_heads > 65535 || a->pages < 0 ||
        a->bt_cols < 0)
        return kErrShape;
    int shift = 4;
    while (shift < 8 && (1 << shift) != a->page_size) ++shift;
    if ((1 << shift) != a->page_size) return kErrBlock;                      // 16, 32, 64, 128 or 256
    // the kernels look up pages up to 32 steps of 64 keys past a row's last key, in 32 bits
    if ((long long)a->bt_cols * a->page_size > 0x7fff0000LL) return kErrMaxSeq;
    if (a->batch == 0 || tokens == 0) return -1;                             // nothing to do
    if (!a->cache || !a->scales || !a->seq_lens || (a->bt_cols > 0 && !a->block_table)) return kErrNull;
    if (reinterpret_cast<uintptr_t>(a->cache) % 16 || reinterpret_cast<uintptr_t>(a->scales) % 2 || a->k_off % 16 || a->v_off % 16 || a->page_stride % 16 ||
        a->token_stride % 16 || a->head_stride % 16 || reinterpret_cast<uintptr_t>(a->block_table) % 4 ||
        reinterpret_cast<uintptr_t>(a->seq_lens) % 4 || reinterpret_cast<uintptr_t>(a->cu_seqlens) % 4)
        return kErrAlign;
    if (!a->cu_seqlens && tokens < a->batch) return kErrShape;
    c.cache = static_cast<uint8_t*>(a->cache);
    c.scales = static_cast<uint8_t*>(a->scales);
    c.k_off = a->k_off; c.v_off = a->v_off;
    c.page_stride = a->page_stride; c.token_stride = a->token_stride; c.head_stride = a->head_stride;
    c.pages = a->pages; c.page_shift = shift; c.kv_heads = a->kv_heads;
    c.block_table = static_cast<const int*>(a->block_table);
    c.bt_stride = a->bt_stride; c.bt_cols = a->bt_cols;
    c.seq_lens = static_cast<const int*>(a->seq_lens);
    c.cu = static_cast<const int*>(a->cu_seqlens);
    c.batch = a->batch; c.tokens = tokens;
    return kOk;
}

}  // namespace pk

// Bounded waits of the prompt kernel that gave up on the current device since the library was loaded (0 in normal
// operation; rows of a launch that could not be finished are NaN).  Waits for all work on the device.
extern "C" long long pk_kv8_wait_timeouts(void) {
    unsigned int n = 0;
    if (cudaDeviceSynchronize() != cudaSuccess) return -1;
    if (cudaMemcpyFromSymbol(&n, pk::g_kv8_wait_timeouts, sizeof(n)) != cudaSuccess) return -1;
    return (long long)n;
}

// Polls after which a wait of later launches gives up; 0: at the first one that is not over already; < 0: the default.
extern "C" void pk_kv8_set_wait_limit(int polls) {
    pk::g_wait_limit.store(polls < 0 ? pk::kWaitLimit : (unsigned)polls, std::memory_order_relaxed);
}

extern "C" int pk_kv8_append(const PkKv8Cache* cache, const void* k, long long k_token_stride, long long k_head_stride,
                             const void* v, long long v_token_stride, long long v_head_stride, int tokens, void* stream) {
    using namespace pk;
    AppendParams p{};
    const int rc = kv8_params(cache, tokens, p.c);
    if (rc != kOk) return rc < 0 ? kOk : rc;
    if (!k || !v) return kErrNull;
    if (reinterpret_cast<uintptr_t>(k) % 16 || reinterpret_cast<uintptr_t>(v) % 16 || k_token_stride % 8 || k_head_stride % 8 ||
        v_token_stride % 8 || v_head_stride % 8)
        return kErrAlign;
    p.k = static_cast<const uint16_t*>(k);
    p.v = static_cast<const uint16_t*>(v);
    p.k_token = k_token_stride; p.k_head = k_head_stride;
    p.v_token = v_token_stride; p.v_head = v_head_stride;
    const int group = p.c.cu ? 16 : 1;
    const long long blocks = (((long long)tokens + group - 1) / group * p.c.kv_heads + 7) / 8;
    if (blocks > 0x7fffffffLL) return kErrShape;
    if (p.c.cu) kv8_append_kernel<16><<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
    else kv8_append_kernel<1><<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return (int)cudaPeekAtLastError();
}

extern "C" int pk_kv8_attention(const PkKv8Cache* cache, const void* q, long long q_token_stride, long long q_head_stride,
                                void* out, long long out_token_stride, long long out_head_stride, void* lse, int tokens,
                                int q_heads, int max_query_len, float scale, void* stream) {
    using namespace pk;
    AttendParams p{};
    const int rc = kv8_params(cache, tokens, p.c);
    if (rc != kOk) return rc < 0 ? kOk : rc;
    if (q_heads <= 0 || q_heads % p.c.kv_heads || max_query_len < 0) return kErrShape;
    if (!q || !out) return kErrNull;
    if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(out) % 16 || q_token_stride % 8 || q_head_stride % 8 ||
        out_token_stride % 8 || out_head_stride % 8 || reinterpret_cast<uintptr_t>(lse) % 4)
        return kErrAlign;
    p.q = static_cast<const uint16_t*>(q);
    p.out = static_cast<uint16_t*>(out);
    p.q_token = q_token_stride; p.q_head = q_head_stride;
    p.o_token = out_token_stride; p.o_head = out_head_stride;
    p.lse = static_cast<float*>(lse);
    p.q_heads = q_heads;
    p.group = q_heads / p.c.kv_heads;
    p.scale = scale * 1.4426950408889634f;
    int longest = p.c.cu ? (max_query_len > 0 && max_query_len < tokens ? max_query_len : tokens) : 1;
    if ((long long)(p.c.cu ? tokens : 1) * p.group > 0x3fffff00LL) return kErrShape;     // row + a turn of tiles: 32 bits
    const long long mean = ((long long)tokens + p.c.batch - 1) / p.c.batch * p.group;      // rows of a request
    // The prompt kernel's tile of 128 rows takes 1.2 us for 64 keys however few of them there are, and no tile's keys are
    // split; the other kernel's rate does not depend on either.  They meet at 740 tiles of 16 rows where the SMs are not
    // full, and at tiles of 128 rows that are 45 % full: 1 request of 128 tokens, 15/5 heads (120 tiles) 77 us against
    // 23; 8 of 32, 32/32 heads (512) 45 against 29; 16 of 256, 9/3 heads (2304) 85 against 131; 32 of 64, 32/32 heads
    // (4096, half full) 77 against 108.
    const long long sets = (long long)p.c.kv_heads * p.c.batch, small = (mean + 15) / 16 * sets;
    // Tiles a request gets CTAs for (more are taken in turns): all that the longest can have, but CTAs with nothing to do
    // cost 1.5 ns each, so no more than twice the mean or what fills the GPU if one request has nearly all rows.  (256
    // requests of 4 tokens, 15/5 heads, 2048 keys, longest not known: 98 us, 457 with a CTA for every possible tile.)
    auto tiles_of = [&](int rows) {
        const long long tiles = ((long long)longest * p.group + rows - 1) / rows;
        const long long likely = (mean + rows - 1) / rows * 2, some = 8192 / sets, most = likely > some ? likely : some;
        return (int)(tiles < most ? tiles : most);
    };
    if (small >= 740 && 10 * small >= 36 * ((mean + kTileRows - 1) / kTileRows) * sets) {
        p.tiles = tiles_of(kTileRows);
        p.wait_limit = g_wait_limit.load(std::memory_order_relaxed);
        const cudaError_t e = allow_shared(kv8_prompt_kernel, kPromptBytes, g_prompt_ready);
        if (e != cudaSuccess) return (int)e;
        kv8_prompt_kernel<<<dim3((unsigned)p.tiles, (unsigned)p.c.kv_heads, (unsigned)p.c.batch), kPromptThreads, kPromptBytes,
                            static_cast<cudaStream_t>(stream)>>>(p);
        return (int)cudaPeekAtLastError();
    }
    const int tile_rows = (long long)longest * p.group <= 8 ? 8 : 16;
    p.tiles = tiles_of(tile_rows);
    const long long items = (mean + tile_rows - 1) / tile_rows * sets;
    const long long steps = (((long long)p.c.bt_cols << p.c.page_shift) + 31) / 32;
    // CTAs that share the keys of one item: as many as are resident at once (two on each of 148 SMs), at least two steps
    // for each warp.  Where that leaves eight steps or more an eighth more CTAs is worth a second wave (32 requests x 5 kv
    // heads at 8192 keys: 27.7 us with two CTAs an item, 38.9 with one); with two steps it is not (16 requests at 2048
    // keys: 13.1 us with four, 10.0 with three).  Fewer than two steps cost more in merging than they save (8 requests of
    // 5 tokens at 2047 keys: 12.3 us, 9.4).  Lengths are on the device, so the table's width stands for them: the same 8
    // requests with a table for 8192 keys take 12.4 us, one request of 520 keys 6.1 us with either.
    const long long worth = steps / (2 * kAttWarps);
    long long fit = 340 / items;
    if (fit > steps / (8 * kAttWarps)) fit = 296 / items;
    const long long share = fit < worth ? fit : worth;
    const int c = (int)(share < 1 ? 1 : (share < 8 ? share : 8));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(p.tiles * c), (unsigned)p.c.kv_heads, (unsigned)p.c.batch);
    cfg.blockDim = dim3(kAttWarps * 32);
    cfg.dynamicSmemBytes = kAttShared;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)c;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const auto kernel = tile_rows == 8 ? kv8_attend_kernel<true> : kv8_attend_kernel<false>;
    const cudaError_t e = allow_shared(kernel, kAttShared, g_attend_ready[tile_rows == 8]);
    return (int)(e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, kernel, p));
}
