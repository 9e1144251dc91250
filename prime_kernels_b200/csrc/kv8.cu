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
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {     // low 16 bits; exact
    uint32_t r;
    asm("{\n.reg .b16 t;\ncvt.u16.u32 t, %1;\ncvt.rn.f16x2.e4m3x2 %0, t;\n}" : "=r"(r) : "r"(two));
    return r;
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
// One warp per (token, kv head); the first new token of a page leads and stores all new tokens of that page.
struct AppendParams {
    Kv8Params c;
    const uint16_t *k, *v;
    long long k_token, k_head, v_token, v_head;        // elements
};

__device__ __forceinline__ float finite_abs(float x) {
    x = fabsf(x);
    return x < __int_as_float(0x7f800000) ? x : 0.f;   // NaN and Inf do not count
}
__device__ __forceinline__ float amax8(const uint4 q) {
    float a = fmaxf(finite_abs(bf16_lo(q.x)), finite_abs(bf16_hi(q.x)));
    a = fmaxf(a, fmaxf(finite_abs(bf16_lo(q.y)), finite_abs(bf16_hi(q.y))));
    a = fmaxf(a, fmaxf(finite_abs(bf16_lo(q.z)), finite_abs(bf16_hi(q.z))));
    return fmaxf(a, fmaxf(finite_abs(bf16_lo(q.w)), finite_abs(bf16_hi(q.w))));
}

__global__ void __launch_bounds__(256) kv8_append_kernel(AppendParams p) {
    const Kv8Params& c = p.c;
    const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (item >= (long long)c.tokens * c.kv_heads) return;
    const int t = (int)(item / c.kv_heads), h = (int)(item - (long long)t * c.kv_heads);
    int r, first, count;
    if (!request_of(c, t, r, first, count)) return;
    const int size = 1 << c.page_shift;
    const long long pos = (long long)c.seq_lens[r] - count + (t - first);
    if (pos < 0) return;
    const int slot = (int)(pos & (size - 1));
    if (slot != 0 && t != first) return;               // another token of this page leads
    const long long col = pos >> c.page_shift;
    if (col >= c.bt_cols) return;
    const int page = c.block_table[r * c.bt_stride + col];
    if (page < 0 || page >= c.pages) return;
    const int m = min(size - slot, first + count - t);
    uint8_t* base = c.cache + (long long)page * c.page_stride + (long long)h * c.head_stride;
    uint8_t* scale = c.scales + ((long long)page * c.kv_heads + h) * 2;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const uint16_t* src = x ? p.v + (long long)t * p.v_token + (long long)h * p.v_head
                                : p.k + (long long)t * p.k_token + (long long)h * p.k_head;
        const long long step = x ? p.v_token : p.k_token;
        uint8_t* dst = base + (x ? c.v_off : c.k_off);
        float amax = 0.f;
        for (int i = lane >> 3; i < m; i += 4)
            amax = fmaxf(amax, amax8(*reinterpret_cast<const uint4*>(src + i * step + (lane & 7) * 8)));
        amax = warp_max(amax);
        uint32_t e = e8m0_roundup(__fmul_rn(amax, 1.f / 448.f));
        if (slot) {
            const uint32_t old = min((uint32_t)scale[x], 254u);
            if (e > old) {                             // the scale grows: values held move by 2^(old - e)
                const float f = exp2_biased(127u - min(e - old, 126u));
                for (int i = lane >> 2; i < slot; i += 8) {
                    uint4* q = reinterpret_cast<uint4*>(dst + (long long)i * c.token_stride + (lane & 3) * 16);
                    uint4 a = *q;
                    uint32_t* w = reinterpret_cast<uint32_t*>(&a);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t lo = e4m3x2_to_f16x2(w[j] & 0xffffu), hi = e4m3x2_to_f16x2(w[j] >> 16);
                        const float2 fl = __half22float2(*reinterpret_cast<const __half2*>(&lo));
                        const float2 fh = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                        w[j] = e4m3x2(fl.x * f, fl.y * f) | (e4m3x2(fh.x * f, fh.y * f) << 16);
                    }
                    *q = a;
                }
            } else {
                e = old;
            }
        }
        const float inv = exp2_biased(254u - e);
        for (int i = lane >> 3; i < m; i += 4) {
            const uint4 q = *reinterpret_cast<const uint4*>(src + i * step + (lane & 7) * 8);
            uint2 o;
            o.x = e4m3x2(bf16_lo(q.x) * inv, bf16_hi(q.x) * inv) | (e4m3x2(bf16_lo(q.y) * inv, bf16_hi(q.y) * inv) << 16);
            o.y = e4m3x2(bf16_lo(q.z) * inv, bf16_hi(q.z) * inv) | (e4m3x2(bf16_lo(q.w) * inv, bf16_hi(q.w) * inv) << 16);
            *reinterpret_cast<uint2*>(dst + (long long)(slot + i) * c.token_stride + (lane & 7) * 8) = o;
        }
        __syncwarp();
        if (lane == 0) scale[x] = (uint8_t)e;
    }
}

// ---------------------------------------------------------------- attention
// Rows of one (request, kv head): (token, query head of the group), row = token * G + head; tiles of 16 rows.  A
// tile's keys are dealt to the CTAs of a cluster and, in steps of 16 keys, to the warps of a CTA; every warp keeps a
// running softmax of its own (one pass over the cache), merged at the end in shared memory and then through
// distributed shared memory.  Products run on m16n8k16 f16 with fp32 accumulation: e4m3 converts to f16 exactly, and
// q is divided by a power of two per row so that its bf16 bits fit f16 (elements 2^-22 below the row's largest lose
// bits).  The cache goes from global memory straight into the operand registers: a lane's 16 bytes of a K row are
// its dims of all four k-steps, and pairs of V rows are interleaved by byte permutation.
//
// V scales differ from page to page, so weights enter the second product as 2^(s + eV - top) with a running maximum
// `top` of s + eV of their own, apart from the running maximum of s that the sum uses: neither over- nor underflows
// whatever the scales are.
struct AttendParams {
    Kv8Params c;
    const uint16_t* q;
    long long q_token, q_head;                         // elements
    uint16_t* out;
    long long o_token, o_head;
    float* lse;                                        // [tokens, q heads] or null
    int q_heads, group, tiles;
    float scale;                                       // softmax scale * log2(e)
};

constexpr int kAttWarps = 8;
constexpr float kNegInf = -__builtin_huge_valf();

struct __align__(16) AttendShared {
    float o[16][kHeadDim + 4];
    float m[16], top[16], l[16];                       // running maxima (log2) and sum
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
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
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(kFullMask, v, 1));
    return fmaxf(v, __shfl_xor_sync(kFullMask, v, 2));
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

__global__ void __launch_bounds__(kAttWarps * 32) kv8_attend_kernel(AttendParams p) {
    const Kv8Params& c = p.c;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    __shared__ AttendShared sh[kAttWarps];
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
    for (int tile = blockIdx.x / C; tile * 16 < rows; tile += p.tiles) {
        // ---- the two rows of this lane
        int len[2], ex[2];
        uint32_t qa[2][8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = tile * 16 + g + 8 * i;
            const int tok = row / p.group;
            const bool on = row < rows;
            len[i] = on ? (int)min((long long)max(seq - count + tok + 1, 0), capacity) : 0;
            ex[i] = load_q(on ? p.q + (long long)(first + tok) * p.q_token + (long long)(h * p.group + row - tok * p.group) * p.q_head
                              : nullptr, t, qa[i]);
        }
        const int last = (min(tile * 16 + 16, rows) - 1) / p.group, lead = tile * 16 / p.group;
        const int len_max = (int)min((long long)max(seq - count + last + 1, 0), capacity);
        const int len_min = tile * 16 + 16 > rows ? 0 : (int)min((long long)max(seq - count + lead + 1, 0), capacity);
        const float qs[2] = {p.scale * exp2_biased(127 + ex[0]), p.scale * exp2_biased(127 + ex[1])};
        // ---- keys: steps of 16 keys, a contiguous share per CTA, dealt to its warps
        const int steps = (len_max + 15) / 16, share = (steps + C - 1) / C;
        const int s_end = min((rank + 1) * share, steps);
        float o[8][4], m[2] = {kNegInf, kNegInf}, top[2] = {kNegInf, kNegInf}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        for (int st = rank * share + warp; st < s_end; st += kAttWarps) {
            const int key0 = st * 16;
            const int page = table[key0 >> c.page_shift];
            if (page < 0 || page >= c.pages) continue;                       // masked
            const uint8_t* base = c.cache + (long long)page * c.page_stride + (long long)h * c.head_stride +
                                  (long long)(key0 & ((1 << c.page_shift) - 1)) * c.token_stride;
            const uint8_t* sc = c.scales + ((long long)page * c.kv_heads + h) * 2;
            const uint32_t ek = sc[0];
            const int ev = (int)sc[1] - 127;
            uint4 kw[2] = {};
            uint2 vw[4] = {};
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (key0 + g + 8 * j < len_max)
                    kw[j] = *reinterpret_cast<const uint4*>(base + c.k_off + (g + 8 * j) * c.token_stride + 16 * t);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = 2 * t + (j & 1) + 8 * (j >> 1);
                if (key0 + key < len_max)
                    vw[j] = *reinterpret_cast<const uint2*>(base + c.v_off + key * c.token_stride + 8 * g);
            }
            float s[2][4] = {};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t w[4] = {kw[j].x, kw[j].y, kw[j].z, kw[j].w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma_f16(s[j], qa[0][2 * k], qa[1][2 * k], qa[0][2 * k + 1], qa[1][2 * k + 1],
                            e4m3x2_to_f16x2(w[k] & 0xffffu), e4m3x2_to_f16x2(w[k] >> 16));
            }
            const float ks = exp2_biased(ek);
            const bool edge = key0 + 16 > len_min;
            float mx[2] = {kNegInf, kNegInf};
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 8 * j + 2 * t + (i & 1);
                    s[j][i] = s[j][i] * ks * qs[i >> 1];
                    if (edge && key >= len[i >> 1]) s[j][i] = kNegInf;
                    mx[i >> 1] = fmaxf(mx[i >> 1], s[j][i]);
                }
            float pw[2][4];
            float turn[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                mx[i] = quad_max(mx[i]);
                const float m1 = fmaxf(m[i], mx[i]), t1 = fmaxf(top[i], mx[i] + (float)ev);
                const float mu = m1 == kNegInf ? 0.f : m1, tu = t1 == kNegInf ? 0.f : t1;
                l[i] *= ex2(m[i] - mu);
                turn[i] = ex2(top[i] - tu);
                const float f = ex2(fminf(mu + (float)ev - tu, 127.f));      // 2^(s - m) -> 2^(s + ev - top)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float e = ex2(s[j][2 * i + k] - mu);
                        l[i] += e;
                        pw[j][2 * i + k] = e * f;
                    }
                m[i] = m1;
                top[i] = t1;
            }
            const uint32_t a0 = pack_f16x2(pw[0][0], pw[0][1]), a1 = pack_f16x2(pw[0][2], pw[0][3]);
            const uint32_t a2 = pack_f16x2(pw[1][0], pw[1][1]), a3 = pack_f16x2(pw[1][2], pw[1][3]);
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                o[d][0] *= turn[0]; o[d][1] *= turn[0]; o[d][2] *= turn[1]; o[d][3] *= turn[1];
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {                                    // dims 8g + 2d, 8g + 2d + 1
                const uint32_t sel = (d & 1) ? 0x7362u : 0x5140u;
                const uint32_t lo = __byte_perm(d < 2 ? vw[0].x : vw[0].y, d < 2 ? vw[1].x : vw[1].y, sel);
                const uint32_t hi = __byte_perm(d < 2 ? vw[2].x : vw[2].y, d < 2 ? vw[3].x : vw[3].y, sel);
                mma_f16(o[2 * d], a0, a1, a2, a3, e4m3x2_to_f16x2(lo & 0xffffu), e4m3x2_to_f16x2(hi & 0xffffu));
                mma_f16(o[2 * d + 1], a0, a1, a2, a3, e4m3x2_to_f16x2(lo >> 16), e4m3x2_to_f16x2(hi >> 16));
            }
        }
        // ---- merge the warps, then the CTAs
#pragma unroll
        for (int i = 0; i < 2; ++i) {
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
        __syncthreads();
        const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * 4;       // 16 threads per row, 4 dims each
        auto merge = [&](int n, auto&& part, float& M, float& TOP, float& L, float (&acc)[4]) {
            M = TOP = kNegInf;
            L = 0.f;
            for (int i = 0; i < n; ++i) {
                M = fmaxf(M, part(i).m[row]);
                TOP = fmaxf(TOP, part(i).top[row]);
            }
            acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
            for (int i = 0; i < n; ++i) {
                const AttendShared& x = part(i);
                if (x.l[row] == 0.f) continue;
                L += x.l[row] * ex2(x.m[row] - M);
                const float f = ex2(x.top[row] - TOP);
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[k] += x.o[row][d0 + k] * f;
            }
        };
        float M, TOP, L, acc[4];
        merge(kAttWarps, [&](int i) -> const AttendShared& { return sh[i]; }, M, TOP, L, acc);
        if (C > 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 4; ++k) sh[0].o[row][d0 + k] = acc[k];
            if (d0 == 0) {
                sh[0].m[row] = M;
                sh[0].top[row] = TOP;
                sh[0].l[row] = L;
            }
            cluster.sync();
            if (rank == 0)
                merge(C, [&](int i) -> const AttendShared& { return *cluster.map_shared_rank(&sh[0], i); }, M, TOP, L, acc);
        }
        const int at = tile * 16 + row;
        if (rank == 0 && at < rows) {
            const int tok = at / p.group, head = h * p.group + at - tok * p.group;
            const float f = L == 0.f ? 0.f : ex2(TOP - M) / L;
            uint2 w;
            w.x = pack_bf16x2(acc[0] * f, acc[1] * f);
            w.y = pack_bf16x2(acc[2] * f, acc[3] * f);
            *reinterpret_cast<uint2*>(p.out + (long long)(first + tok) * p.o_token + (long long)head * p.o_head + d0) = w;
            if (p.lse && d0 == 0)
                p.lse[(long long)(first + tok) * p.q_heads + head] = L == 0.f ? kNegInf : (M + log2f(L)) * 0.6931471805599453f;
        }
        if (C > 1) cluster.sync(); else __syncthreads();                     // the parts are read before they are written again
    }
}

// ---------------------------------------------------------------- host
int kv8_params(const PkKv8Cache* a, int tokens, Kv8Params& c) {
    if (!a) return kErrNull;
    if (a->batch < 0 || a->batch > 65535 || tokens < 0 || a->kv_heads <= 0 || a->kv_heads > 65535 || a->pages < 0 ||
        a->bt_cols < 0)
        return kErrShape;
    int shift = 4;
    while (shift < 8 && (1 << shift) != a->page_size) ++shift;
    if ((1 << shift) != a->page_size) return kErrBlock;                      // 16, 32, 64, 128 or 256
    if ((long long)a->bt_cols * a->page_size > 0x7fffffffLL) return kErrMaxSeq;
    if (a->batch == 0 || tokens == 0) return -1;                             // nothing to do
    if (!a->cache || !a->scales || !a->seq_lens || (a->bt_cols > 0 && !a->block_table)) return kErrNull;
    if (reinterpret_cast<uintptr_t>(a->cache) % 16 || a->k_off % 16 || a->v_off % 16 || a->page_stride % 16 ||
        a->token_stride % 16 || a->head_stride % 16)
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
    const long long blocks = ((long long)tokens * p.c.kv_heads + 7) / 8;
    if (blocks > 0x7fffffffLL) return kErrShape;
    kv8_append_kernel<<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
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
    if ((long long)longest * p.group > 0x7fffffffLL - 16) return kErrShape;
    const long long tiles = ((long long)longest * p.group + 15) / 16;
    const long long items = tiles * p.c.kv_heads * p.c.batch;
    const long long steps = (((long long)p.c.bt_cols << p.c.page_shift) + 15) / 16;
    int c = 1;
    while (c < 8 && items * c < 296 && steps > 2 * kAttWarps * c) c *= 2;
    p.tiles = (int)(tiles < (1 << 24) ? tiles : (1 << 24));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(p.tiles * c), (unsigned)p.c.kv_heads, (unsigned)p.c.batch);
    cfg.blockDim = dim3(kAttWarps * 32);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)c;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kv8_attend_kernel, p);
}
