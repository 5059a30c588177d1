// Attention over the pages of a cache that a cheap score picks for every query row and KV head.
//
//   score(page) = sum over the KV head's query heads h of sum_d max(q_hd lo_d, q_hd hi_d)
//               = sum_d (sum_h max(q_hd, 0)) hi_d + (sum_h min(q_hd, 0)) lo_d   (a sum of no head times infinity: 0)
//   out_h       = sum_t w_t v_t / sum_t w_t,  w_t = exp(scale q_h . k_t), t in the picked pages, t <= position
//
// A page's score is one product of 2 head_dim terms, whatever the number of heads. Pages are
// picked by plain fp32 sums with a bound on their error; those too close to call (and all, where
// CTAs share the work or there are more than 512) are summed in twice fp32's precision, so that neither the order
// of a sum nor the split over CTAs decides which of two pages is taken.
//
// One launch does it all. A cluster of 1 to 8 CTAs serves one (row, KV head): its CTAs score
// contiguous parts of the pages, hand the scores to one another through distributed shared
// memory and pick, all alike; then every warp of the cluster attends over 16-key tiles of its own
// with a running maximum and sum, and the parts are joined in shared memory. No workspace, no
// atomics on floating point, sums in a fixed order.
//
// A token's step is bound by reading the picked pages once (2 head_dim elements a key for at most
// 16 query heads: a few operations a byte), many rows of one prompt by the L1 and the instruction
// slots of the SMs, through which every row's pages pass by themselves. So keys and values go from
// global memory to the matrix instructions' registers without a stop in shared memory, by 32-byte
// loads of which 4 lanes take a whole 128-byte line: the 16 keys of a tile are the rows of
// mma.m16n8k16, up to 8 query heads its columns, and the elements of a head are contracted in the
// order in which a lane's bytes hold them; values are turned in registers (movmatrix). tcgen05 would want
// 64 or 128 rows that share their columns' operand; one row's heads and its own pages have 8 or 16 columns.
//
// Measured (device time). 61 rows, 32 pages of 64 keys, bf16, 8 KV heads of 128 with 4 query heads: 88 us, 6.1 TB/s
// of the 6.5 that a plain copy reaches. 1023 rows, 16 of 158 pages of 64 keys, f16, 2 KV heads of 64 with 8
// query heads: 65.7 us (when each was tried, 16-byte loads 84.6, keys by 32 bytes 78.8, values too 68.5, a pick of fewer registers 64.7; tiles
// through TMA and shared memory, which leaves room for fewer CTAs, 94.7 against 84.6). Two rows of 131000 fp32
// keys, 64 of 2000 pages: 26.7 us. One row of 700 keys: 7.3 us. Every CTA keeps 8 bytes of shared memory for each page
// that the table has room for: with 8192 entries instead of 160 the 1023 rows take 102 us, with 16384 179, and 61
// rows of 8192 bf16 keys 63, 114 and 212.
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace vxc {
namespace {

constexpr int kMaxTop = 256;
constexpr int kMaxGroup = 16;
constexpr int kTile = 16;  // keys of a tile; a page holds a whole number of them
constexpr int kMaxCluster = 8;
constexpr int kAlone = 128;  // pages that every CTA of a cluster scores for itself

struct Args {
    vxc_sparse_query a;
    vxc_pages p;
    int layer;
    int cluster;  // CTAs per (row, KV head)
    int keys;     // length of the score array
    int near;     // and of the near scores'
    float scale;
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ uint4 ld16(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p));
    return r;
}

// 32 bytes by one lane, so that 4 lanes take a whole 128-byte line.
__device__ __forceinline__ void ld32(const void* p, uint32_t (&r)[8]) {
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p));
}

template <typename T>
__device__ __forceinline__ void unpack16(const uint4 v, float* x) {
    if constexpr (sizeof(T) == 4) {
        x[0] = __uint_as_float(v.x);
        x[1] = __uint_as_float(v.y);
        x[2] = __uint_as_float(v.z);
        x[3] = __uint_as_float(v.w);
    } else {
        const T* h = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f(h[i]);
    }
}

template <typename T, int N>
__device__ __forceinline__ void unpack_pairs(const uint4 v, float2 (&x)[N]) {
    if constexpr (sizeof(T) == 4) {
        x[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
        x[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
    } else if constexpr (std::is_same_v<T, __half>) {
        const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __half22float2(h[i]);
    } else {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __bfloat1622float2(h[i]);
    }
}
// Elementwise largest magnitude of a 32-bit word of T; a NaN stays.
template <typename T>
__device__ __forceinline__ uint32_t most_abs(uint32_t most, uint32_t v) {
    if constexpr (sizeof(T) == 4) asm("max.NaN.f32 %0, %1, %2;" : "=r"(most) : "r"(most), "r"(v & 0x7fffffffu));
    else if constexpr (std::is_same_v<T, __half>) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(most) : "r"(most), "r"(v & 0x7fff7fffu));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(most) : "r"(most), "r"(v & 0x7fff7fffu));
    return most;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
template <typename T>
__device__ __forceinline__ float largest(uint32_t v) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(v);
    } else {
        const T* h = reinterpret_cast<const T*>(&v);
        return max_nan(to_f(h[0]), to_f(h[1]));
    }
}

// Four consecutive outputs, rounded once.
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
__device__ __forceinline__ void store4(__half* p, float a, float b, float c, float d) {
    __half2 v[2] = {__floats2half2_rn(a, b), __floats2half2_rn(c, d)};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(v);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, float a, float b, float c, float d) {
    __nv_bfloat162 v[2] = {__floats2bfloat162_rn(a, b), __floats2bfloat162_rn(c, d)};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(v);
}

// Scores as integers of the same order; NaN as +infinity, -0 as 0.
__device__ __forceinline__ unsigned long long order_key(float sum, float rest) {
    double s = isfinite(sum) ? static_cast<double>(sum) + static_cast<double>(rest) : static_cast<double>(sum);
    s = s != s ? __longlong_as_double(0x7ff0000000000000ll) : s + 0.0;
    const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(s));
    return b >> 63 ? ~b : b | 1ull << 63;
}

// ------------------------------------------------------------------ cluster
// The wait for a cluster_arrive; every thread does either once.
__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();  // the aligned forms want whole warps
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    __syncthreads();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Every thread of the cluster; what came before is visible to what comes after.
__device__ __forceinline__ void cluster_sync() {
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(const void* local, uint32_t rank) {
    uint32_t addr;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                 : "=r"(addr)
                 : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(local))), "r"(rank));
    return addr;
}
__device__ __forceinline__ float peer_ld(const float* local, uint32_t rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_addr(local, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 peer_ld4(const float* local, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(peer_addr(local, rank))
                 : "memory");
    return v;
}

// ------------------------------------------------------------------ picking
constexpr int kMostWarps = 8;
struct PickSmem {
    unsigned long long lo[kMostWarps], hi[kMostWarps];
    int count[kMostWarps];
    int hist[256];
    int bucket, above;
};

// The m largest of key[0, n), equal ones lowest index first, 0 < m < n: their indices in
// ascending order go to emit(i, rank). Two forms.
//
// n <= 32 kEach, one warp, the keys in registers: the m-th largest by halving the keys' span until exactly m lie
// in the upper part, about 10 rounds for scores that are not equal.
template <int kEach, typename F>
__device__ void pick_warp(const unsigned long long* key, int n, int m, F&& emit) {
    const int lane = threadIdx.x & 31;
    unsigned long long k[kEach];
    unsigned least = ~0u, most = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const bool in = i * 32 + lane < n;
        k[i] = in ? key[i * 32 + lane] : 0;  // no key is 0: that would be a NaN
        if (in) {
            least = min(least, static_cast<unsigned>(k[i] >> 32));
            most = max(most, static_cast<unsigned>(k[i] >> 32));
        }
    }
    // at least m keys >= lo, fewer than m > hi
    unsigned long long lo = static_cast<unsigned long long>(__reduce_min_sync(0xffffffffu, least)) << 32;
    unsigned long long hi = static_cast<unsigned long long>(__reduce_max_sync(0xffffffffu, most)) << 32 | 0xffffffffu;
    int ties = 0;  // keys equal to lo that are taken, where not all are
    bool exact = false;
    while (lo < hi) {
        const unsigned long long mid = hi - (hi - lo) / 2;
        int c = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) c += k[i] >= mid;
        c = __reduce_add_sync(0xffffffffu, c);
        if (c >= m) lo = mid;
        else hi = mid - 1;
        if (c == m) {
            exact = true;
            break;
        }
    }
    if (!exact) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) c += k[i] > lo;
        ties = m - __reduce_add_sync(0xffffffffu, c);
    }
    int at = 0, equal = 0;
    const unsigned below = (1u << lane) - 1;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        bool in = k[i] >= lo && i * 32 + lane < n;
        if (!exact) {
            const bool tie = in && k[i] == lo;
            const unsigned t = __ballot_sync(0xffffffffu, tie);
            if (tie) in = equal + __popc(t & below) < ties;
            equal += __popc(t);
        }
        const unsigned b = __ballot_sync(0xffffffffu, in);
        if (in) emit(i * 32 + lane, at + __popc(b & below));
        at += __popc(b);
    }
}

// Any n, the whole CTA: a radix select on the span of the keys: 256 buckets, then the bucket of
// the m-th largest in 256 again, until it is taken whole or holds one value. Scores of real pages take
// two rounds.
template <int kThreads, typename F>
__device__ __noinline__ void pick(const unsigned long long* key, int n, int m, PickSmem& S, F&& emit) {
    constexpr int kWarps = kThreads / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (n <= 256) {
        if (warp == 0) pick_warp<8>(key, n, m, emit);
        __syncthreads();
        return;
    }
    unsigned long long lo = ~0ull, hi = 0;
    for (int i = tid; i < n; i += kThreads) {
        lo = min(lo, key[i]);
        hi = max(hi, key[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (lane == 0) {
        S.lo[warp] = lo;
        S.hi[warp] = hi;
    }
    for (int i = tid; i < 256; i += kThreads) S.hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        lo = min(lo, S.lo[w]);
        hi = max(hi, S.hi[w]);
    }
    // the wanted key lies in [lo, lo + 2^bits); 'need' of the keys there are taken, and all above
    int bits = hi == lo ? 0 : 64 - __clzll(static_cast<long long>(hi - lo)), need = m;
    while (bits > 0) {
        const int shift = max(0, bits - 8);
        for (int i = tid; i < n; i += kThreads) {
            const unsigned long long d = key[i] - lo;
            if (key[i] >= lo && (bits == 64 || d >> bits == 0)) atomicAdd(&S.hist[d >> shift], 1);
        }
        __syncthreads();
        if (warp == 0) {  // 8 buckets a lane, the highest first
            int c[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                c[i] = S.hist[255 - lane * 8 - i];
                S.hist[255 - lane * 8 - i] = 0;
                sum += c[i];
            }
            int x = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            int before = x - sum;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (before < need && need <= before + c[i]) {
                    S.bucket = 255 - lane * 8 - i;
                    S.above = before;
                    S.count[0] = c[i];
                }
                before += c[i];
            }
        }
        __syncthreads();
        lo += static_cast<unsigned long long>(S.bucket) << shift;
        need -= S.above;
        bits = shift;
        if (S.count[0] == need) break;  // the bucket is taken whole
        // the next round's atomics come after every thread has read this one's answer
        __syncthreads();
    }
    // taken: keys of [lo, lo + 2^bits) and above, of the equal ones (bits == 0) the first 'need'
    __syncthreads();
    const int per = (n + kThreads - 1) / kThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    const auto inside = [&](unsigned long long k) { return k >= lo && (bits == 64 || (k - lo) >> bits == 0); };
    int sure = 0, maybe = 0;
    for (int i = i0; i < i1; ++i) {
        const bool in = inside(key[i]);
        maybe += in;
        sure += key[i] >= lo && !in;
    }
    int x = sure | maybe << 16;  // at most 16384 of each
    const int mine = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) S.count[warp] = x;
    __syncthreads();
    int before = x - mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
        if (w < warp) before += S.count[w];
    int in_before = before >> 16, at = (before & 0xffff) + min(in_before, need);
    for (int i = i0; i < i1; ++i) {
        const unsigned long long k = key[i];
        if (k < lo) continue;
        const bool in = inside(k);
        if (!in || in_before < need) emit(i, at++);
        in_before += in;
    }
    __syncthreads();
}

// Sums of products in two fp32 words: s the plain sum, c what its roundings and the products'
// lost, each found exactly (the error of a product by fma, of a sum by Knuth's two-sum). As good as a sum in
// twice the precision, off by at most a few 2^-40 of the terms' sum: two pages are told apart, and
// pages of equal bounds are equal. (fp64 sums would want every element converted, which kept the
// conversion pipe busy 99 % of the time where many rows are scored.)
struct Sum2 {
    float s = 0.f, c = 0.f;
};
// a += x + rest, the same whichever of the two is a: where a page stands does not change its sum.
__device__ __forceinline__ void add_exact(Sum2& a, float x, float rest) {
    const float t = __fadd_rn(a.s, x), z = __fsub_rn(t, a.s);
    const float lost = __fadd_rn(__fsub_rn(a.s, __fsub_rn(t, z)), __fsub_rn(x, z));
    a.s = t;
    a.c = __fadd_rn(__fadd_rn(a.c, rest), lost);
}
// a += (hi + lo) x
__device__ __forceinline__ void add_product(Sum2& a, float hi, float lo, float x) {
    const float p = __fmul_rn(hi, x);
    add_exact(a, p, __fmaf_rn(lo, x, __fmaf_rn(hi, x, -p)));
}
__device__ __forceinline__ Sum2 shuffle_xor(const Sum2 v, int o) {
    Sum2 r;
    r.s = __shfl_xor_sync(0xffffffffu, v.s, o);
    r.c = __shfl_xor_sync(0xffffffffu, v.c, o);
    return r;
}

// s becomes the sum rounded once, c what that leaves (terms of one sign: |c| < |s|; infinities and NaN stay).
__device__ __forceinline__ void settle(Sum2& a) {
    const float t = __fadd_rn(a.s, a.c);
    if (!isfinite(t)) return;
    a.c = __fsub_rn(a.c, __fsub_rn(t, a.s));
    a.s = t;
}

// Sums of kN values per lane over kLanes neighbouring lanes, halving the values with the
// lanes: value j's sum ends on the lanes whose upper bits spell j.
template <int kN, int kLanes>
__device__ __forceinline__ Sum2 spread_sum(Sum2 (&s)[kN], int l) {
    static_assert(kN <= kLanes);
    int o = kLanes / 2;
#pragma unroll
    for (int n = kN / 2; n > 0; n >>= 1, o >>= 1) {
        const bool up = (l & o) != 0;
#pragma unroll
        for (int j = 0; j < n; ++j) {
            const Sum2 give = up ? s[j] : s[n + j], got = shuffle_xor(give, o);
            s[j] = up ? s[n + j] : s[j];
            add_exact(s[j], got.s, got.c);
        }
    }
#pragma unroll
    for (int x = kLanes / kN / 2; x > 0; x >>= 1) {
        const Sum2 got = shuffle_xor(s[0], x);
        add_exact(s[0], got.s, got.c);
    }
    return s[0];
}

template <int kN, int kLanes>
__device__ __forceinline__ float spread_sum1(float (&s)[kN], int l) {
    int o = kLanes / 2;
#pragma unroll
    for (int n = kN / 2; n > 0; n >>= 1, o >>= 1) {
        const bool up = (l & o) != 0;
#pragma unroll
        for (int j = 0; j < n; ++j) {
            const float give = up ? s[j] : s[n + j], keep = up ? s[n + j] : s[j];
            s[j] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
#pragma unroll
    for (int x = kLanes / kN / 2; x > 0; x >>= 1) s[0] += __shfl_xor_sync(0xffffffffu, s[0], x);
    return s[0];
}

// A weight of a dimension in which no head looks at that bound: its product with an infinite bound counts as 0. (A
// weight of 0 because of a head's 0 gives NaN with infinity, as that head's own product does.)
constexpr float kNoHead = -0.f;
__device__ __forceinline__ bool no_head(float w) { return __float_as_uint(w) == 0x80000000u; }

// Scores of the n pages in table[] (those numbered list[0, n), where there is a list), as order keys. w: the 2 D weights in the bounds' layout, written before by
// other threads: the wait for them comes after the first page ids are on their way. Each warp
// has kAhead loads of 512 bytes in flight.
template <typename T, int D, int kWarps>
__device__ __noinline__ void score_pages(const Args& g, const int* table, const int* list, int n, size_t plane, int head, const Sum2* w,
                            unsigned long long* key) {
    constexpr int kVec = 16 / sizeof(T), kNum = 2 * D / kVec;  // 16-byte pieces of a page's bounds
    constexpr int kLanes = kNum < 32 ? kNum : 32, kRep = kNum / kLanes, kPages = 32 / kLanes, kAhead = (sizeof(T) == 4 ? 16 : 8) / kRep;
    constexpr int kStep = kWarps * kPages * kAhead;
    const vxc_pages& p = g.p;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % kLanes, sub = lane / kLanes;
    const char* base = static_cast<const char*>(p.bounds) + (plane * p.kv_heads + head) * (2 * D * sizeof(T)) + l * 16;
    const size_t stride = static_cast<size_t>(p.kv_heads) * (2 * D * sizeof(T));
    int id[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
        const int i = (warp * kAhead + j) * kPages + sub;
        id[j] = i < n ? table[list ? list[i] : i] : -1;
    }
    __syncthreads();
    float hi[kRep * kVec], lo[kRep * kVec];
#pragma unroll
    for (int r = 0; r < kRep; ++r)
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            hi[r * kVec + i] = w[(r * kLanes + l) * kVec + i].s;
            lo[r * kVec + i] = w[(r * kLanes + l) * kVec + i].c;
        }
    for (int i0 = warp * kPages * kAhead; i0 < n; i0 += kStep) {
        uint4 v[kAhead][kRep];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
#pragma unroll
            for (int r = 0; r < kRep; ++r)
                v[j][r] = id[j] >= 0 && id[j] < p.n_pages ? ld16(base + id[j] * stride + r * kLanes * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = i0 + kStep + j * kPages + sub;
            id[j] = i < n ? table[list ? list[i] : i] : -1;
        }
        Sum2 s[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
#pragma unroll
            for (int r = 0; r < kRep; ++r) {
                float x[kVec];
                unpack16<T>(v[j][r], x);
#pragma unroll
                for (int i = 0; i < kVec; ++i) add_product(s[j], hi[r * kVec + i], lo[r * kVec + i], x[i]);
            }
        }
        Sum2 sum = spread_sum<kAhead, kLanes>(s, l);
        if (__any_sync(0xffffffffu, !isfinite(sum.s))) {
            // infinite bounds: once more, in the same order, without those that no head looks at
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int i = i0 + j * kPages + sub;
                const int page = i < n ? table[list ? list[i] : i] : -1;
                s[j] = Sum2{};
#pragma unroll
                for (int r = 0; r < kRep; ++r) {
                    float x[kVec];
                    unpack16<T>(page >= 0 && page < p.n_pages ? ld16(base + page * stride + r * kLanes * 16) : make_uint4(0, 0, 0, 0), x);
#pragma unroll
                    for (int e = 0; e < kVec; ++e)
                        add_product(s[j], hi[r * kVec + e], lo[r * kVec + e], no_head(hi[r * kVec + e]) && fabsf(x[e]) == INFINITY ? 0.f : x[e]);
                }
            }
            sum = spread_sum<kAhead, kLanes>(s, l);
        }
        const int i = i0 + l / (kLanes / kAhead) * kPages + sub;
        if (l % (kLanes / kAhead) == 0 && i < n) key[i] = order_key(sum.s, sum.c);
    }
    __syncthreads();
}

// The same scores as plain fp32 sums to near[], with what bounds their error: the scores of pages
// dealt to this warp are off by at most *err (written by lane 0). A sum of 2 D products in this order takes at
// most 4 + 1 + 5 roundings, the weights one (settle), so 2^-20 of the terms' absolute sum covers it; that
// sum is bounded by the lanes' weights and the largest element that each has met.
template <typename T, int D, int kWarps>
__device__ void near_scores(const Args& g, const int* table, int n, size_t plane, int head, const Sum2* w, float* near,
                            float* err) {
    constexpr int kVec = 16 / sizeof(T), kNum = 2 * D / kVec;
    constexpr int kLanes = kNum < 32 ? kNum : 32, kRep = kNum / kLanes, kPages = 32 / kLanes, kAhead = 8 / kRep;
    constexpr int kStep = kWarps * kPages * kAhead;
    const vxc_pages& p = g.p;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % kLanes, sub = lane / kLanes;
    const char* base = static_cast<const char*>(p.bounds) + (plane * p.kv_heads + head) * (2 * D * sizeof(T)) + l * 16;
    const size_t stride = static_cast<size_t>(p.kv_heads) * (2 * D * sizeof(T));
    int id[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
        const int i = (warp * kAhead + j) * kPages + sub;
        id[j] = i < n ? table[i] : -1;
    }
    __syncthreads();
    float2 wr[kRep][kVec / 2];
    float total[kRep];
#pragma unroll
    for (int r = 0; r < kRep; ++r) {
        total[r] = 0.f;
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) {
            const int at = (r * kLanes + l) * kVec + 2 * i;
            wr[r][i] = make_float2(w[at].s, w[at + 1].s);
            total[r] += fabsf(wr[r][i].x) + fabsf(wr[r][i].y);
        }
    }
    float most[kRep];
    uint32_t big[kRep][4];
#pragma unroll
    for (int r = 0; r < kRep; ++r) {
        most[r] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) big[r][i] = 0;
    }
    for (int i0 = warp * kPages * kAhead; i0 < n; i0 += kStep) {
        uint4 v[kAhead][kRep];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
#pragma unroll
            for (int r = 0; r < kRep; ++r)
                v[j][r] = id[j] >= 0 && id[j] < p.n_pages ? ld16(base + id[j] * stride + r * kLanes * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = i0 + kStep + j * kPages + sub;
            id[j] = i < n ? table[i] : -1;
        }
        float s[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            float2 a = make_float2(0.f, 0.f);
#pragma unroll
            for (int r = 0; r < kRep; ++r) {
                float2 x[kVec / 2];
                unpack_pairs<T>(v[j][r], x);
#pragma unroll
                for (int i = 0; i < kVec / 2; ++i) a = __ffma2_rn(wr[r][i], x[i], a);
                const uint32_t raw[4] = {v[j][r].x, v[j][r].y, v[j][r].z, v[j][r].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) big[r][i] = most_abs<T>(big[r][i], raw[i]);
            }
            s[j] = a.x + a.y;
        }
        const float sum = spread_sum1<kAhead, kLanes>(s, l);
        const int i = i0 + l / (kLanes / kAhead) * kPages + sub;
        if (l % (kLanes / kAhead) == 0 && i < n) near[i] = sum;
    }
    float e = 0.f;
#pragma unroll
    for (int r = 0; r < kRep; ++r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) most[r] = max_nan(most[r], largest<T>(big[r][i]));
        e += total[r] * most[r];
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) e += __shfl_xor_sync(0xffffffffu, e, o);
    if (kPages == 2) e = max_nan(e, __shfl_xor_sync(0xffffffffu, e, 16));
    if (lane == 0) *err = e * 0x1p-20f;
}

// Which of n <= 512 pages are the m best (0 < m < n), from near scores that are off by at most err, as a
// bit mask: words [n / 32 + 1] to mask[]. With t the m-th largest near score, whoever is above t + 2 err is
// among the best, whoever is below t - 2 err is not, and if no more than the rest of m lie
// between, all of them are. Otherwise these are listed (their number is returned, how many of
// them to take goes to *need) for a look at their full scores. One warp.
constexpr int kNear = 512;
template <int kEach>  // n <= 32 kEach
__device__ int pick_near(const float* near, int n, int m, float err, uint32_t* mask, int* list, int* need) {
    const int lane = threadIdx.x & 31;
    uint32_t k[kEach], least = ~0u, most = 0;  // as integers of the same order; a NaN comes with an infinite err
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const bool in = i * 32 + lane < n;
        const uint32_t b = in ? __float_as_uint(near[i * 32 + lane]) : 0u;
        k[i] = in ? (b >> 31 ? ~b : b | 0x80000000u) : 0u;
        if (in) {
            least = min(least, k[i]);
            most = max(most, k[i]);
        }
    }
    uint32_t lo = __reduce_min_sync(0xffffffffu, least), hi = __reduce_max_sync(0xffffffffu, most);
    const bool finite = lo > 0x007fffffu && hi < 0xff800000u;
    while (lo < hi) {  // at least m keys >= lo, fewer than m > hi
        const uint32_t mid = hi - (hi - lo) / 2;
        int c = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) c += k[i] >= mid;
        c = __reduce_add_sync(0xffffffffu, c);
        if (c >= m) lo = mid;
        else hi = mid - 1;
        if (c == m) break;
    }
    uint32_t t = ~0u;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        if (k[i] >= lo) t = min(t, k[i]);
    t = __reduce_min_sync(0xffffffffu, t);
    const float at = __uint_as_float(t >> 31 ? t & 0x7fffffffu : ~t);
    const bool known = finite && err < INFINITY;
    const float up = known ? __fadd_ru(at, 2.f * err) : INFINITY, down = known ? __fsub_rd(at, 2.f * err) : -INFINITY;
    int sure = 0, between = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const float x = __uint_as_float(k[i] >> 31 ? k[i] & 0x7fffffffu : ~k[i]);
        const bool in = i * 32 + lane < n, above = in && known && x > up, maybe = in && !above && !(known && x < down);
        const uint32_t a = __ballot_sync(0xffffffffu, above), b = __ballot_sync(0xffffffffu, maybe);
        if (lane == 0 && i * 32 < n) mask[i] = a;
        if (maybe) list[between + __popc(b & ((1u << lane) - 1))] = i * 32 + lane;
        sure += __popc(a);
        between += __popc(b);
    }
    __syncwarp();
    *need = m - sure;
    if (between != m - sure) return between;
    for (int i = lane; i < between; i += 32) atomicOr(mask + list[i] / 32, 1u << (list[i] & 31));
    __syncwarp();
    return 0;
}

// ------------------------------------------------------------------ attention of one warp
// The tiles of the picked pages in order; the last page holds only the keys up to the row's.
struct Tiles {
    const int* id;    // [take] page ids, -1 = refused
    int per_page;     // tiles of a page
    int count;        // all tiles
    int last_keys;    // keys of the last tile
};

template <bool kBf16>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
    if constexpr (kBf16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
template <int N>
__device__ __forceinline__ void clear(uint32_t (&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = 0;
}

// Partial outputs [head][out_row]: 4 elements more than a head, for the banks.
template <int D>
constexpr int out_row() { return D + 4; }

// fp16 and bf16: S^T (16 keys x 8 heads) = K Q^T, O^T (16 elements x 8 heads) += V^T P^T.
// Weights are split into two 16-bit pieces, so that rounding them does not add to the output's
// own rounding. kGroups: 8-head column groups. Writes (max, sum, sum of weighted values) of each
// head to m[], l[], o[head][D].
template <typename T, int D, int kGroups>
__device__ void attend16(const T* q, int G, const T* k0, const T* v0, size_t page_stride, const Tiles& tiles, int first,
                         int step, float scale, float* m_out, float* l_out, float* o_out) {
    constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
    constexpr int kAhead = D == 64 ? 2 : 1;  // tiles whose loads are in flight together (64 registers)
    const int lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
    const float to2 = scale * 1.4426950408889634f;  // weights are powers of 2
    // fp16 weights are kept 2^15 times as large, below its largest number: at most 1, they would lose what lies under
    // 2^-25 of the largest, which thousands of keys can add up to
    constexpr float kLift = kBf16 ? 0.f : 15.f;
    uint4 qf[kGroups][D / 32];  // of each 64 elements, a lane's 16: two pieces of 8
#pragma unroll
    for (int n = 0; n < kGroups; ++n)
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
            qf[n][c] = n * 8 + g8 < G ? ld16(q + (n * 8 + g8) * D + (c / 2) * 64 + t4 * 16 + (c % 2) * 8) : make_uint4(0, 0, 0, 0);
    float o[kGroups][D / 16][4], mx[kGroups][2], ref[kGroups][2], sum[kGroups][2];  // ref: mx once there is one
#pragma unroll
    for (int n = 0; n < kGroups; ++n) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][j][i] = 0.f;
        mx[n][0] = mx[n][1] = -INFINITY;
        ref[n][0] = ref[n][1] = 0.f;
        sum[n][0] = sum[n][1] = 0.f;
    }
    for (int tile0 = first * kAhead; tile0 < tiles.count; tile0 += step * kAhead) {
        uint32_t kr[kAhead][2][D / 64][8], vr[kAhead][2][D / 64][8];  // [keys 0-7, 8-15][64 elements]
        int keys[kAhead];  // valid keys of the tile
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int tile = tile0 + a, page = tile / tiles.per_page;
            const int id = tile < tiles.count ? tiles.id[page] : -1;
            keys[a] = id < 0 ? 0 : tile == tiles.count - 1 ? tiles.last_keys : kTile;
            const size_t at = static_cast<size_t>(max(id, 0)) * page_stride + (tile - page * tiles.per_page) * (kTile * D);
            const T *kp = k0 + at, *vp = v0 + at;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < D / 64; ++c)
                    if (id >= 0) ld32(kp + (h * 8 + g8) * D + c * 64 + t4 * 16, kr[a][h][c]);
                    else clear(kr[a][h][c]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < D / 64; ++c)
                    if (h * 8 + g8 < keys[a]) ld32(vp + (h * 8 + g8) * D + c * 64 + t4 * 16, vr[a][h][c]);
                    else clear(vr[a][h][c]);
        }
        float s[kGroups][kAhead][4], top[kGroups][2];
#pragma unroll
        for (int n = 0; n < kGroups; ++n) {
            top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][a][i] = 0.f;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    const uint32_t *lo = kr[a][0][c / 2] + c % 2 * 4, *hi = kr[a][1][c / 2] + c % 2 * 4;
                    mma16<kBf16>(s[n][a], lo[0], hi[0], lo[1], hi[1], qf[n][c].x, qf[n][c].y);
                    mma16<kBf16>(s[n][a], lo[2], hi[2], lo[3], hi[3], qf[n][c].z, qf[n][c].w);
                }
                if (keys[a] < kTile) {
                    if (g8 >= keys[a]) s[n][a][0] = s[n][a][1] = -INFINITY;
                    if (g8 + 8 >= keys[a]) s[n][a][2] = s[n][a][3] = -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) top[n][i & 1] = fmaxf(top[n][i & 1], s[n][a][i]);
            }
        }
        // a new maximum is shared by the 8 lanes of a head; rare after the first tiles
        bool grows = false;
#pragma unroll
        for (int n = 0; n < kGroups; ++n) grows |= top[n][0] > mx[n][0] || top[n][1] > mx[n][1];
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
            for (int n = 0; n < kGroups; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = fmaxf(top[n][e], mx[n][e]);
#pragma unroll
                    for (int b = 4; b < 32; b <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, b));
                    const float fix = x == -INFINITY ? 1.f : exp2_fast((mx[n][e] - x) * to2);
                    mx[n][e] = x;
                    ref[n][e] = x == -INFINITY ? 0.f : x;
                    sum[n][e] *= fix;
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        o[n][j][e] *= fix;
                        o[n][j][e + 2] *= fix;
                    }
                }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            uint32_t hi[kGroups][2], lo[kGroups][2];
#pragma unroll
            for (int n = 0; n < kGroups; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        // 0 for masked keys and scores of -infinity
                        w[e] = exp2_fast(fmaf(s[n][a][2 * h + e] - ref[n][e], to2, kLift));
                        sum[n][e] += w[e];
                    }
                    const uint32_t big = pack2<T>(w[0], w[1]);
                    const float2 back = unpack2<T>(big);
                    hi[n][h] = transpose8(big);
                    lo[n][h] = transpose8(pack2<T>(w[0] - back.x, w[1] - back.y));
                }
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                // 8 keys x 8 elements each, turned: keys become the columns
                const uint32_t *x = vr[a][0][j / 4] + j % 4 * 2, *y = vr[a][1][j / 4] + j % 4 * 2;
                const uint32_t a0 = transpose8(x[0]), a1 = transpose8(x[1]), a2 = transpose8(y[0]), a3 = transpose8(y[1]);
#pragma unroll
                for (int n = 0; n < kGroups; ++n) {
                    mma16<kBf16>(o[n][j], a0, a1, a2, a3, hi[n][0], hi[n][1]);
                    mma16<kBf16>(o[n][j], a0, a1, a2, a3, lo[n][0], lo[n][1]);
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < kGroups; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int b = 4; b < 32; b <<= 1) sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], b);
            const int h = n * 8 + 2 * t4 + e;
            if (h >= G) continue;
            if (g8 == 0) {
                m_out[h] = mx[n][e] == -INFINITY ? -INFINITY : mx[n][e] * scale;
                l_out[h] = sum[n][e];
            }
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {  // rows g8 and g8 + 8 of block j: elements of lane g8 / 2's sixteen
                float* to = o_out + h * out_row<D>() + (j / 4) * 64 + (g8 >> 1) * 16 + (j % 4) * 4 + (g8 & 1);
                to[0] = o[n][j][e];
                to[2] = o[n][j][e + 2];
            }
        }
}

// fp32 on the CUDA cores (the matrix units' fp32 sums are cut, not rounded, and their tf32
// products short: neither keeps fp32 results). Scores: 8 key rows x 4 lanes, a lane holding a quarter of
// each of 4 keys. Values: a lane holds 4 elements of the outputs of all heads. A tile pair's
// values are summed by themselves before they join the total, which keeps chains short.
template <int D, int kHeads>
__device__ void attend32(const float* q_s, int G, const float* k0, const float* v0, size_t page_stride, const Tiles& tiles,
                         int first, int step, float scale, float* w_s, float* m_out, float* l_out, float* o_out) {
    constexpr int kPart = kHeads / 4;          // heads whose scores a lane ends up with
    constexpr int kVLanes = D / 4, kVKeys = 32 / kVLanes;  // lanes per key row of values, rows at once
    const int lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3, vl = lane % kVLanes, vk = lane / kVLanes;
    float2 o[kHeads][2];
    float mx[kPart], sum[kPart];
#pragma unroll
    for (int h = 0; h < kHeads; ++h) o[h][0] = o[h][1] = make_float2(0.f, 0.f);
#pragma unroll
    for (int h = 0; h < kPart; ++h) {
        mx[h] = -INFINITY;
        sum[h] = 0.f;
    }
    for (int tile0 = first * 2; tile0 < tiles.count; tile0 += step * 2) {
        const float *kp[2], *vp[2];
        int keys[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int tile = tile0 + a, page = tile / tiles.per_page;
            const int id = tile < tiles.count ? tiles.id[page] : -1;
            keys[a] = id < 0 ? 0 : tile == tiles.count - 1 ? tiles.last_keys : kTile;
            const size_t at = static_cast<size_t>(max(id, 0)) * page_stride + (tile - page * tiles.per_page) * (kTile * D);
            kp[a] = k0 + at;
            vp[a] = v0 + at;
        }
        // the values' first rows leave together with the keys
        constexpr int kRows = kVKeys == 2 ? 8 : 4;  // of 32 keys: 2 or 8 batches
        uint4 vr[kRows];
        const auto fetch = [&](int j0) {
#pragma unroll
            for (int j = 0; j < kRows; ++j) {
                const int key = j0 + j * kVKeys + vk;
                vr[j] = (key & 15) < keys[j0 >> 4] ? ld16(vp[j0 >> 4] + (key & 15) * D + vl * 4) : make_uint4(0, 0, 0, 0);
            }
        };
        float s[kHeads][4];  // key g8 + 8 (i & 1) of tile i >> 1
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[h][i] = 0.f;
#pragma unroll
        for (int c0 = 0; c0 < D / 16; c0 += 4) {
            uint32_t kr[2][4][8];  // 32 elements of a key by 4 lanes, 8 each
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (g8 + 8 * (i & 1) < keys[i >> 1]) ld32(kp[i >> 1] + (g8 + 8 * (i & 1)) * D + c0 * 16 + c * 32 + t4 * 8, kr[c][i]);
                    else clear(kr[c][i]);
            if (c0 == 0) fetch(0);
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int h = 0; h < kHeads; ++h) {
                    const float4 q = *reinterpret_cast<const float4*>(q_s + h * D + c0 * 16 + (c / 2) * 32 + t4 * 8 + (c % 2) * 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t* k = kr[c / 2][i] + (c % 2) * 4;
                        s[h][i] = fmaf(q.x, __uint_as_float(k[0]), s[h][i]);
                        s[h][i] = fmaf(q.y, __uint_as_float(k[1]), s[h][i]);
                        s[h][i] = fmaf(q.z, __uint_as_float(k[2]), s[h][i]);
                        s[h][i] = fmaf(q.w, __uint_as_float(k[3]), s[h][i]);
                    }
                }
        }
        // sums over the 4 lanes; lane t4 keeps heads [t4 kPart, + kPart)
        float r[kPart][4], fix[kPart];
        const bool up1 = (t4 & 2) != 0, up0 = (t4 & 1) != 0;
#pragma unroll
        for (int h = 0; h < kPart; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = (up1 ? s[2 * kPart + h][i] : s[h][i]) +
                                __shfl_xor_sync(0xffffffffu, up1 ? s[h][i] : s[2 * kPart + h][i], 2);
                const float b = (up1 ? s[3 * kPart + h][i] : s[kPart + h][i]) +
                                __shfl_xor_sync(0xffffffffu, up1 ? s[kPart + h][i] : s[3 * kPart + h][i], 2);
                const float x = (up0 ? b : a) + __shfl_xor_sync(0xffffffffu, up0 ? a : b, 1);
                r[h][i] = g8 + 8 * (i & 1) < keys[i >> 1] ? x * scale : -INFINITY;
            }
        __syncwarp();  // the weights of the tiles before have been read
#pragma unroll
        for (int h = 0; h < kPart; ++h) {
            float x = fmaxf(fmaxf(r[h][0], r[h][1]), fmaxf(r[h][2], r[h][3]));
#pragma unroll
            for (int b = 4; b < 32; b <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, b));
            x = fmaxf(x, mx[h]);
            fix[h] = x == -INFINITY ? 1.f : expf(mx[h] - x);
            mx[h] = x;
            sum[h] *= fix[h];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w = expf(r[h][i] - (x == -INFINITY ? 0.f : x));  // 0 for masked keys and scores of -infinity
                sum[h] += w;
                w_s[(g8 + 8 * i) * kHeads + t4 * kPart + h] = w;
            }
        }
        __syncwarp();
        float2 part[kHeads][2];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) part[h][0] = part[h][1] = make_float2(0.f, 0.f);
#pragma unroll
        for (int j0 = 0; j0 < 32; j0 += kRows * kVKeys) {
            uint4 now[kRows];
#pragma unroll
            for (int j = 0; j < kRows; ++j) now[j] = vr[j];
            if (j0 + kRows * kVKeys < 32) fetch(j0 + kRows * kVKeys);
#pragma unroll
            for (int j = 0; j < kRows; ++j) {
                const int key = j0 + j * kVKeys + vk;
                const float2 v0 = make_float2(__uint_as_float(now[j].x), __uint_as_float(now[j].y));
                const float2 v1 = make_float2(__uint_as_float(now[j].z), __uint_as_float(now[j].w));
#pragma unroll
                for (int h = 0; h < kHeads; h += 4) {
                    const float4 w = *reinterpret_cast<const float4*>(w_s + key * kHeads + h);
                    const float ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        part[h + e][0] = __ffma2_rn(make_float2(ww[e], ww[e]), v0, part[h + e][0]);
                        part[h + e][1] = __ffma2_rn(make_float2(ww[e], ww[e]), v1, part[h + e][1]);
                    }
                }
            }
        }
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            const float f = __shfl_sync(0xffffffffu, fix[h % kPart], h / kPart);
#pragma unroll
            for (int i = 0; i < 2; ++i) o[h][i] = __ffma2_rn(o[h][i], make_float2(f, f), part[h][i]);
        }
    }
#pragma unroll
    for (int h = 0; h < kPart; ++h) {
#pragma unroll
        for (int b = 4; b < 32; b <<= 1) sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], b);
        if (g8 == 0 && t4 * kPart + h < G) {
            m_out[t4 * kPart + h] = mx[h];
            l_out[t4 * kPart + h] = sum[h];
        }
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
        if (kVKeys == 2) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                o[h][i].x += __shfl_xor_sync(0xffffffffu, o[h][i].x, 16);
                o[h][i].y += __shfl_xor_sync(0xffffffffu, o[h][i].y, 16);
            }
        }
        if (h < G && vk == 0) store4(o_out + h * out_row<D>() + vl * 4, o[h][0].x, o[h][0].y, o[h][1].x, o[h][1].y);
    }
}

// A second look at outputs that the sums left as NaN although the head's sum of weights is a number: of this thread's
// items in the last loop of sparse_kernel (4 elements of a head each) those in the bit mask. The sums turn an infinite value into NaN
// where its weight was split (into pieces of either sign, or 0), fell below what fp32 holds, or was scaled down to 0
// by a later maximum, though any weight but that of a score of -infinity is positive. The values decide: infinities
// of one sign are that, of both NaN; no weight times infinity is NaN. No score is NaN or +infinity here, so a key with
// an element that is not finite (its page's bounds tell) has the score -infinity. One thread's walk over the row's
// values per item; only rows that have infinite ones take it.
// (Everything but the page ids is looked up again, so that no register is kept for it.)
template <typename T, int D>
__device__ __noinline__ void past_numbers(const Args& g, const int* ids, unsigned mask) {
    const vxc_pages& p = g.p;
    const int P = p.page_size, G = g.a.q_heads / p.kv_heads, item = blockIdx.x / g.cluster;
    const int r = item / p.kv_heads, head = item - r * p.kv_heads, pos = g.a.row_pos[r];
    const int take = min(pos / P + 1, g.a.top_pages), last = pos % P + 1;
    const size_t page0 = (static_cast<size_t>(g.layer) * p.n_pages) * p.kv_heads + head;
    T* out = static_cast<T*>(g.a.out) + static_cast<size_t>(r) * g.a.out_stride + static_cast<size_t>(head) * G * D;
    int i = blockIdx.x % g.cluster * blockDim.x + threadIdx.x;
    for (; mask != 0; i += g.cluster * blockDim.x, mask >>= 1) {
        if (!(mask & 1)) continue;
        const int h = i / (D / 4), d = (i - h * (D / 4)) * 4;
        float extra[4] = {};
        for (int j = 0; j < take; ++j) {
            if (ids[j] < 0) continue;
            const size_t page = page0 + static_cast<size_t>(ids[j]) * p.kv_heads;
            const T *k = static_cast<const T*>(p.k) + page * P * D, *v = static_cast<const T*>(p.v) + page * P * D + d;
            const T* b = static_cast<const T*>(p.bounds) + page * 2 * D;
            const int keys = j == take - 1 ? last : P;
            bool looked = false, odd = false;  // whether a key of the page is not finite
#pragma unroll 8
            for (int t = 0; t < keys; ++t) {
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = to_f(v[t * D + e]);
                if (isfinite(x[0]) && isfinite(x[1]) && isfinite(x[2]) && isfinite(x[3])) continue;
                if (!looked)
                    for (int e = 0; e < 2 * D; ++e) odd |= !isfinite(to_f(b[e]));
                looked = true;
                bool none = false;
                if (odd)
                    for (int e = 0; e < D; ++e) none |= !isfinite(to_f(k[t * D + e]));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!isfinite(x[e])) extra[e] += none ? NAN : x[e];
            }
            if (extra[0] != extra[0] && extra[1] != extra[1] && extra[2] != extra[2] && extra[3] != extra[3]) break;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            T* y = out + h * D + d + e;
            if (to_f(*y) != to_f(*y) && extra[e] == extra[e] && extra[e] != 0.f) *y = T(extra[e]);  // 0: the NaN has another cause
        }
    }
}

// ------------------------------------------------------------------ the kernel
// Dynamic shared memory, in this order (every part a multiple of 16 bytes):
//   o[kWarps][kHeads][D] partial outputs; (max, sum)[kWarps][2][kHeads]; joined o[kHeads][D], (max, sum)[2][kHeads];
//   fp32 only: q[kHeads][D], weights[kWarps][32][kHeads];
//   full scores[keys]; plain sums[near]
template <typename T, int D, int kHeads, int kWarps>
constexpr size_t fixed_smem() {
    size_t f = static_cast<size_t>(kWarps) * kHeads * out_row<D>() + kWarps * 2 * kHeads + kHeads * D + 2 * kHeads;
    if (sizeof(T) == 4) f += static_cast<size_t>(kHeads) * D + kWarps * 32 * kHeads;
    return f * 4;
}

// CTAs that an SM should hold by their registers: the phases of one CTA are chains of
// dependent steps, which others fill.
template <typename T, int D, int kHeads, int kWarps>
constexpr int resident_ctas() {
    const int warps = kHeads == 16 ? (sizeof(T) == 2 && D == 64 ? 12 : 8) : sizeof(T) == 4 ? 12 : D == 64 ? 20 : 16;
    return warps > kWarps ? warps / kWarps : 1;
}

template <typename T, int D, int kHeads, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, resident_ctas<T, D, kHeads, kWarps>()) sparse_kernel(const __grid_constant__ Args g) {
    constexpr int kThreads = kWarps * 32;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ Sum2 s_w[2 * D];
    __shared__ PickSmem s_pick;
    __shared__ int s_list[kMaxTop], s_id[kMaxTop], s_again[kNear];
    __shared__ uint32_t s_mask[kNear / 32];
    __shared__ float s_err[kWarps];
    float* s_o = reinterpret_cast<float*>(smem);
    float* s_ml = s_o + kWarps * kHeads * out_row<D>();
    float* s_fo = s_ml + kWarps * 2 * kHeads;
    float* s_fml = s_fo + kHeads * D;
    float* s_q = s_fml + 2 * kHeads;
    float* s_wt = s_q + kHeads * D;
    unsigned long long* key = reinterpret_cast<unsigned long long*>(smem + fixed_smem<T, D, kHeads, kWarps>());
    pdl_launch_dependents();
    pdl_wait();
    const vxc_pages& p = g.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, P = p.page_size, C = g.cluster;
    const int rank = blockIdx.x % C, item = blockIdx.x / C;
    const int r = item / p.kv_heads, head = item - r * p.kv_heads, G = g.a.q_heads / p.kv_heads;
    const T* q = static_cast<const T*>(g.a.q) + static_cast<size_t>(r) * g.a.q_stride + static_cast<size_t>(head) * G * D;
    const int seq = g.a.row_seq[r], pos = g.a.row_pos[r];
    // the heads' elements of this thread's dimensions, on their way while the row's place is looked up
    constexpr int kCols = (D + kThreads - 1) / kThreads;
    T column[kCols][kHeads];
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int h = 0; h < kHeads; ++h) column[c][h] = h < G && c * kThreads + tid < D ? q[h * D + c * kThreads + tid] : T(0.f);
    if (seq < 0) return;  // the whole cluster
    if (seq >= p.n_seqs || pos < 0 || pos >= p.max_pages * P) {
        if (tid == 0 && rank == 0) report(p.status, VXC_PAGES_BAD_ROW);
        return;
    }
    const int* table = p.table + static_cast<size_t>(seq) * p.max_pages;
    const size_t plane = static_cast<size_t>(g.layer) * p.n_pages;
    if constexpr (sizeof(T) == 4)
        for (int i = tid; i < kHeads * D; i += kThreads) s_q[i] = i < G * D ? q[i] : 0.f;
    const int seen = pos / P + 1, take = min(seen, g.a.top_pages);
    // ---- which pages
    if (seen <= take) {
        for (int i = tid; i < take; i += kThreads) s_list[i] = i;
    } else {
        const int sink = g.a.sink_pages, local = g.a.local_pages, n = seen - sink - local, m = take - sink - local;
        for (int i = tid; i < sink; i += kThreads) s_list[i] = i;
        for (int i = tid; i < local; i += kThreads) s_list[take - local + i] = seen - local + i;
        if (m > 0) {
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                const int d = c * kThreads + tid;
                Sum2 up, down;
                int zeros = G - kHeads;  // heads whose element is 0
#pragma unroll
                for (int h = 0; h < kHeads; ++h) {
                    const float x = to_f(column[c][h]);
                    add_exact(up, x > 0.f || x != x ? x : 0.f, 0.f);
                    add_exact(down, x < 0.f ? x : 0.f, 0.f);
                    zeros += x == 0.f;
                }
                settle(up);
                settle(down);
                if (zeros == 0) {  // see kNoHead
                    if (up.s == 0.f) up.s = kNoHead;
                    if (down.s == 0.f) down.s = kNoHead;
                }
                if (d < D) {
                    s_w[d] = down;
                    s_w[D + d] = up;
                }
            }
            const int parts = n <= kAlone ? 1 : C;  // CTAs that the pages are dealt to
            if (parts > 1) cluster_arrive();
            const int per = (n + parts - 1) / parts, i0 = min(n, rank * per), mine = min(n, i0 + per) - i0;
            if (parts == 1) {
                if (n > kNear) {
                    score_pages<T, D, kWarps>(g, table + sink, nullptr, n, plane, head, s_w, key);
                    pick<kThreads>(key, n, m, s_pick, [&](int i, int at) { s_list[sink + at] = sink + i; });
                } else {
                    // plain sums tell all but a few pages apart; those few are looked at again
                    float* near = reinterpret_cast<float*>(key + g.keys);
                    near_scores<T, D, kWarps>(g, table + sink, n, plane, head, s_w, near, s_err + warp);
                    __syncthreads();
                    if (warp == 0) {
                        float err = 0.f;
#pragma unroll
                        for (int w = 0; w < kWarps; ++w) err = max_nan(err, s_err[w]);
                        int need;
                        const int again = n <= 192 ? pick_near<6>(near, n, m, err, s_mask, s_again, &need)
                                                   : pick_near<kNear / 32>(near, n, m, err, s_mask, s_again, &need);
                        if (tid == 0) {
                            s_pick.bucket = again;
                            s_pick.above = need;
                        }
                    }
                    __syncthreads();
                    const int again = s_pick.bucket, need = s_pick.above;
                    if (again > 0) {
                        score_pages<T, D, kWarps>(g, table + sink, s_again, again, plane, head, s_w, key);
                        pick<kThreads>(key, again, need, s_pick,
                                       [&](int i, int) { atomicOr(s_mask + s_again[i] / 32, 1u << (s_again[i] & 31)); });
                    }
                    if (warp == 0) {
                        int at = sink;
                        for (int i = 0; i * 32 < n; ++i) {
                            const uint32_t b = s_mask[i];
                            if (b >> lane & 1) s_list[at + __popc(b & ((1u << lane) - 1))] = sink + i * 32 + lane;
                            at += __popc(b);
                        }
                    }
                }
            } else {
                // every CTA scores its part and hands it to the others; all of them pick alike
                score_pages<T, D, kWarps>(g, table + sink + i0, nullptr, mine, plane, head, s_w, key + i0);
                cluster_wait();  // all CTAs of the cluster run
                for (int c = 1; c < C; ++c) {
                    const uint32_t to = peer_addr(key + i0, (rank + c) % C);
                    for (int i = tid; i < mine; i += kThreads)
                        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + i * 8), "l"(key[i0 + i]) : "memory");
                }
                cluster_sync();
                pick<kThreads>(key, n, m, s_pick, [&](int i, int at) { s_list[sink + at] = sink + i; });
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < take; i += kThreads) {
        const int id = table[s_list[i]];
        const bool ok = id >= 0 && id < p.n_pages;
        s_id[i] = ok ? id : -1;
        if (!ok) report(p.status, VXC_PAGES_BAD_ID);
    }
    if (g.a.selected && rank == 0)
        for (int i = tid; i < g.a.top_pages; i += kThreads)
            g.a.selected[(static_cast<size_t>(r) * p.kv_heads + head) * g.a.top_pages + i] = i < take ? s_list[i] : -1;
    __syncthreads();
    // ---- attention of every warp over tiles of its own
    Tiles tiles;
    tiles.id = s_id;
    tiles.per_page = P / kTile;
    const int tail = pos - (seen - 1) * P;  // the last page's last key
    tiles.count = (take - 1) * tiles.per_page + tail / kTile + 1;
    tiles.last_keys = tail % kTile + 1;
    const size_t head_off = (plane * p.kv_heads + head) * static_cast<size_t>(P) * D;
    const size_t page_stride = static_cast<size_t>(p.kv_heads) * P * D;
    const T *k0 = static_cast<const T*>(p.k) + head_off, *v0 = static_cast<const T*>(p.v) + head_off;
    float *m_w = s_ml + warp * 2 * kHeads, *l_w = m_w + kHeads, *o_w = s_o + warp * kHeads * out_row<D>();
    if constexpr (sizeof(T) == 4)
        attend32<D, kHeads>(s_q, G, k0, v0, page_stride, tiles, rank * kWarps + warp, C * kWarps, g.scale,
                            s_wt + warp * 32 * kHeads, m_w, l_w, o_w);
    else
        attend16<T, D, kHeads / 8>(q, G, k0, v0, page_stride, tiles, rank * kWarps + warp, C * kWarps, g.scale, m_w, l_w, o_w);
    __syncthreads();
    // ---- the warps' parts, then the CTAs'; a part without keys has maximum -infinity and counts for nothing
    T* out = static_cast<T*>(g.a.out) + static_cast<size_t>(r) * g.a.out_stride + static_cast<size_t>(head) * G * D;
    unsigned odd = 0;  // this thread's outputs that need a second look
    const auto finish = [&](int h, int d, float L, const float (&x)[4], unsigned bit) {
        const float inv = L == 0.f ? 0.f : 1.f / L;  // 0: every page was refused, or every score is -infinity
        store4(out + h * D + d, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        const float any = (x[0] + x[1]) + (x[2] + x[3]);
        if (any != any && L == L && L != 0.f) odd |= bit;  // L is NaN: a score is, or is +infinity
    };
    unsigned bit = 1;
    for (int i = tid; i < G * (D / 4); i += kThreads, bit <<= 1) {
        const int h = i / (D / 4), d = (i - h * (D / 4)) * 4;
        float M = -INFINITY, L = 0.f, x[4] = {};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_ml[w * 2 * kHeads + h]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float l = s_ml[w * 2 * kHeads + kHeads + h], mw = s_ml[w * 2 * kHeads + h];
            const float f = l == 0.f ? 0.f : expf(mw - M);
            const float4 v = *reinterpret_cast<const float4*>(s_o + (w * kHeads + h) * out_row<D>() + d);
            L = fmaf(f, l, L);
            x[0] = fmaf(f, v.x, x[0]);
            x[1] = fmaf(f, v.y, x[1]);
            x[2] = fmaf(f, v.z, x[2]);
            x[3] = fmaf(f, v.w, x[3]);
        }
        if (C == 1) {
            finish(h, d, L, x, bit);
        } else {
            store4(s_fo + h * D + d, x[0], x[1], x[2], x[3]);
            if (d == 0) {
                s_fml[h] = M;
                s_fml[kHeads + h] = L;
            }
        }
    }
    if (C == 1) {
        if (odd) past_numbers<T, D>(g, s_id, odd);
        return;
    }
    cluster_sync();
    bit = 1;
    for (int i = rank * kThreads + tid; i < G * (D / 4); i += C * kThreads, bit <<= 1) {
        const int h = i / (D / 4), d = (i - h * (D / 4)) * 4;
        float M = -INFINITY, L = 0.f, x[4] = {}, mc[kMaxCluster];
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) {
            mc[c] = c < C ? peer_ld(s_fml + h, c) : -INFINITY;
            M = fmaxf(M, mc[c]);
        }
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) {
            if (c >= C) break;
            const float l = peer_ld(s_fml + kHeads + h, c), f = l == 0.f ? 0.f : expf(mc[c] - M);
            const float4 v = peer_ld4(s_fo + h * D + d, c);
            L = fmaf(f, l, L);
            x[0] = fmaf(f, v.x, x[0]);
            x[1] = fmaf(f, v.y, x[1]);
            x[2] = fmaf(f, v.z, x[2]);
            x[3] = fmaf(f, v.w, x[3]);
        }
        finish(h, d, L, x, bit);
    }
    if (odd) past_numbers<T, D>(g, s_id, odd);
    cluster_sync();  // no CTA ends while its part is being read
}

template <typename T, int D, int kHeads, int kWarps>
size_t dynamic_smem(int max_pages) {
    return fixed_smem<T, D, kHeads, kWarps>() + sizeof(unsigned long long) * (max_pages + (max_pages & 1)) +
           sizeof(float) * ((std::min(kNear, max_pages) + 3) & ~3);
}

template <typename T, int D, int kHeads, int kWarps>
void launch(Args g, long long items, cudaStream_t s) {
    const auto kernel = sparse_kernel<T, D, kHeads, kWarps>;
    paged_require(items * g.cluster <= 0x7fffffffll, "vxc_sparse_attention: too many rows");
    g.keys = g.p.max_pages + (g.p.max_pages & 1);
    g.near = (std::min(kNear, g.p.max_pages) + 3) & ~3;
    const size_t smem = dynamic_smem<T, D, kHeads, kWarps>(g.p.max_pages);
    allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem, "vxc_sparse_attention");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(items * g.cluster));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = g.cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g.cluster > 1 ? 2 : 1;
    paged_ck(cudaLaunchKernelEx(&cfg, kernel, g), "vxc_sparse_attention");
}

template <typename T, int D, int kHeads>
void launch_size(Args g, cudaStream_t s) {
    int dev = 0, sms = 0;
    paged_ck(cudaGetDevice(&dev), "cudaGetDevice");
    paged_ck(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
    // Many items: CTAs of 4 warps by themselves, several on an SM, fill one another's waits. Few: CTAs of
    // 8 warps, in clusters as large as still fit on the GPU at once (their registers let one or two
    // be on an SM; clusters of 8 leave SMs of a GPC unused where only one is), but no more warps than tile
    // pairs. Measured with 8 heads of 64 a KV head, 32 of 128 pages of 64, CTAs x warps (what the rule takes first).
    // f16: 2 items 8x8 9.5 us, 4x4 11.0; 16 items 8x8 11.3, 4x8 10.6; 64 items 4x8 15.5, 1x8 18.1; 256 items 1x8 21.4,
    // 1x4 28.4; 512 items 1x4 37.0, 1x8 37.4; 8 of 32 pages, 2 items: 4x4 7.6, 1x8 7.5. fp32: 2 items 8x8 11.6, 4x8
    // 13.6; 64 items 2x8 21.0, 4x8 30.2; 256 items 1x8 59.2, 1x4 70.9; 512 items 1x4 115.7, 2x4 112.0; 64 of 1024
    // pages, 16 items: 4x8 31.1, 8x8 43.5.
    const long long items = static_cast<long long>(g.a.rows) * g.p.kv_heads;
    constexpr int kResident = sizeof(T) == 4 || (D == 128 && kHeads == 16) ? 1 : 2;  // CTAs of 8 warps on an SM
    const int pairs = std::max(1, g.a.top_pages * g.p.page_size / kTile / 2), room = kResident * (sms - sms / 8);
    g.cluster = 1;
    // (8 warps' outputs of 16 wide fp32 heads do not fit beside the scores of the longest tables.)
    if (items > 2 * sms || dynamic_smem<T, D, kHeads, 8>(g.p.max_pages) > kDynamicLimit) {
        launch<T, D, kHeads, 4>(g, items, s);
        return;
    }
    const bool four = pairs <= 16 && items <= 32;
    while (g.cluster < kMaxCluster && g.cluster * 2 * (four ? 4 : 8) <= pairs &&
           items * g.cluster * 2 <= (kResident == 1 && g.cluster == 4 ? room / 2 : room))
        g.cluster *= 2;
    if (four) launch<T, D, kHeads, 4>(g, items, s);
    else launch<T, D, kHeads, 8>(g, items, s);
}

template <typename T, int D>
void launch_group(const Args& g, cudaStream_t s) {
    if (g.a.q_heads / g.p.kv_heads <= 8) launch_size<T, D, 8>(g, s);
    else launch_size<T, D, 16>(g, s);
}

void check_query(const vxc_sparse_query* a, const vxc_pages* p, int layer) {
    check_page_sizes(p);
    paged_require(a->rows > 0 && static_cast<int64_t>(a->rows) * p->kv_heads <= 0x7fffffff,
                  "vxc_sparse_attention: rows must be positive, rows x kv_heads below 2^31");
    paged_require(a->q_heads > 0 && a->q_heads % p->kv_heads == 0 && a->q_heads / p->kv_heads <= kMaxGroup,
                  "vxc_sparse_attention: q_heads must be a multiple of kv_heads, at most 16 per KV head");
    paged_require(a->top_pages >= 1 && a->top_pages <= kMaxTop, "vxc_sparse_attention: top_pages must be 1 to 256");
    paged_require(a->sink_pages >= 0 && a->local_pages >= 1 && a->sink_pages <= a->top_pages &&
                      a->local_pages <= a->top_pages - a->sink_pages,
                  "vxc_sparse_attention: sink_pages >= 0 and local_pages >= 1 must fit in top_pages");
    paged_require(a->scale >= 0.f && a->scale <= 3.4e38f, "vxc_sparse_attention: scale must be finite and not negative");
    paged_require(layer >= 0 && layer < p->layers, "vxc_sparse_attention: layer out of range");
    paged_require(a->q && a->out && a->row_seq && a->row_pos, "null argument");
    const int unit = 16 / dtype_size(p->dtype);
    const int64_t row = static_cast<int64_t>(a->q_heads) * p->head_dim;
    paged_require(aligned16(a->q) && aligned16(a->out) && aligned4(a->row_seq) && aligned4(a->row_pos) && aligned4(a->selected),
                  "vxc_sparse_attention: q and out must start on 16-byte boundaries");
    paged_require(a->q_stride >= row && a->out_stride >= row && a->q_stride % unit == 0 && a->out_stride % unit == 0,
                  "vxc_sparse_attention: strides must cover a row and be multiples of 16 bytes");
    check_page_arrays(p);
    DeviceMemory mem("vxc_sparse_attention");
    mem.require(a->q, "q");
    mem.require(a->out, "out");
    mem.require(a->row_seq, "row_seq");
    mem.require(a->row_pos, "row_pos");
    mem.require(a->selected, "selected");
    check_page_memory(p, mem);
}

}  // namespace
}  // namespace vxc

using namespace vxc;

extern "C" VXC_API int32_t vxc_sparse_attention(const vxc_sparse_query* a, const vxc_pages* p, int32_t layer,
                                                void* cuda_stream) {
    return paged_guard([&] {
        paged_require(a && p, "null argument");
        check_query(a, p, layer);
        Args g = {};
        g.a = *a;
        g.p = *p;
        g.layer = layer;
        g.scale = a->scale == 0.f ? 1.f / std::sqrt(static_cast<float>(p->head_dim)) : a->scale;
        const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
        const bool wide = p->head_dim == 128;
        if (p->dtype == VXC_F32) wide ? launch_group<float, 128>(g, cs) : launch_group<float, 64>(g, cs);
        else if (p->dtype == VXC_F16) wide ? launch_group<__half, 128>(g, cs) : launch_group<__half, 64>(g, cs);
        else wide ? launch_group<__nv_bfloat16, 128>(g, cs) : launch_group<__nv_bfloat16, 64>(g, cs);
    });
}
