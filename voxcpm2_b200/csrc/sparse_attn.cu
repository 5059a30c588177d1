// Attention over the pages of a cache that a cheap score picks for every query row and KV head.
//
//   score(page) = sum over the KV head's query heads h of sum_d max(q_hd lo_d, q_hd hi_d)
//               = sum_d (sum_h max(q_hd, 0)) hi_d + (sum_h min(q_hd, 0)) lo_d
//
// so one product with 2 head_dim terms per page, whatever the number of heads. It is summed in
// fp64: fp16 and bf16 products are exact there, so the order of summation does not decide which of two pages is
// taken. The picked pages are attended over with a running maximum and sum.
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace vxc {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 256;
constexpr int kMaxGroup = 16;

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// fp64 scores as integers of the same order; NaN as +infinity, -0 as 0.
__device__ __forceinline__ unsigned long long order_key(double s) {
    s = s != s ? __longlong_as_double(0x7ff0000000000000ll) : s + 0.0;
    const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(s));
    return b >> 63 ? ~b : b | 1ull << 63;
}

struct Args {
    vxc_sparse_query a;
    vxc_pages p;
    int layer;
    float scale;
};

// The m largest of key[0, n), equal ones lowest index first, as ascending indices + base at list[]. 0 < m < n.
__device__ void pick(const unsigned long long* key, int n, int m, int base, int* list, int* s_scan) {
    const int tid = threadIdx.x;
    unsigned long long lo = 0;  // count(key >= lo) >= m
    for (int bit = 63; bit >= 0; --bit) {
        const unsigned long long t = lo | 1ull << bit;
        int c = 0;
        for (int i = tid; i < n; i += kThreads) c += key[i] >= t;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
        if ((tid & 31) == 0) s_scan[tid >> 5] = c;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) all += s_scan[w];
        __syncthreads();
        if (all >= m) lo = t;
        if (all == m) break;
    }
    // lo is the m-th largest key (or below it with nothing between): all above it, and the first of the equal ones
    const int per = (n + kThreads - 1) / kThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    int above = 0, equal = 0;
    for (int i = i0; i < i1; ++i) {
        above += key[i] > lo;
        equal += key[i] == lo;
    }
    int x = above | equal << 16;  // n <= 16384 of each
    const int mine = x, lane = tid & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s_scan[tid >> 5] = x;
    __syncthreads();
    int before = x - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < tid >> 5) before += s_scan[w];
        total += s_scan[w];
    }
    const int ties = m - (total & 0xffff);
    int eq = before >> 16, at = (before & 0xffff) + min(eq, ties);
    for (int i = i0; i < i1; ++i) {
        const bool tie = key[i] == lo;
        if (key[i] > lo || (tie && eq < ties)) list[at++] = base + i;
        eq += tie;
    }
    __syncthreads();
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) sparse_kernel(const Args g) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ double s_up[D], s_down[D];
    __shared__ float s_q[kMaxGroup][D], s_score[kMaxGroup][128], s_m[kMaxGroup], s_l[kMaxGroup], s_fix[kMaxGroup];
    __shared__ int s_list[kMaxTop], s_scan[kWarps];
    unsigned long long* key = reinterpret_cast<unsigned long long*>(smem);
    pdl_launch_dependents();
    pdl_wait();
    const vxc_pages& p = g.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, P = p.page_size;
    const int r = blockIdx.x / p.kv_heads, head = blockIdx.x % p.kv_heads, G = g.a.q_heads / p.kv_heads;
    const int seq = g.a.row_seq[r], pos = g.a.row_pos[r];
    if (seq < 0) return;
    if (seq >= p.n_seqs || pos < 0 || pos >= p.max_pages * P) {
        if (tid == 0) report(p.status, VXC_PAGES_BAD_ROW);
        return;
    }
    const int* table = p.table + static_cast<size_t>(seq) * p.max_pages;
    const size_t plane = static_cast<size_t>(g.layer) * p.n_pages;
    const T* q = static_cast<const T*>(g.a.q) + static_cast<size_t>(r) * g.a.q_stride + static_cast<size_t>(head) * G * D;
    for (int i = tid; i < G * D; i += kThreads) s_q[i / D][i % D] = to_f(q[i]);
    __syncthreads();
    const int seen = pos / P + 1, take = min(seen, g.a.top_pages);
    if (seen <= take) {
        for (int i = tid; i < take; i += kThreads) s_list[i] = i;
    } else {
        const int sink = g.a.sink_pages, local = g.a.local_pages, n = seen - sink - local, m = take - sink - local;
        for (int d = tid; d < D; d += kThreads) {
            double up = 0, down = 0;
            for (int h = 0; h < G; ++h) {
                up += fmaxf(s_q[h][d], 0.f) + (s_q[h][d] != s_q[h][d] ? s_q[h][d] : 0.f);
                down += fminf(s_q[h][d], 0.f);
            }
            s_up[d] = up;
            s_down[d] = down;
        }
        __syncthreads();
        for (int i = tid; i < sink; i += kThreads) s_list[i] = i;
        for (int i = tid; i < local; i += kThreads) s_list[take - local + i] = seen - local + i;
        if (m > 0) {
            for (int i = warp; i < n; i += kWarps) {
                const int id = table[sink + i];
                double s = 0;
                if (id >= 0 && id < p.n_pages) {
                    const T* b = static_cast<const T*>(p.bounds) + ((plane + id) * p.kv_heads + head) * 2 * D;
                    for (int d = lane; d < D; d += 32)
                        s += s_up[d] * static_cast<double>(to_f(b[D + d])) + s_down[d] * static_cast<double>(to_f(b[d]));
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                if (lane == 0) key[i] = order_key(s);
            }
            __syncthreads();
            pick(key, n, m, sink, s_list + sink, s_scan);
        }
    }
    __syncthreads();
    if (g.a.selected)
        for (int i = tid; i < g.a.top_pages; i += kThreads)
            g.a.selected[(static_cast<size_t>(r) * p.kv_heads + head) * g.a.top_pages + i] = i < take ? s_list[i] : -1;
    // attention: thread (head, elements) of the output; the scores of one page at a time
    constexpr int kOut = kMaxGroup * D / kThreads;  // 4 or 8
    float acc[kOut] = {};
    if (tid < kMaxGroup) {
        s_m[tid] = -INFINITY;
        s_l[tid] = 0.f;
    }
    __syncthreads();
    for (int j = 0; j < take; ++j) {
        const int id = table[s_list[j]];
        if (id < 0 || id >= p.n_pages) {
            if (tid == 0) report(p.status, VXC_PAGES_BAD_ID);
            continue;
        }
        const size_t at = ((plane + id) * p.kv_heads + head) * static_cast<size_t>(P) * D;
        const T *k = static_cast<const T*>(p.k) + at, *v = static_cast<const T*>(p.v) + at;
        const int keys = min(P, pos + 1 - s_list[j] * P);
        for (int i = tid; i < G * keys; i += kThreads) {
            const int h = i / keys, t = i - h * keys;
            float s = 0.f;
            for (int d = 0; d < D; ++d) s = fmaf(s_q[h][d], to_f(k[t * D + d]), s);
            s_score[h][t] = s * g.scale;
        }
        __syncthreads();
        for (int h = warp; h < G; h += kWarps) {
            float mx = -INFINITY;
            for (int t = lane; t < keys; t += 32) mx = fmaxf(mx, s_score[h][t]);
            mx = fmaxf(warp_max(mx), s_m[h]);
            float sum = 0.f;
            for (int t = lane; t < keys; t += 32) {
                const float w = expf(s_score[h][t] - mx);
                s_score[h][t] = w;
                sum += w;
            }
            sum = warp_sum(sum);
            if (lane == 0) {
                s_fix[h] = expf(s_m[h] - mx);
                s_l[h] = s_l[h] * s_fix[h] + sum;
                s_m[h] = mx;
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kOut; ++e) {
            const int o = tid + e * kThreads, h = o / D, d = o % D;
            if (h >= G) continue;
            float x = acc[e] * s_fix[h];
            for (int t = 0; t < keys; ++t) x = fmaf(s_score[h][t], to_f(v[t * D + d]), x);
            acc[e] = x;
        }
        __syncthreads();
    }
    T* out = static_cast<T*>(g.a.out) + static_cast<size_t>(r) * g.a.out_stride + static_cast<size_t>(head) * G * D;
#pragma unroll
    for (int e = 0; e < kOut; ++e) {
        const int o = tid + e * kThreads, h = o / D;
        if (h < G) out[o] = from_f<T>(s_l[h] == 0.f ? 0.f : acc[e] / s_l[h]);  // 0: every page was refused
    }
}

template <typename T, int D>
void launch(const Args& g, cudaStream_t s) {
    const size_t smem = sizeof(unsigned long long) * g.p.max_pages;
    if (smem > 16 * 1024)
        paged_ck(cudaFuncSetAttribute(sparse_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)),
                 "vxc_sparse_attention");
    paged_launch(sparse_kernel<T, D>, static_cast<unsigned>(g.a.rows) * g.p.kv_heads, kThreads, smem, s,
                 "vxc_sparse_attention", g);
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
    check_pages(p);
    check_device_pointer(a->q, "vxc_sparse_attention: q is not memory of the current device");
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
        if (p->dtype == VXC_F32) wide ? launch<float, 128>(g, cs) : launch<float, 64>(g, cs);
        else if (p->dtype == VXC_F16) wide ? launch<__half, 128>(g, cs) : launch<__half, 64>(g, cs);
        else wide ? launch<__nv_bfloat16, 128>(g, cs) : launch<__nv_bfloat16, 64>(g, cs);
    });
}
