// RMS norm of every query and key head, the position rotation, and the append to a paged KV
// cache, in one pass over the rows a q/k/v projection left.
//
//   y = x * rsqrt(mean(x^2) + eps) * gain;  (a, b) -> (a cos - b sin, b cos + a sin)
//
// The work is elementwise but for the mean, so it is bound by reading and writing the rows once
// (and by launch latency for a few rows). A head is spread over head_dim * size / 16 neighbouring
// lanes, one 16-byte load each: the mean is a butterfly over those lanes, the rotation partner of
// an element sits in the same lane (interleaved pairs) or half the lanes away. Everything is fp32
// until the one rounding on store.
//
// Keys also move the cached bounds (elementwise min and max of a page's keys). The rows that
// one call adds to one page are handled by one CTA, so bounds need no atomics and do not depend on
// order: a CTA takes the page runs that begin within kChunkRows rows of its own, keeps the rounded
// keys in shared memory and folds them into the bounds (which start anew with slot 0).
#include <algorithm>
#include <mutex>

#include "paged.cuh"

namespace vxc {
namespace {

constexpr int kThreads = 256;
constexpr int kChunkRows = 32;
constexpr int kMaxSpan = kChunkRows + 128;  // a CTA's runs end at most one page after its own rows

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int kVec = 4;
    __device__ static void unpack(const uint4 v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x);
        x[1] = __uint_as_float(v.y);
        x[2] = __uint_as_float(v.z);
        x[3] = __uint_as_float(v.w);
    }
    __device__ static uint4 pack(const float (&x)[4]) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
    __device__ static float to_float(float v) { return v; }
    __device__ static float from_float(float v) { return v; }
};
template <>
struct Elem<__half> {
    static constexpr int kVec = 8;
    __device__ static void unpack(const uint4 v, float (&x)[8]) {
        const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(h[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
    __device__ static uint4 pack(const float (&x)[8]) {
        uint4 v;
        __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        return v;
    }
    __device__ static float to_float(__half v) { return __half2float(v); }
    __device__ static __half from_float(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int kVec = 8;
    __device__ static void unpack(const uint4 v, float (&x)[8]) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __bfloat1622float2(h[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
    __device__ static uint4 pack(const float (&x)[8]) {
        uint4 v;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        return v;
    }
    __device__ static float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
    __device__ static __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
};

struct Args {
    vxc_qk_rows a;
    vxc_pages p;     // with a cache
    int layer;
    int flat_heads;  // heads of the flat part: the query heads, and the key heads without a cache
    int flat_ctas;
};

// The position of row r, or -1 where the row is skipped; a row out of range is reported.
__device__ __forceinline__ int row_position(const Args& g, int r, bool paged) {
    const int seq = g.a.row_seq ? g.a.row_seq[r] : 0;
    if (seq < 0) return -1;
    const int pos = g.a.row_pos[r];
    if (pos < 0 || (g.a.cos && pos >= g.a.positions) ||
        (paged && (seq >= g.p.n_seqs || pos >= g.p.max_pages * g.p.page_size))) {
        report(g.a.status, VXC_PAGES_BAD_ROW);
        return -1;
    }
    return pos;
}

template <typename T, int D>
struct Lanes {
    static constexpr int kVec = Elem<T>::kVec;
    static constexpr int kPer = D / kVec;    // lanes of a head: 8, 16 or 32
    static constexpr int kSlots = kThreads / kPer;
};

// cos and sin of this lane's elements (rotate-half: one per element; interleaved: one per pair, doubled).
template <typename T, int D>
__device__ __forceinline__ void load_turn(const Args& g, int pos, int l, float (&c)[Lanes<T, D>::kVec],
                                          float (&s)[Lanes<T, D>::kVec]) {
    constexpr int V = Lanes<T, D>::kVec;
    const float* ct = g.a.cos + static_cast<size_t>(pos) * D;
    const float* st = g.a.sin + static_cast<size_t>(pos) * D;
    if (g.a.interleaved) {
#pragma unroll
        for (int i = 0; i < V / 2; i += 2) {
            const float2 cv = *reinterpret_cast<const float2*>(ct + l * (V / 2) + i);
            const float2 sv = *reinterpret_cast<const float2*>(st + l * (V / 2) + i);
            c[2 * i] = c[2 * i + 1] = cv.x;
            c[2 * i + 2] = c[2 * i + 3] = cv.y;
            s[2 * i] = s[2 * i + 1] = sv.x;
            s[2 * i + 2] = s[2 * i + 3] = sv.y;
        }
    } else {
        const int j = (l * V) % (D / 2);
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 cv = *reinterpret_cast<const float4*>(ct + j + i);
            const float4 sv = *reinterpret_cast<const float4*>(st + j + i);
            c[i] = cv.x, c[i + 1] = cv.y, c[i + 2] = cv.z, c[i + 3] = cv.w;
            s[i] = sv.x, s[i + 1] = sv.y, s[i + 2] = sv.z, s[i + 3] = sv.w;
        }
    }
}

// Norm (of the lanes whose head has a gain; any: some head of the call has) and rotation of one head
// held by kPer lanes, in place. Every lane of the warp takes part.
template <typename T, int D>
__device__ __forceinline__ void norm_turn(float (&x)[Lanes<T, D>::kVec], const float (&gain)[Lanes<T, D>::kVec], bool any,
                                          bool norm, float eps, const float (&c)[Lanes<T, D>::kVec],
                                          const float (&s)[Lanes<T, D>::kVec], bool turn, bool pairs, int l) {
    constexpr int V = Lanes<T, D>::kVec, N = Lanes<T, D>::kPer;
    if (any) {
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) q = fmaf(x[i], x[i], q);
#pragma unroll
        for (int o = N / 2; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
        const float r = rsqrtf(q * (1.f / D) + eps);
        if (norm) {
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = x[i] * r * gain[i];
        }
    }
    if (!turn) return;
    if (pairs) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float a = x[i], b = x[i + 1];
            x[i] = a * c[i] - b * s[i];
            x[i + 1] = b * c[i] + a * s[i];
        }
    } else {
        const float sign = l < N / 2 ? -1.f : 1.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float other = __shfl_xor_sync(0xffffffffu, x[i], N / 2);
            x[i] = x[i] * c[i] + sign * other * s[i];
        }
    }
}

template <typename T, int D>
__device__ __forceinline__ void load_gain(const void* gain, int l, float (&x)[Lanes<T, D>::kVec]) {
    if (gain) Elem<T>::unpack(*reinterpret_cast<const uint4*>(static_cast<const T*>(gain) + l * Lanes<T, D>::kVec), x);
}

// Heads of single rows, in place or to another array: CTAs [0, flat_ctas).
template <typename T, int D>
__device__ void flat_heads(const Args& g, bool paged) {
    using L = Lanes<T, D>;
    const int slot = threadIdx.x / L::kPer, l = threadIdx.x % L::kPer;
    const long long items = static_cast<long long>(g.a.rows) * g.flat_heads;
    const long long it = static_cast<long long>(blockIdx.x) * L::kSlots + slot;
    const bool in = it < items;
    const int r = in ? static_cast<int>(it / g.flat_heads) : 0, h = in ? static_cast<int>(it - static_cast<long long>(r) * g.flat_heads) : 0;
    const int pos = in ? row_position(g, r, paged) : -1;
    const bool key = h >= g.a.q_heads, live = pos >= 0;
    const void* gain_p = key ? g.a.k_gain : g.a.q_gain;
    float x[L::kVec] = {}, gain[L::kVec] = {}, c[L::kVec] = {}, s[L::kVec] = {};
    if (live) {
        const T* from = key ? static_cast<const T*>(g.a.k) + static_cast<size_t>(r) * g.a.k_stride + (h - g.a.q_heads) * D
                            : static_cast<const T*>(g.a.q) + static_cast<size_t>(r) * g.a.q_stride + h * D;
        Elem<T>::unpack(*reinterpret_cast<const uint4*>(from + l * L::kVec), x);
        load_gain<T, D>(gain_p, l, gain);
        if (g.a.cos) load_turn<T, D>(g, pos, l, c, s);
    }
    norm_turn<T, D>(x, gain, g.a.q_gain || g.a.k_gain, gain_p != nullptr, g.a.eps, c, s, g.a.cos != nullptr,
                    g.a.interleaved != 0, l);
    if (live) {
        T* to = key ? static_cast<T*>(g.a.k_out) + static_cast<size_t>(r) * g.a.k_out_stride + (h - g.a.q_heads) * D
                    : static_cast<T*>(g.a.q_out) + static_cast<size_t>(r) * g.a.q_out_stride + h * D;
        *reinterpret_cast<uint4*>(to + l * L::kVec) = Elem<T>::pack(x);
    }
}

// Keys and values of one KV head: the page runs that begin in rows [chunk * kChunkRows, + kChunkRows).
template <typename T, int D>
__device__ void cache_rows(const Args& g, int chunk, int head, T* keys) {
    using L = Lanes<T, D>;
    __shared__ int s_page[kMaxSpan], s_slot[kMaxSpan], s_pos[kMaxSpan];
    __shared__ unsigned s_start[kMaxSpan / 32];
    __shared__ int s_runs[kChunkRows + 1];
    const vxc_pages& p = g.p;
    const int tid = threadIdx.x, lane = tid & 31, P = p.page_size;
    const int r0 = chunk * kChunkRows, span = kChunkRows + P;
    // which rows begin a run: all but those that follow their predecessor within a page
    if (tid < kMaxSpan) {
        const int r = r0 + tid;
        bool start = true;
        if (tid < span && r < g.a.rows && r > 0) {
            const int seq = g.a.row_seq[r], pos = g.a.row_pos[r];
            start = seq < 0 || pos <= 0 || pos % P == 0 || g.a.row_seq[r - 1] != seq || g.a.row_pos[r - 1] != pos - 1;
        }
        const unsigned b = __ballot_sync(0xffffffffu, start);
        if (lane == 0) s_start[tid >> 5] = b;
    }
    __syncthreads();
    if (s_start[0] == 0) return;
    const int first = __ffs(s_start[0]) - 1;
    int end = span;
    for (int w = 1; w < kMaxSpan / 32; ++w)
        if (s_start[w]) {
            end = min(end, w * 32 + __ffs(s_start[w]) - 1);
            break;
        }
    end = min(end, g.a.rows - r0);
    const int runs = __popc(s_start[0]);
    for (int j = tid; j < kChunkRows; j += kThreads)
        if (s_start[0] >> j & 1) s_runs[__popc(s_start[0] & ((1u << j) - 1))] = j;
    if (tid == 0) s_runs[runs] = max(end, first);
    for (int j = first + tid; j < end; j += kThreads) {
        const int pos = row_position(g, r0 + j, true);
        int page = -1;
        if (pos >= 0) {
            page = p.table[static_cast<size_t>(g.a.row_seq[r0 + j]) * p.max_pages + pos / P];
            if (page < 0 || page >= p.n_pages) {
                report(g.a.status, VXC_PAGES_BAD_ID);
                page = -1;
            }
        }
        s_page[j] = page;
        s_slot[j] = pos % P;
        s_pos[j] = pos;
    }
    __syncthreads();
    const size_t plane = (static_cast<size_t>(g.layer) * p.n_pages);
    const int slot = tid / L::kPer, l = tid % L::kPer;
    float gain[L::kVec] = {};
    load_gain<T, D>(g.a.k_gain, l, gain);
    for (int j0 = first; j0 < end; j0 += L::kSlots) {
        const int j = j0 + slot;
        const bool live = j < end && s_page[j] >= 0;
        float x[L::kVec] = {}, c[L::kVec] = {}, s[L::kVec] = {};
        uint4 v = make_uint4(0, 0, 0, 0);
        if (live) {
            const size_t r = static_cast<size_t>(r0 + j);
            Elem<T>::unpack(*reinterpret_cast<const uint4*>(static_cast<const T*>(g.a.k) + r * g.a.k_stride + head * D + l * L::kVec), x);
            v = *reinterpret_cast<const uint4*>(static_cast<const T*>(g.a.v) + r * g.a.v_stride + head * D + l * L::kVec);
            if (g.a.cos) load_turn<T, D>(g, s_pos[j], l, c, s);
        }
        norm_turn<T, D>(x, gain, g.a.k_gain != nullptr, true, g.a.eps, c, s, g.a.cos != nullptr, g.a.interleaved != 0, l);
        if (live) {
            const size_t at = (((plane + s_page[j]) * p.kv_heads + head) * P + s_slot[j]) * D + l * L::kVec;
            const uint4 k = Elem<T>::pack(x);
            *reinterpret_cast<uint4*>(static_cast<T*>(p.k) + at) = k;
            *reinterpret_cast<uint4*>(static_cast<T*>(p.v) + at) = v;
            *reinterpret_cast<uint4*>(keys + static_cast<size_t>(j - first) * D + l * L::kVec) = k;
        }
    }
    __syncthreads();
    for (int i = tid; i < runs * D; i += kThreads) {
        const int run = i / D, d = i - run * D, b = s_runs[run], e = min(s_runs[run + 1], end);
        if (b >= e || s_page[b] < 0) continue;
        T* bd = static_cast<T*>(p.bounds) + ((plane + s_page[b]) * p.kv_heads + head) * 2 * D + d;
        float lo, hi;
        int j = b;
        if (s_slot[b] == 0) {
            lo = hi = Elem<T>::to_float(keys[static_cast<size_t>(b - first) * D + d]);
            ++j;
        } else {
            lo = Elem<T>::to_float(bd[0]);
            hi = Elem<T>::to_float(bd[D]);
        }
        for (; j < e; ++j) {
            if (s_page[j] < 0) continue;
            const float x = Elem<T>::to_float(keys[static_cast<size_t>(j - first) * D + d]);
            // a NaN stays, so that the page's score is one too
            lo = x < lo || x != x ? x : lo;
            hi = x > hi || x != x ? x : hi;
        }
        bd[0] = Elem<T>::from_float(lo);
        bd[D] = Elem<T>::from_float(hi);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) qk_rows_kernel(const Args g, int paged) {
    extern __shared__ __align__(16) unsigned char keys[];
    pdl_launch_dependents();
    pdl_wait();
    if (static_cast<int>(blockIdx.x) < g.flat_ctas) {
        flat_heads<T, D>(g, paged != 0);
    } else {
        const int c = blockIdx.x - g.flat_ctas;
        cache_rows<T, D>(g, c / g.p.kv_heads, c % g.p.kv_heads, reinterpret_cast<T*>(keys));
    }
}

template <typename T, int D>
void launch(Args g, bool paged, cudaStream_t s) {
    using L = Lanes<T, D>;
    const long long items = static_cast<long long>(g.a.rows) * g.flat_heads;
    const long long flat = (items + L::kSlots - 1) / L::kSlots;
    const long long chunks = paged ? (static_cast<long long>(g.a.rows) + kChunkRows - 1) / kChunkRows * g.p.kv_heads : 0;
    paged_require(flat + chunks <= 0x7fffffffll, "vxc_qk_norm_rope: too many rows");
    g.flat_ctas = static_cast<int>(flat);
    const size_t smem = paged ? static_cast<size_t>(kChunkRows + g.p.page_size) * D * sizeof(T) : 0;
    if (smem > 48 * 1024)
        paged_ck(cudaFuncSetAttribute(qk_rows_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)),
                 "vxc_qk_norm_rope");
    paged_launch(qk_rows_kernel<T, D>, static_cast<unsigned>(flat + chunks), kThreads, smem, s, "vxc_qk_norm_rope", g,
                 paged ? 1 : 0);
}

void check_rows(const vxc_qk_rows* a, const vxc_pages* p, int layer) {
    paged_require(a->dtype == VXC_F32 || a->dtype == VXC_F16 || a->dtype == VXC_BF16,
                  "vxc_qk_norm_rope: dtype must be f32, f16 or bf16");
    paged_require(a->rows > 0, "vxc_qk_norm_rope: rows must be positive");
    paged_require(a->q_heads > 0 && a->q_heads <= 1024 && a->kv_heads > 0 && a->kv_heads <= kMaxKvHeads,
                  "vxc_qk_norm_rope: q_heads must be 1 to 1024, kv_heads 1 to 256");
    paged_require(a->head_dim == 64 || a->head_dim == 128, "vxc_qk_norm_rope: head_dim must be 64 or 128");
    paged_require(a->q && a->k && a->q_out && a->row_pos && a->status, "null argument");
    paged_require((a->cos != nullptr) == (a->sin != nullptr), "vxc_qk_norm_rope: cos and sin go together");
    paged_require(!a->cos || a->positions > 0, "vxc_qk_norm_rope: positions must be positive");
    paged_require(a->eps >= 0.f, "vxc_qk_norm_rope: eps must not be negative");
    const int unit = 16 / dtype_size(a->dtype);
    const int64_t q_row = static_cast<int64_t>(a->q_heads) * a->head_dim, k_row = static_cast<int64_t>(a->kv_heads) * a->head_dim;
    paged_require(aligned16(a->q) && aligned16(a->k) && aligned16(a->q_out) && aligned16(a->q_gain) && aligned16(a->k_gain) &&
                      aligned16(a->cos) && aligned16(a->sin) && aligned4(a->row_seq) && aligned4(a->row_pos) &&
                      aligned4(a->status),
                  "vxc_qk_norm_rope: rows, gains and tables must start on 16-byte boundaries");
    paged_require(a->q_stride >= q_row && a->k_stride >= k_row && a->q_out_stride >= q_row && a->q_stride % unit == 0 &&
                      a->k_stride % unit == 0 && a->q_out_stride % unit == 0,
                  "vxc_qk_norm_rope: strides must cover a row and be multiples of 16 bytes");
    if (p) {
        paged_require(a->v && a->row_seq, "null argument");
        paged_require(aligned16(a->v) && a->v_stride >= k_row && a->v_stride % unit == 0,
                      "vxc_qk_norm_rope: v must be laid out as k");
        check_page_sizes(p);
        paged_require(p->dtype == a->dtype && p->kv_heads == a->kv_heads && p->head_dim == a->head_dim,
                      "vxc_qk_norm_rope: rows and cache differ in dtype, kv_heads or head_dim");
        paged_require(layer >= 0 && layer < p->layers, "vxc_qk_norm_rope: layer out of range");
        check_pages(p);
    } else {
        paged_require(a->k_out != nullptr, "null argument");
        paged_require(aligned16(a->k_out) && a->k_out_stride >= k_row && a->k_out_stride % unit == 0,
                      "vxc_qk_norm_rope: k_out must be laid out as k");
    }
    check_device_pointer(a->q, "vxc_qk_norm_rope: q is not memory of the current device");
}

}  // namespace
}  // namespace vxc

using namespace vxc;

extern "C" VXC_API int32_t vxc_qk_norm_rope(const vxc_qk_rows* a, const vxc_pages* p, int32_t layer, void* cuda_stream) {
    return paged_guard([&] {
        paged_require(a != nullptr, "null argument");
        check_rows(a, p, layer);
        Args g = {};
        g.a = *a;
        if (p) g.p = *p;
        g.layer = layer;
        g.flat_heads = a->q_heads + (p ? 0 : a->kv_heads);
        const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
        const bool wide = a->head_dim == 128;
        if (a->dtype == VXC_F32) wide ? launch<float, 128>(g, p != nullptr, cs) : launch<float, 64>(g, p != nullptr, cs);
        else if (a->dtype == VXC_F16) wide ? launch<__half, 128>(g, p != nullptr, cs) : launch<__half, 64>(g, p != nullptr, cs);
        else wide ? launch<__nv_bfloat16, 128>(g, p != nullptr, cs) : launch<__nv_bfloat16, 64>(g, p != nullptr, cs);
    });
}
