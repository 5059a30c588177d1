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
    int cache_ctas;  // CTAs of the cached keys and values; the first, because theirs is the longer way
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

// Elements from one kept key to the next: 16 bytes more than a key, so that lanes on successive rows use other banks.
template <typename T, int D>
constexpr int key_row() {
    return D + 16 / static_cast<int>(sizeof(T));
}

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

// kHeads heads of one row per slot, in place or to another array. All their loads leave before the row's
// position is known; its cos and sin serve all of them.
template <typename T, int D, int kHeads>
__device__ void flat_heads(const Args& g, int cta, bool paged) {
    using L = Lanes<T, D>;
    const int slot = threadIdx.x / L::kPer, l = threadIdx.x % L::kPer;
    const int per_row = (g.flat_heads + kHeads - 1) / kHeads;
    const long long it = static_cast<long long>(cta) * L::kSlots + slot;
    const bool in = it < static_cast<long long>(g.a.rows) * per_row;
    const int r = in ? static_cast<int>(it / per_row) : 0;
    const int h0 = in ? static_cast<int>(it - static_cast<long long>(r) * per_row) * kHeads : 0;
    const T* q = static_cast<const T*>(g.a.q) + static_cast<size_t>(r) * g.a.q_stride + l * L::kVec;
    const T* k = static_cast<const T*>(g.a.k) + static_cast<size_t>(r) * g.a.k_stride + l * L::kVec;
    uint4 raw[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int h = h0 + i;
        raw[i] = make_uint4(0, 0, 0, 0);
        if (in && h < g.flat_heads)
            raw[i] = *reinterpret_cast<const uint4*>(h < g.a.q_heads ? q + h * D : k + (h - g.a.q_heads) * D);
    }
    float gq[L::kVec] = {}, gk[L::kVec] = {}, c[L::kVec] = {}, s[L::kVec] = {};
    load_gain<T, D>(g.a.q_gain, l, gq);
    if (g.flat_heads > g.a.q_heads) load_gain<T, D>(g.a.k_gain, l, gk);
    const int pos = in ? row_position(g, r, paged) : -1;
    if (pos >= 0 && g.a.cos) load_turn<T, D>(g, pos, l, c, s);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int h = h0 + i;
        const bool key = h >= g.a.q_heads;
        float x[L::kVec], gain[L::kVec];
        Elem<T>::unpack(raw[i], x);
#pragma unroll
        for (int j = 0; j < L::kVec; ++j) gain[j] = key ? gk[j] : gq[j];
        // query and key heads of one warp may differ in having a gain
        norm_turn<T, D>(x, gain, g.a.q_gain || g.a.k_gain, (key ? g.a.k_gain : g.a.q_gain) != nullptr, g.a.eps, c, s,
                        g.a.cos != nullptr, g.a.interleaved != 0, l);
        if (pos >= 0 && h < g.flat_heads) {
            T* to = key ? static_cast<T*>(g.a.k_out) + static_cast<size_t>(r) * g.a.k_out_stride + (h - g.a.q_heads) * D
                        : static_cast<T*>(g.a.q_out) + static_cast<size_t>(r) * g.a.q_out_stride + h * D;
            *reinterpret_cast<uint4*>(to + l * L::kVec) = Elem<T>::pack(x);
        }
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
    const int slot = tid / L::kPer, l = tid % L::kPer;
    const T* k_in = static_cast<const T*>(g.a.k) + head * D + l * L::kVec;
    const T* v_in = static_cast<const T*>(g.a.v) + head * D + l * L::kVec;
    // the first rows' loads do not wait for the look at their places
    uint4 k_raw = make_uint4(0, 0, 0, 0), v_raw = k_raw;
    if (r0 + slot < g.a.rows) {
        k_raw = *reinterpret_cast<const uint4*>(k_in + static_cast<size_t>(r0 + slot) * g.a.k_stride);
        v_raw = *reinterpret_cast<const uint4*>(v_in + static_cast<size_t>(r0 + slot) * g.a.v_stride);
    }
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
    const size_t plane = static_cast<size_t>(g.layer) * p.n_pages;
    // the bounds as they stand, for runs that go on in a begun page: (run, 16 bytes of lo or hi) per item, each item's rows
    // dealt to 'parts' neighbouring lanes
    const int items = runs * L::kPer;
    int parts = 1;
    while (parts < 32 && items * parts * 2 <= kThreads) parts *= 2;
    const int part = tid & (parts - 1);
    uint4 old_lo = make_uint4(0, 0, 0, 0), old_hi = old_lo;
    const auto bounds_at = [&](int run, int piece) {
        return static_cast<T*>(p.bounds) + ((plane + s_page[s_runs[run]]) * p.kv_heads + head) * 2 * D + piece * L::kVec;
    };
    const auto begun = [&](int run) {
        const int b = s_runs[run];
        return b < end && s_page[b] >= 0 && s_slot[b] != 0;
    };
    if (const int i = tid / parts; i < items && part == 0 && begun(i / L::kPer)) {
        const T* bd = bounds_at(i / L::kPer, i % L::kPer);
        old_lo = *reinterpret_cast<const uint4*>(bd);
        old_hi = *reinterpret_cast<const uint4*>(bd + D);
    }
    float gain[L::kVec] = {};
    load_gain<T, D>(g.a.k_gain, l, gain);
    for (int j0 = first; j0 < end; j0 += L::kSlots) {
        const int j = j0 + slot;
        const bool live = j < end && s_page[j] >= 0;
        float x[L::kVec] = {}, c[L::kVec] = {}, s[L::kVec] = {};
        if (live) {
            if (j != slot) {
                const size_t r = static_cast<size_t>(r0 + j);
                k_raw = *reinterpret_cast<const uint4*>(k_in + r * g.a.k_stride);
                v_raw = *reinterpret_cast<const uint4*>(v_in + r * g.a.v_stride);
            }
            Elem<T>::unpack(k_raw, x);
            if (g.a.cos) load_turn<T, D>(g, s_pos[j], l, c, s);
        }
        norm_turn<T, D>(x, gain, g.a.k_gain != nullptr, true, g.a.eps, c, s, g.a.cos != nullptr, g.a.interleaved != 0, l);
        if (live) {
            const size_t at = (((plane + s_page[j]) * p.kv_heads + head) * P + s_slot[j]) * D + l * L::kVec;
            const uint4 k = Elem<T>::pack(x);
            *reinterpret_cast<uint4*>(static_cast<T*>(p.k) + at) = k;
            *reinterpret_cast<uint4*>(static_cast<T*>(p.v) + at) = v_raw;
            *reinterpret_cast<uint4*>(keys + static_cast<size_t>(j - first) * key_row<T, D>() + l * L::kVec) = k;
        }
    }
    __syncthreads();
    for (int i0 = 0; i0 < items; i0 += kThreads / parts) {
        const int i = i0 + tid / parts, run = i / L::kPer, piece = i % L::kPer;
        const bool in = i < items && s_runs[run] < end && s_page[s_runs[run]] >= 0;
        const int b = in ? s_runs[run] : 0, e = in ? min(s_runs[run + 1], end) : 0;
        float lo[L::kVec], hi[L::kVec];
#pragma unroll
        for (int n = 0; n < L::kVec; ++n) {
            lo[n] = INFINITY;
            hi[n] = -INFINITY;
        }
        const auto fold = [&](const uint4 a, const uint4 z) {
            float x[L::kVec], y[L::kVec];
            Elem<T>::unpack(a, x);
            Elem<T>::unpack(z, y);
#pragma unroll
            for (int n = 0; n < L::kVec; ++n) {  // a NaN stays, so that the page's score is one too
                lo[n] = x[n] < lo[n] || x[n] != x[n] ? x[n] : lo[n];
                hi[n] = y[n] > hi[n] || y[n] != y[n] ? y[n] : hi[n];
            }
        };
        if (in && part == 0 && s_slot[b] != 0) {
            const T* bd = bounds_at(run, piece);
            if (i0 == 0) fold(old_lo, old_hi);
            else fold(*reinterpret_cast<const uint4*>(bd), *reinterpret_cast<const uint4*>(bd + D));
        }
        for (int j = b + part; j < e; j += parts) {
            if (s_page[j] < 0) continue;
            const uint4 x = *reinterpret_cast<const uint4*>(keys + static_cast<size_t>(j - first) * key_row<T, D>() + piece * L::kVec);
            fold(x, x);
        }
        for (int o = parts / 2; o > 0; o >>= 1)
#pragma unroll
            for (int n = 0; n < L::kVec; ++n) {
                const float x = __shfl_xor_sync(0xffffffffu, lo[n], o), y = __shfl_xor_sync(0xffffffffu, hi[n], o);
                lo[n] = x < lo[n] || x != x ? x : lo[n];
                hi[n] = y > hi[n] || y != y ? y : hi[n];
            }
        if (in && part == 0) {
            T* bd = bounds_at(run, piece);
            *reinterpret_cast<uint4*>(bd) = Elem<T>::pack(lo);
            *reinterpret_cast<uint4*>(bd + D) = Elem<T>::pack(hi);
        }
    }
}

template <typename T, int D, int kHeads>
__global__ void __launch_bounds__(kThreads) qk_rows_kernel(const Args g, int paged) {
    extern __shared__ __align__(16) unsigned char keys[];
    pdl_launch_dependents();
    pdl_wait();
    const int c = blockIdx.x;
    if (c < g.cache_ctas) cache_rows<T, D>(g, c / g.p.kv_heads, c % g.p.kv_heads, reinterpret_cast<T*>(keys));
    else flat_heads<T, D, kHeads>(g, c - g.cache_ctas, paged != 0);
}

template <typename T, int D, int kHeads>
void launch_heads(Args& g, bool paged, cudaStream_t s) {
    using L = Lanes<T, D>;
    const long long items = static_cast<long long>(g.a.rows) * ((g.flat_heads + kHeads - 1) / kHeads);
    const long long flat = (items + L::kSlots - 1) / L::kSlots;
    const long long cache = paged ? (static_cast<long long>(g.a.rows) + kChunkRows - 1) / kChunkRows * g.p.kv_heads : 0;
    paged_require(flat + cache <= 0x7fffffffll, "vxc_qk_norm_rope: too many rows");
    g.cache_ctas = static_cast<int>(cache);
    const size_t smem = paged ? static_cast<size_t>(kChunkRows + g.p.page_size) * key_row<T, D>() * sizeof(T) : 0;
    if (smem > 40 * 1024)
        paged_ck(cudaFuncSetAttribute(qk_rows_kernel<T, D, kHeads>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(smem)),
                 "vxc_qk_norm_rope");
    paged_launch(qk_rows_kernel<T, D, kHeads>, static_cast<unsigned>(flat + cache), kThreads, smem, s, "vxc_qk_norm_rope",
                 g, paged ? 1 : 0);
}

template <typename T, int D>
void launch(Args g, bool paged, cudaStream_t s) {
    // few rows: a head per slot, as many CTAs as there are; many: four, whose loads overlap
    if (static_cast<long long>(g.a.rows) * g.flat_heads <= 8ll * 148 * Lanes<T, D>::kSlots) launch_heads<T, D, 1>(g, paged, s);
    else launch_heads<T, D, 4>(g, paged, s);
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
