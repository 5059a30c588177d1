// RMS norm of every query and key head, the position rotation, and the append to a paged KV
// cache, in one pass over the rows a q/k/v projection left.
//
//   y = x * rsqrt(mean(x^2) + eps) * gain;  (a, b) -> (a cos - b sin, b cos + a sin)
//
// The work is elementwise but for the mean, so it is bound by reading and writing the rows once,
// by a launch for few rows (1 row of 16 + 2 heads 4 us back to back, 61 rows of 32 + 8 heads 6.7 us). A head is spread
// over head_dim * size / 16 neighbouring lanes, one 16-byte load each: the mean is a butterfly
// over those lanes, the rotation partner of an element sits in the same lane (interleaved pairs) or half
// the lanes away. Everything is fp32 until the one rounding on store. Rows in bulk fill no unit: 6176 rows of 32 + 8
// heads of 128 bf16, 151 MB, take 38.9 us, 3.9 TB/s. The kernel of the heads that pass through keeps 53 % of the issue
// slots and 39 % of the ALU busy; its 16 warps an SM wait for memory, fixed latencies and shuffles in turn. 4 heads a
// slot instead of 1 brought the rows from 79 to 52 us, fp32 pairs and integer indices of 32 bits to 39. Rotated by
// halves instead of pairs they take 2.7 us more.
//
// Keys also move the cached bounds (elementwise min and max of a page's keys). The rows that
// one call adds to one page are handled by one CTA, so bounds need no atomics and do not depend on
// order: a CTA takes the page runs that begin within kChunkRows rows of its own, keeps the rounded
// keys in shared memory and folds them into the bounds (which start anew with slot 0).
#include <algorithm>

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
    __device__ static void unpack(const uint4 v, float2 (&x)[2]) {
        x[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
        x[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
    }
    __device__ static uint4 pack(const float2 (&x)[2]) {
        return make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x), __float_as_uint(x[1].y));
    }
    static constexpr uint32_t kInf = 0x7f800000u, kMinusInf = 0xff800000u;
    __device__ static uint32_t least(uint32_t a, uint32_t b) {
        float r;
        asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
        return __float_as_uint(r);
    }
    __device__ static uint32_t most(uint32_t a, uint32_t b) {
        float r;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
        return __float_as_uint(r);
    }
};
template <>
struct Elem<__half> {
    static constexpr int kVec = 8;
    __device__ static void unpack(const uint4 v, float2 (&x)[4]) {
        const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __half22float2(h[i]);
    }
    __device__ static uint4 pack(const float2 (&x)[4]) {
        uint4 v;
        __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[i].x, x[i].y);
        return v;
    }
    static constexpr uint32_t kInf = 0x7c007c00u, kMinusInf = 0xfc00fc00u;
    __device__ static uint32_t least(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    __device__ static uint32_t most(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int kVec = 8;
    __device__ static void unpack(const uint4 v, float2 (&x)[4]) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __bfloat1622float2(h[i]);
    }
    __device__ static uint4 pack(const float2 (&x)[4]) {
        uint4 v;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[i].x, x[i].y);
        return v;
    }
    static constexpr uint32_t kInf = 0x7f807f80u, kMinusInf = 0xff80ff80u;
    __device__ static uint32_t least(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    __device__ static uint32_t most(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
};

struct Args {
    vxc_qk_rows a;
    vxc_pages p;     // with a cache
    int layer;
    int paged;
    int rotation;
    int cache_ctas;  // CTAs of the cached keys and values; the first, because theirs is the longer way
};

// The position of a row, or -1 where it is skipped; a row out of range is reported.
__device__ __forceinline__ int row_position(const Args& g, int seq, int pos) {
    if (seq < 0) return -1;
    if (pos < 0 || (g.a.cos && pos >= g.a.positions) ||
        (g.paged && (seq >= g.p.n_seqs || pos >= g.p.max_pages * g.p.page_size))) {
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

// Norm and rotation of a head as y_i = r (x_i a_i + x_j b_i), j the rotation partner of i: the
// gains, cos and sin of a row go into a and b once and serve all of its heads. Two elements per
// instruction (fp32 pairs).
enum Rotation : int { kNone = 0, kHalves = 1, kPairs = 2 };
template <typename T, int D>
struct Turn {
    static constexpr int V = Lanes<T, D>::kVec, N = Lanes<T, D>::kPer;
    float2 a[V / 2], b[V / 2];

    __device__ __forceinline__ void load(const Args& g, int rotation, const void* gain, int pos, int l) {
        const float* ct = g.a.cos + static_cast<size_t>(pos) * D;
        const float* st = g.a.sin + static_cast<size_t>(pos) * D;
        const T* gp = static_cast<const T*>(gain);
        float2 own[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) own[i] = make_float2(1.f, 1.f);
        if (gain) Elem<T>::unpack(*reinterpret_cast<const uint4*>(gp + l * V), own);
        if (rotation == kNone) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                a[i] = own[i];
                b[i] = make_float2(0.f, 0.f);
            }
        } else if (rotation == kPairs) {
#pragma unroll
            for (int i = 0; i < V / 2; i += 2) {
                const float2 c = *reinterpret_cast<const float2*>(ct + l * (V / 2) + i);
                const float2 s = *reinterpret_cast<const float2*>(st + l * (V / 2) + i);
                a[i] = make_float2(own[i].x * c.x, own[i].y * c.x);
                b[i] = make_float2(-own[i].y * s.x, own[i].x * s.x);
                a[i + 1] = make_float2(own[i + 1].x * c.y, own[i + 1].y * c.y);
                b[i + 1] = make_float2(-own[i + 1].y * s.y, own[i + 1].x * s.y);
            }
        } else {
            const int j = (l & (N / 2 - 1)) * V;
            const float sign = l < N / 2 ? -1.f : 1.f;
            float2 other[V / 2];
#pragma unroll
            for (int i = 0; i < V / 2; ++i) other[i] = make_float2(sign, sign);
            if (gain) {
                Elem<T>::unpack(*reinterpret_cast<const uint4*>(gp + (l ^ (N / 2)) * V), other);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) other[i] = __fmul2_rn(other[i], make_float2(sign, sign));
            }
#pragma unroll
            for (int i = 0; i < V / 2; i += 2) {
                const float4 c = *reinterpret_cast<const float4*>(ct + j + 2 * i), s = *reinterpret_cast<const float4*>(st + j + 2 * i);
                a[i] = __fmul2_rn(own[i], make_float2(c.x, c.y));
                a[i + 1] = __fmul2_rn(own[i + 1], make_float2(c.z, c.w));
                b[i] = __fmul2_rn(other[i], make_float2(s.x, s.y));
                b[i + 1] = __fmul2_rn(other[i + 1], make_float2(s.z, s.w));
            }
        }
    }

    // Every lane of the warp takes part; any: some head of the call has a norm, norm: this one has.
    __device__ __forceinline__ uint4 apply(const Args& g, int rotation, const uint4 raw, bool any, bool norm) const {
        float2 x[V / 2];
        Elem<T>::unpack(raw, x);
        float r = 1.f;
        if (any) {
            float2 q2 = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) q2 = __ffma2_rn(x[i], x[i], q2);
            float q = q2.x + q2.y;
#pragma unroll
            for (int o = N / 2; o > 0; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
            if (norm) r = rsqrtf(q * (1.f / D) + g.a.eps);
        }
        const float2 rr = make_float2(r, r);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            float2 y;
            if (rotation == kNone) {
                y = __fmul2_rn(x[i], a[i]);
            } else {
                const float2 z = rotation == kPairs ? make_float2(x[i].y, x[i].x)
                                                    : make_float2(__shfl_xor_sync(0xffffffffu, x[i].x, N / 2),
                                                                  __shfl_xor_sync(0xffffffffu, x[i].y, N / 2));
                y = __ffma2_rn(x[i], a[i], __fmul2_rn(z, b[i]));
            }
            x[i] = __fmul2_rn(y, rr);
        }
        return Elem<T>::pack(x);
    }
};

// Up to kHeads heads of one row and one kind (queries; keys, without a cache): what a slot takes at a time.
template <typename T, int D, int kHeads>
struct Flat {
    using L = Lanes<T, D>;
    uint4 raw[kHeads] = {};
    int r = 0, h0 = 0, n = 0, seq = -1, pos = -1;  // n heads from h0
    bool key = false;

    __device__ static int per_row(const Args& g) {
        return (g.a.q_heads + kHeads - 1) / kHeads + (g.paged ? 0 : (g.a.kv_heads + kHeads - 1) / kHeads);
    }
    // Part 'part' of row 'row' (none if the rows end before). The heads' loads do not wait for the look at
    // the row's place.
    __device__ __forceinline__ void load(const Args& g, int row, int part, int l) {
        n = 0;
        seq = -1;
        r = row;
        if (row < g.a.rows) {
            const int q_parts = (g.a.q_heads + kHeads - 1) / kHeads;
            key = part >= q_parts;
            h0 = (key ? part - q_parts : part) * kHeads;
            n = min(kHeads, (key ? g.a.kv_heads : g.a.q_heads) - h0);
            const T* from = (key ? static_cast<const T*>(g.a.k) + static_cast<size_t>(r) * g.a.k_stride
                                 : static_cast<const T*>(g.a.q) + static_cast<size_t>(r) * g.a.q_stride) + h0 * D + l * L::kVec;
#pragma unroll
            for (int i = 0; i < kHeads; ++i)
                if (i < n) raw[i] = *reinterpret_cast<const uint4*>(from + i * D);
            seq = g.a.row_seq ? g.a.row_seq[r] : 0;
            pos = g.a.row_pos[r];
        }
    }
    // After that: whether the row is taken.
    __device__ __forceinline__ bool live(const Args& g) {
        pos = row_position(g, seq, pos);
        return pos >= 0;
    }
    __device__ __forceinline__ void finish(const Args& g, int rotation, const Turn<T, D>& t, int l) const {
        T* to = (key ? static_cast<T*>(g.a.k_out) + static_cast<size_t>(r) * g.a.k_out_stride
                     : static_cast<T*>(g.a.q_out) + static_cast<size_t>(r) * g.a.q_out_stride) + h0 * D + l * L::kVec;
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const uint4 y = t.apply(g, rotation, raw[i], g.a.q_gain || g.a.k_gain, (key ? g.a.k_gain : g.a.q_gain) != nullptr);
            if (pos >= 0 && i < n) *reinterpret_cast<uint4*>(to + i * D) = y;
        }
    }
};

// Keys and values of up to kHeads KV heads from head0: the page runs that begin in rows [chunk * kChunkRows, + kChunkRows).
// keys: the rounded keys, [kHeads][kChunkRows + page_size][key_row].
template <typename T, int D, int kHeads>
__device__ void cache_rows(const Args& g, int chunk, int head0, T* keys) {
    using L = Lanes<T, D>;
    __shared__ int s_page[kMaxSpan], s_slot[kMaxSpan], s_pos[kMaxSpan];
    __shared__ unsigned s_start[kMaxSpan / 32];
    __shared__ int s_runs[kChunkRows + 1];
    const vxc_pages& p = g.p;
    const int tid = threadIdx.x, lane = tid & 31, P = p.page_size;
    const int r0 = chunk * kChunkRows, span = kChunkRows + P;
    const int slot = tid / L::kPer, l = tid % L::kPer;
    const int rotation = g.rotation, heads = min(kHeads, p.kv_heads - head0), key_plane = span * key_row<T, D>();
    const T* k_in = static_cast<const T*>(g.a.k) + head0 * D + l * L::kVec;
    const T* v_in = static_cast<const T*>(g.a.v) + head0 * D + l * L::kVec;
    // a row's keys and values; the first rows' loads do not wait for the look at their places
    uint4 k_raw[kHeads] = {}, v_raw[kHeads] = {};
    int held = slot;
    const auto fetch = [&](int j) {
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
            if (h < heads) {
                k_raw[h] = *reinterpret_cast<const uint4*>(k_in + static_cast<size_t>(r0 + j) * g.a.k_stride + h * D);
                v_raw[h] = *reinterpret_cast<const uint4*>(v_in + static_cast<size_t>(r0 + j) * g.a.v_stride + h * D);
            }
        held = j;
    };
    if (r0 + slot < g.a.rows) fetch(slot);
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
        const int pos = row_position(g, g.a.row_seq[r0 + j], g.a.row_pos[r0 + j]);
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
    // the bounds as they stand, for runs that go on in a begun page: (run, head, 16 bytes of lo or hi) per item, each
    // item's rows dealt to 'parts' neighbouring lanes
    const int items = runs * heads * L::kPer;
    int parts = 1;
    while (parts < 32 && items * parts * 2 <= kThreads) parts *= 2;
    const int part = tid & (parts - 1);
    uint4 old_lo = make_uint4(0, 0, 0, 0), old_hi = old_lo;
    const auto bounds_at = [&](int run, int h, int piece) {
        return static_cast<T*>(p.bounds) + ((plane + s_page[s_runs[run]]) * p.kv_heads + head0 + h) * 2 * D + piece * L::kVec;
    };
    const auto begun = [&](int run) {
        const int b = s_runs[run];
        return b < end && s_page[b] >= 0 && s_slot[b] != 0;
    };
    if (const int i = tid / parts, ih = i / L::kPer; i < items && part == 0 && begun(ih / heads)) {
        const T* bd = bounds_at(ih / heads, ih % heads, i % L::kPer);
        old_lo = *reinterpret_cast<const uint4*>(bd);
        old_hi = *reinterpret_cast<const uint4*>(bd + D);
    }
    for (int j0 = first; j0 < end; j0 += L::kSlots) {
        const int j = j0 + slot;
        const bool live = j < end && s_page[j] >= 0;
        if (live && held != j) fetch(j);
        uint4 k_now[kHeads], v_now[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            k_now[h] = k_raw[h];
            v_now[h] = v_raw[h];
        }
        if (j + L::kSlots < end) fetch(j + L::kSlots);
        Turn<T, D> turn = {};
        if (live) turn.load(g, rotation, g.a.k_gain, s_pos[j], l);
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            const uint4 k = turn.apply(g, rotation, k_now[h], g.a.k_gain != nullptr, true);
            if (live && h < heads) {
                const size_t at = (((plane + s_page[j]) * p.kv_heads + head0 + h) * P + s_slot[j]) * D + l * L::kVec;
                *reinterpret_cast<uint4*>(static_cast<T*>(p.k) + at) = k;
                *reinterpret_cast<uint4*>(static_cast<T*>(p.v) + at) = v_now[h];
                *reinterpret_cast<uint4*>(keys + h * key_plane + (j - first) * key_row<T, D>() + l * L::kVec) = k;
            }
        }
    }
    __syncthreads();
    for (int i0 = 0; i0 < items; i0 += kThreads / parts) {
        const int i = i0 + tid / parts, piece = i % L::kPer, ih = i / L::kPer, run = ih / heads, h = ih - run * heads;
        const bool in = i < items && s_runs[run] < end && s_page[s_runs[run]] >= 0;
        const int b = in ? s_runs[run] : 0, e = in ? min(s_runs[run + 1], end) : 0;
        // elementwise, in the type itself; a NaN stays, so that the page's score is one too
        uint4 lo = make_uint4(Elem<T>::kInf, Elem<T>::kInf, Elem<T>::kInf, Elem<T>::kInf);
        uint4 hi = make_uint4(Elem<T>::kMinusInf, Elem<T>::kMinusInf, Elem<T>::kMinusInf, Elem<T>::kMinusInf);
        const auto fold = [&](const uint4 a, const uint4 z) {
            lo.x = Elem<T>::least(lo.x, a.x), lo.y = Elem<T>::least(lo.y, a.y);
            lo.z = Elem<T>::least(lo.z, a.z), lo.w = Elem<T>::least(lo.w, a.w);
            hi.x = Elem<T>::most(hi.x, z.x), hi.y = Elem<T>::most(hi.y, z.y);
            hi.z = Elem<T>::most(hi.z, z.z), hi.w = Elem<T>::most(hi.w, z.w);
        };
        if (in && part == 0 && s_slot[b] != 0) {
            const T* bd = bounds_at(run, h, piece);
            if (i0 == 0) fold(old_lo, old_hi);
            else fold(*reinterpret_cast<const uint4*>(bd), *reinterpret_cast<const uint4*>(bd + D));
        }
        for (int j = b + part; j < e; j += parts) {
            if (s_page[j] < 0) continue;
            const uint4 x = *reinterpret_cast<const uint4*>(keys + h * key_plane + (j - first) * key_row<T, D>() + piece * L::kVec);
            fold(x, x);
        }
        for (int o = parts / 2; o > 0; o >>= 1) {
            uint4 a, z;
            a.x = __shfl_xor_sync(0xffffffffu, lo.x, o), a.y = __shfl_xor_sync(0xffffffffu, lo.y, o);
            a.z = __shfl_xor_sync(0xffffffffu, lo.z, o), a.w = __shfl_xor_sync(0xffffffffu, lo.w, o);
            z.x = __shfl_xor_sync(0xffffffffu, hi.x, o), z.y = __shfl_xor_sync(0xffffffffu, hi.y, o);
            z.z = __shfl_xor_sync(0xffffffffu, hi.z, o), z.w = __shfl_xor_sync(0xffffffffu, hi.w, o);
            fold(a, z);
        }
        if (in && part == 0) {
            T* bd = bounds_at(run, h, piece);
            *reinterpret_cast<uint4*>(bd) = lo;
            *reinterpret_cast<uint4*>(bd + D) = hi;
        }
    }
}

// Few rows: one launch, a head per slot, the CTAs of cached keys and values first.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) few_rows_kernel(const __grid_constant__ Args g) {
    extern __shared__ __align__(16) unsigned char keys[];
    pdl_launch_dependents();
    pdl_wait();
    const int c = blockIdx.x;
    if (c < g.cache_ctas) {
        cache_rows<T, D, 1>(g, c / g.p.kv_heads, c % g.p.kv_heads, reinterpret_cast<T*>(keys));
        return;
    }
    using L = Lanes<T, D>;
    const int l = threadIdx.x % L::kPer, rotation = g.rotation;
    Flat<T, D, 1> f;
    const unsigned it = static_cast<unsigned>(c - g.cache_ctas) * L::kSlots + threadIdx.x / L::kPer, per = Flat<T, D, 1>::per_row(g);
    f.load(g, static_cast<int>(it / per), static_cast<int>(it % per), l);
    Turn<T, D> turn = {};
    if (f.live(g)) turn.load(g, rotation, f.key ? g.a.k_gain : g.a.q_gain, f.pos, l);
    f.finish(g, rotation, turn, l);
}

// Many rows: the cached part by itself (its registers and shared memory would keep the other part's
// CTAs few) ...
constexpr int kCacheHeads = 2;
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 3) cache_rows_kernel(const __grid_constant__ Args g) {
    extern __shared__ __align__(16) unsigned char keys[];
    pdl_wait();
    pdl_launch_dependents();  // after the wait: see flat_rows_kernel
    const int groups = (g.p.kv_heads + kCacheHeads - 1) / kCacheHeads, chunk = blockIdx.x / groups;
    cache_rows<T, D, kCacheHeads>(g, chunk, (blockIdx.x - chunk * groups) * kCacheHeads, reinterpret_cast<T*>(keys));
}

// ... and the heads that only pass through, by CTAs that stay, the next four heads of a slot on their
// way while it computes the last four. With a cache this kernel comes after cache_rows_kernel, of which it
// needs nothing: it starts once all of that one's CTAs have passed their wait, so what came before both
// is complete and written back, and waits for it only at its own end, so that a later kernel that waits for this one
// has both. The fence stands for the wait that it leaves out: lines that an SM's L1 may hold from before are not
// read. (Waiting first takes 2.6 us more on the rows above, reading past the L1 0.7 to 11.)
// Measured on the 6176 rows above before the fence, heads at a time / CTAs an SM: 4 / 2 38.4 us, 4 / 3 39.2, 2 / 4 38.4, 8 / 2 37.7 (but
// half the slots idle with 4 query heads); two KV heads a CTA of the cached part against one 42.8 and four 57.2.
constexpr int kFlatHeads = 4;
constexpr int kFlatCtas = 2;
template <typename T, int D, int rotation>
__global__ void __launch_bounds__(kThreads, kFlatCtas) flat_rows_kernel(const __grid_constant__ Args g) {
    if (!g.paged) {
        pdl_launch_dependents();
        pdl_wait();
    } else {
        __threadfence();
    }
    using L = Lanes<T, D>;
    using F = Flat<T, D, kFlatHeads>;
    const int l = threadIdx.x % L::kPer, per = F::per_row(g);
    // this slot's (row, part), and how far it goes at a time
    const unsigned it = blockIdx.x * L::kSlots + threadIdx.x / L::kPer, step = gridDim.x * L::kSlots;
    const int row_step = static_cast<int>(step / per), part_step = static_cast<int>(step % per);
    int row = static_cast<int>(it / per), part = static_cast<int>(it % per);
    F f;
    f.load(g, row, part, l);
    while (__any_sync(0xffffffffu, row < g.a.rows)) {
        row += row_step;
        part += part_step;
        if (part >= per) {
            part -= per;
            ++row;
        }
        const bool live = f.live(g);
        F next;
        next.load(g, row, part, l);
        Turn<T, D> turn = {};
        if (live) turn.load(g, rotation, f.key ? g.a.k_gain : g.a.q_gain, f.pos, l);
        f.finish(g, rotation, turn, l);
        f = next;
    }
    if (g.paged) {
        pdl_launch_dependents();
        pdl_wait();
    }
}

template <typename T, int D>
void launch(Args g, cudaStream_t s) {
    using L = Lanes<T, D>;
    const char* what = "vxc_qk_norm_rope";
    int dev = 0, sms = 0;
    paged_ck(cudaGetDevice(&dev), "cudaGetDevice");
    paged_ck(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
    const long long chunks = (static_cast<long long>(g.a.rows) + kChunkRows - 1) / kChunkRows;
    const long long cache = g.paged ? chunks * g.p.kv_heads : 0;
    const size_t keys = g.paged ? static_cast<size_t>(kChunkRows + g.p.page_size) * key_row<T, D>() * sizeof(T) : 0;
    const long long heads = static_cast<long long>(g.a.rows) * (g.a.q_heads + (g.paged ? 0 : g.a.kv_heads));
    const long long few = (heads + L::kSlots - 1) / L::kSlots;
    paged_require(heads <= 0x7fffffffll - (1 << 20) && cache <= 0x3fffffffll, "vxc_qk_norm_rope: too many rows");
    g.cache_ctas = static_cast<int>(cache);
    // Up to 8 CTAs of heads an SM: 753 rows of 16 + 2 heads of 64 fp32 7.6 us. Beyond what their registers and the
    // cached part's shared memory let run at once, CTAs take turns, and the one launch still gains: 1353 rows of 7 + 1
    // fp32 heads of 128 in pages of 128 (2 CTAs an SM) 15.5 us, one row more in two launches 22.
    if (few <= 8ll * sms) {
        allow_dynamic_smem(reinterpret_cast<const void*>(few_rows_kernel<T, D>), keys, what);
        paged_launch(few_rows_kernel<T, D>, static_cast<unsigned>(cache + few), kThreads, keys, s, what, g);
        return;
    }
    if (g.paged) {
        allow_dynamic_smem(reinterpret_cast<const void*>(cache_rows_kernel<T, D>), keys * kCacheHeads, what);
        paged_launch(cache_rows_kernel<T, D>, static_cast<unsigned>(chunks * ((g.p.kv_heads + kCacheHeads - 1) / kCacheHeads)),
                     kThreads, keys * kCacheHeads, s, what, g);
    }
    const auto flat = g.rotation == kNone ? flat_rows_kernel<T, D, kNone>
                      : g.rotation == kPairs ? flat_rows_kernel<T, D, kPairs> : flat_rows_kernel<T, D, kHalves>;
    paged_launch(flat, static_cast<unsigned>(sms * kFlatCtas), kThreads, 0, s, what, g);
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
    paged_require(a->q_out != a->q || a->q_out_stride == a->q_stride || a->rows == 1,
                  "vxc_qk_norm_rope: q_out = q needs the same strides");
    if (p) {
        paged_require(a->v && a->row_seq, "null argument");
        paged_require(aligned16(a->v) && a->v_stride >= k_row && a->v_stride % unit == 0,
                      "vxc_qk_norm_rope: v must be laid out as k");
        check_page_sizes(p);
        paged_require(p->dtype == a->dtype && p->kv_heads == a->kv_heads && p->head_dim == a->head_dim,
                      "vxc_qk_norm_rope: rows and cache differ in dtype, kv_heads or head_dim");
        paged_require(layer >= 0 && layer < p->layers, "vxc_qk_norm_rope: layer out of range");
        check_page_arrays(p);
    } else {
        paged_require(a->k_out != nullptr, "null argument");
        paged_require(aligned16(a->k_out) && a->k_out_stride >= k_row && a->k_out_stride % unit == 0,
                      "vxc_qk_norm_rope: k_out must be laid out as k");
        paged_require(a->k_out != a->k || a->k_out_stride == a->k_stride || a->rows == 1,
                      "vxc_qk_norm_rope: k_out = k needs the same strides");
    }
    DeviceMemory mem("vxc_qk_norm_rope");
    mem.require(a->q, "q");
    mem.require(a->k, "k");
    mem.require(a->q_out, "q_out");
    mem.require(a->q_gain, "q_gain");
    mem.require(a->k_gain, "k_gain");
    mem.require(a->cos, "cos");
    mem.require(a->sin, "sin");
    mem.require(a->row_seq, "row_seq");
    mem.require(a->row_pos, "row_pos");
    mem.require(a->status, "status");
    if (p) {
        mem.require(a->v, "v");
        check_page_memory(p, mem);
    } else {
        mem.require(a->k_out, "k_out");
    }
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
        g.paged = p != nullptr;
        g.rotation = !a->cos ? kNone : a->interleaved ? kPairs : kHalves;
        const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
        const bool wide = a->head_dim == 128;
        if (a->dtype == VXC_F32) wide ? launch<float, 128>(g, cs) : launch<float, 64>(g, cs);
        else if (a->dtype == VXC_F16) wide ? launch<__half, 128>(g, cs) : launch<__half, 64>(g, cs);
        else wide ? launch<__nv_bfloat16, 128>(g, cs) : launch<__nv_bfloat16, 64>(g, cs);
    });
}
