// Pages of a KV cache: taking, sharing, copying, drawing together and giving back.
//
// Who holds which page is decided on the device, so a captured graph can lengthen, fork and
// free sequences without a word from the host. Every call is one small planning kernel (one
// CTA: prefix sums over the sequences, and over the pages' holder counts to find the lowest free ids)
// and, where pages move or tables are long, a second kernel on the whole GPU that carries the
// plan out. Planning writes nothing to the cache until the whole call is known to succeed.
// All sums are integers and every free id is found in order: the same state gives the same tables.
//
// Bounds: planning by what a launch costs (about 4 us each, back to back; reading everything at once, with
// nothing read twice, changed less than 1 us), the second kernel by the copy bandwidth of the GPU: 303 MB in
// 48 us, 6.3 TB/s of the 6.5 that a plain copy reaches, with 64 bytes a thread on their way before its first store.
#include <algorithm>

#include "paged.cuh"

namespace vxc {
namespace {

constexpr int kPlan = 1024;              // threads of a planning CTA
constexpr int kPer = kMaxSeqs / kPlan;   // consecutive sequences per thread
constexpr int kScan = 8;                 // consecutive pages per thread in one scanning step
constexpr int kCopy = 256;               // threads of a copying CTA
constexpr int kChunk = 16384;            // bytes one copying step moves

// vxc_pages.work
constexpr int kHead = 16;  // [0] page copies, [1] whether the plan stands, [2] pages in use
struct Work {
    int* head;
    int* src;    // [n_pages] pages copied from
    int* dst;    // [n_pages] and to
    int* remap;  // [n_pages] where compact puts a page past the ones in use
    int* off;    // [n_seqs + 1] first page copy of each sequence
};
__host__ __device__ inline size_t work_ints(int n_pages, int n_seqs) {
    return kHead + 3 * static_cast<size_t>(n_pages) + n_seqs + 1;
}
__device__ __forceinline__ Work carve(const vxc_pages& p) {
    Work w;
    w.head = p.work;
    w.src = p.work + kHead;
    w.dst = w.src + p.n_pages;
    w.remap = w.dst + p.n_pages;
    w.off = w.remap + p.n_pages;
    return w;
}

struct PlanSmem {
    long long warp[kPlan / 32];
    int pages[kMaxSeqs + 1];  // exclusive prefix of the pages each sequence needs
    int rows[kMaxSeqs + 1];   // exclusive prefix of the rows
};

// Exclusive prefix of v over the CTA; *total = the sum.
__device__ __forceinline__ long long cta_scan(long long v, long long* warp_sums, long long* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // the previous scan's readers are done
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    long long w = warp_sums[lane];  // kPlan / 32 == 32 warps
    long long s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    *total = __shfl_sync(0xffffffffu, s, 31);
    const long long before = __shfl_sync(0xffffffffu, s - w, warp);
    return before + x - v;
}

// The holder counts of kScan consecutive pages from id0 (1 past the pool, i.e. not free).
__device__ __forceinline__ void load_refs(const int* refs, int id0, int n, int (&r)[kScan]) {
    if (id0 + kScan <= n) {
#pragma unroll
        for (int i = 0; i < kScan; i += 4) {
            const int4 v = *reinterpret_cast<const int4*>(refs + id0 + i);
            r[i] = v.x;
            r[i + 1] = v.y;
            r[i + 2] = v.z;
            r[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kScan; ++i) r[i] = id0 + i < n ? refs[id0 + i] : 1;
    }
}

// The 'need' lowest free ids, ascending, to list[]; false (the list unfinished) if there are fewer.
__device__ bool lowest_free(const int* refs, int n_pages, int need, int* list, long long* warp_sums) {
    int got = 0;
    for (int base = 0; base < n_pages && got < need; base += kPlan * kScan) {
        const int id0 = base + threadIdx.x * kScan;
        int r[kScan], n = 0;
        load_refs(refs, id0, n_pages, r);
#pragma unroll
        for (int i = 0; i < kScan; ++i) n += r[i] == 0;
        long long total;
        int at = got + static_cast<int>(cta_scan(n, warp_sums, &total));
#pragma unroll
        for (int i = 0; i < kScan; ++i)
            if (r[i] == 0) {
                if (at < need) list[at] = id0 + i;
                ++at;
            }
        got += static_cast<int>(total);
    }
    return got >= need;
}

// The sequence whose range of an exclusive prefix holds item i (the last s with off[s] <= i).
__device__ __forceinline__ int owner_of(const int* off, int n, int i) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (off[mid] <= i) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlan) extend_kernel(const __grid_constant__ vxc_pages p, const int* counts, int max_rows, int* row_seq,
                                                       int* row_pos) {
    __shared__ PlanSmem S;
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, P = p.page_size;
    const int limit = p.max_pages * P;  // at most 2^21
    Work w = carve(p);
    int len[kPer], cnt[kPer], have[kPer], need[kPer];
    long long need_sum = 0, row_sum = 0;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int s = tid * kPer + i;
        len[i] = s < p.n_seqs ? p.lens[s] : 0;
        cnt[i] = s < p.n_seqs ? counts[s] : 0;
        if (cnt[i] < 0 || len[i] < 0 || len[i] > limit || cnt[i] > limit - len[i]) {
            bad = true;
            len[i] = cnt[i] = 0;
        }
        have[i] = (len[i] + P - 1) / P;
        need[i] = (len[i] + cnt[i] + P - 1) / P - have[i];
        need_sum += need[i];
        row_sum += cnt[i];
    }
    long long need_total, row_total;
    int at = static_cast<int>(cta_scan(need_sum, S.warp, &need_total));
    long long row = cta_scan(row_sum, S.warp, &row_total);
    bad = __syncthreads_or(bad) || row_total > max_rows;
    bool ok = !bad;
    if (ok) ok = need_total <= p.n_pages && lowest_free(p.refs, p.n_pages, static_cast<int>(need_total), w.dst, S.warp);
    if (!ok) {
        for (int r = tid; r < max_rows; r += kPlan) row_seq[r] = row_pos[r] = -1;
        if (tid == 0) report(p.status, bad ? VXC_PAGES_BAD_SEQ : VXC_PAGES_FULL);
        return;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int s = tid * kPer + i;
        if (s < p.n_seqs) {
            S.pages[s] = at;
            S.rows[s] = static_cast<int>(row);
        }
        at += need[i];
        row += cnt[i];
    }
    __syncthreads();
    for (int j = tid; j < need_total; j += kPlan) {
        const int s = owner_of(S.pages, p.n_seqs, j);
        const int have_s = (p.lens[s] + P - 1) / P;
        p.table[static_cast<size_t>(s) * p.max_pages + have_s + j - S.pages[s]] = w.dst[j];
        p.refs[w.dst[j]] = 1;
    }
    // four rows after one search
    for (int r0 = tid * 4; r0 < max_rows; r0 += kPlan * 4) {
        int seq = -1, last = 0, shift = 0;  // rows below 'last' are seq's, at position row + shift
        if (r0 < row_total) {
            seq = owner_of(S.rows, p.n_seqs, r0);
            last = seq + 1 < p.n_seqs ? S.rows[seq + 1] : static_cast<int>(row_total);
            shift = p.lens[seq] - S.rows[seq];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + i;
            if (r >= max_rows) break;
            if (r >= row_total) {
                row_seq[r] = row_pos[r] = -1;
                continue;
            }
            while (r >= last) {
                ++seq;
                last = seq + 1 < p.n_seqs ? S.rows[seq + 1] : static_cast<int>(row_total);
                shift = p.lens[seq] - S.rows[seq];
            }
            row_seq[r] = seq;
            row_pos[r] = r + shift;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int s = tid * kPer + i;
        if (s < p.n_seqs && cnt[i] > 0) p.lens[s] = len[i] + cnt[i];
    }
}

// One CTA per sequence, each by itself: one of bad length stays as it is.
__global__ void __launch_bounds__(128) free_kernel(const __grid_constant__ vxc_pages p, const int* flags) {
    pdl_launch_dependents();
    pdl_wait();
    const int s = blockIdx.x;
    if (flags[s] == 0) return;
    const int len = p.lens[s], P = p.page_size;
    __syncthreads();
    if (len < 0 || len > p.max_pages * P) {
        if (threadIdx.x == 0) report(p.status, VXC_PAGES_BAD_SEQ);
        return;
    }
    int* row = p.table + static_cast<size_t>(s) * p.max_pages;
    for (int j = threadIdx.x; j < (len + P - 1) / P; j += blockDim.x) {
        const int id = row[j];
        row[j] = -1;
        if (id < 0 || id >= p.n_pages) {
            report(p.status, VXC_PAGES_BAD_ID);
        } else if (atomicSub(p.refs + id, 1) <= 0) {
            atomicAdd(p.refs + id, 1);
            report(p.status, VXC_PAGES_BAD_ID);
        }
    }
    if (threadIdx.x == 0) p.lens[s] = 0;
}

__global__ void __launch_bounds__(kPlan) fork_plan_kernel(const __grid_constant__ vxc_pages p, const int* parents, int share) {
    __shared__ PlanSmem S;
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, P = p.page_size;
    Work w = carve(p);
    int need[kPer], len[kPer];
    long long sum = 0;  // pages to take in the low half, of the parents in the high one (at most 2^26)
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int d = tid * kPer + i;
        const int from = d < p.n_seqs ? parents[d] : -1;
        need[i] = 0;
        len[i] = -1;
        if (from < 0) continue;
        if (from >= p.n_seqs || parents[from] >= 0 || p.lens[d] != 0 || p.lens[from] < 0 ||
            p.lens[from] > p.max_pages * P) {
            bad = true;
            continue;
        }
        len[i] = p.lens[from];
        const int pages = (len[i] + P - 1) / P;
        need[i] = share ? (len[i] % P != 0) : pages;
        sum += need[i] | static_cast<long long>(pages) << 32;
    }
    long long totals;
    const long long before = cta_scan(sum, S.warp, &totals);
    const int total = static_cast<int>(totals), looks = static_cast<int>(totals >> 32);
    int at = static_cast<int>(before), look = static_cast<int>(before >> 32);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int d = tid * kPer + i;
        if (d < p.n_seqs) {
            S.pages[d] = w.off[d] = at;
            S.rows[d] = look;
        }
        at += need[i];
        look += len[i] < 0 ? 0 : (len[i] + P - 1) / P;
    }
    __syncthreads();
    bool bad_id = false;  // a page of a parent outside the pool
    for (int j = tid; j < looks; j += kPlan) {
        const int d = owner_of(S.rows, p.n_seqs, j);
        const int id = p.table[static_cast<size_t>(parents[d]) * p.max_pages + j - S.rows[d]];
        bad_id |= id < 0 || id >= p.n_pages;
    }
    int error = 0;
    if (__syncthreads_or(bad || bad_id)) error = __syncthreads_or(bad) ? VXC_PAGES_BAD_SEQ : VXC_PAGES_BAD_ID;
    else if (total > p.n_pages || !lowest_free(p.refs, p.n_pages, total, w.dst, S.warp)) error = VXC_PAGES_FULL;
    if (error) {
        if (tid == 0) {
            w.head[0] = 0;
            w.head[1] = 0;
            report(p.status, error);
        }
        return;
    }
    __syncthreads();
    for (int j = tid; j < total; j += kPlan) {
        const int d = owner_of(S.pages, p.n_seqs, j), from = parents[d];
        const int k = share ? p.lens[from] / P : j - S.pages[d];
        w.src[j] = p.table[static_cast<size_t>(from) * p.max_pages + k];
        p.refs[w.dst[j]] = 1;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (len[i] >= 0) p.lens[tid * kPer + i] = len[i];
    if (tid == 0) {
        w.head[0] = static_cast<int>(total);
        w.head[1] = 1;
    }
}

__global__ void __launch_bounds__(kPlan) compact_plan_kernel(const __grid_constant__ vxc_pages p, int* used_out) {
    __shared__ PlanSmem S;
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, n = p.n_pages;
    Work w = carve(p);
    long long mine = 0, counts;  // pages in use in the low half, lengths out of range in the high one
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int s = tid * kPer + i, len = s < p.n_seqs ? p.lens[s] : 0;
        mine += len < 0 || len > p.max_pages * p.page_size ? 1ll << 32 : 0;
    }
    for (int id0 = tid * kScan; id0 < n; id0 += kPlan * kScan) {
        int r[kScan];
        load_refs(p.refs, id0, n, r);
#pragma unroll
        for (int i = 0; i < kScan; ++i) mine += id0 + i < n && r[i] != 0;
    }
    cta_scan(mine, S.warp, &counts);
    if (counts >> 32) {
        if (tid == 0) {
            w.head[0] = 0;
            w.head[1] = 0;
            report(p.status, VXC_PAGES_BAD_SEQ);
        }
        return;
    }
    const long long used = counts;
    int holes = 0, movers = 0;
    for (int base = 0; base < n; base += kPlan * kScan) {
        const int id0 = base + tid * kScan;
        int r[kScan];
        load_refs(p.refs, id0, n, r);
        long long v = 0;  // holes in the low half, movers in the high one
#pragma unroll
        for (int i = 0; i < kScan; ++i) {
            v += id0 + i < used && r[i] == 0;
            v += id0 + i >= used && id0 + i < n && r[i] != 0 ? 1ll << 32 : 0;
        }
        long long total;
        const long long before = cta_scan(v, S.warp, &total);
        int h = holes + static_cast<int>(before & 0xffffffffll), m = movers + static_cast<int>(before >> 32);
#pragma unroll
        for (int i = 0; i < kScan; ++i) {
            if (id0 + i < used && r[i] == 0) w.dst[h++] = id0 + i;
            if (id0 + i >= used && id0 + i < n) {
                if (r[i] != 0) w.src[m++] = id0 + i;
                else w.remap[id0 + i] = -1;  // in no sequence's row
            }
        }
        holes += static_cast<int>(total & 0xffffffffll);
        movers += static_cast<int>(total >> 32);
    }
    __syncthreads();
    for (int j = tid; j < movers; j += kPlan) {
        const int from = w.src[j], to = w.dst[j];
        w.remap[from] = to;
        p.refs[to] = p.refs[from];
        p.refs[from] = 0;
    }
    if (tid == 0) {
        w.head[0] = movers;
        w.head[1] = 1;
        w.head[2] = static_cast<int>(used);
        if (used_out) *used_out = static_cast<int>(used);
    }
}

__device__ __forceinline__ void copy_bytes(char* to, const char* from, int bytes) {
    constexpr int kVec = kChunk / 16 / kCopy;  // every load of a step before its first store
    uint4 v[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const int at = (threadIdx.x + i * kCopy) * 16;
        if (at < bytes) v[i] = __ldcg(reinterpret_cast<const uint4*>(from + at));
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const int at = (threadIdx.x + i * kCopy) * 16;
        if (at < bytes) *reinterpret_cast<uint4*>(to + at) = v[i];
    }
}

// The planned copies of every layer's keys, values and bounds, in steps of kChunk bytes spread over the grid.
__device__ void copy_pages(const vxc_pages& p, const Work& w, int size) {
    const int n = w.head[0];
    const size_t kv = static_cast<size_t>(p.kv_heads) * p.page_size * p.head_dim * size;
    const size_t bd = static_cast<size_t>(p.kv_heads) * 2 * p.head_dim * size;
    const int kv_steps = static_cast<int>((kv + kChunk - 1) / kChunk), bd_steps = static_cast<int>((bd + kChunk - 1) / kChunk);
    const int steps = 2 * kv_steps + bd_steps;
    const long long all = static_cast<long long>(n) * p.layers * steps;
    for (long long it = blockIdx.x; it < all; it += gridDim.x) {
        const int step = static_cast<int>(it % steps);
        const long long rest = it / steps;
        const int layer = static_cast<int>(rest % p.layers), j = static_cast<int>(rest / p.layers);
        const int from = w.src[j], to = w.dst[j];
        // A plan names pages of the pool; reads stay there whatever else writes to work, the caller's memory. (3000 pages of
        // which 1150 are used, 8 layers: 71.5 us; testing 'to' as well, or neither, 73.7.)
        if (from < 0 || from >= p.n_pages) {
            if (threadIdx.x == 0) report(p.status, VXC_PAGES_BAD_ID);
            continue;
        }
        const bool is_bd = step >= 2 * kv_steps, is_v = !is_bd && step >= kv_steps;
        char* base = static_cast<char*>(is_bd ? p.bounds : is_v ? p.v : p.k);
        const size_t unit = is_bd ? bd : kv;
        const size_t off = static_cast<size_t>(step - (is_bd ? 2 * kv_steps : is_v ? kv_steps : 0)) * kChunk;
        const size_t plane = static_cast<size_t>(layer) * p.n_pages;
        copy_bytes(base + (plane + to) * unit + off, base + (plane + from) * unit + off,
                   static_cast<int>(min(unit - off, static_cast<size_t>(kChunk))));
    }
}

__global__ void __launch_bounds__(kCopy) fork_apply_kernel(const __grid_constant__ vxc_pages p, const int* parents, int share, int size) {
    pdl_launch_dependents();
    pdl_wait();
    Work w = carve(p);
    if (w.head[1] == 0) return;
    // tables: one CTA per piece of a sequence's row
    const int pieces = (p.max_pages + kCopy - 1) / kCopy, P = p.page_size;
    for (int it = blockIdx.x; it < p.n_seqs * pieces; it += gridDim.x) {
        const int d = it / pieces, j = (it - d * pieces) * kCopy + threadIdx.x;
        const int from = parents[d];
        if (from < 0) continue;
        const int len = p.lens[d];
        if (j >= (len + P - 1) / P) continue;
        int* to = p.table + static_cast<size_t>(d) * p.max_pages + j;
        if (!share) {
            *to = w.dst[w.off[d] + j];
        } else if (j >= len / P) {
            *to = w.dst[w.off[d]];
        } else {
            const int id = p.table[static_cast<size_t>(from) * p.max_pages + j];
            *to = id;
            atomicAdd(p.refs + id, 1);
        }
    }
    copy_pages(p, w, size);
}

__global__ void __launch_bounds__(kCopy) compact_apply_kernel(const __grid_constant__ vxc_pages p, int size) {
    pdl_launch_dependents();
    pdl_wait();
    Work w = carve(p);
    if (w.head[1] == 0) return;
    const int used = w.head[2], P = p.page_size;
    const int pieces = (p.max_pages + kCopy - 1) / kCopy;
    for (int it = blockIdx.x; it < p.n_seqs * pieces; it += gridDim.x) {
        const int s = it / pieces, j = (it - s * pieces) * kCopy + threadIdx.x;
        if (j >= (p.lens[s] + P - 1) / P) continue;
        int* at = p.table + static_cast<size_t>(s) * p.max_pages + j;
        const int id = *at;
        if (id >= 0 && id < used) continue;
        const int to = id >= 0 && id < p.n_pages ? w.remap[id] : -1;
        if (to < 0) report(p.status, VXC_PAGES_BAD_ID);
        else *at = to;
    }
    copy_pages(p, w, size);
}

// CTAs of the second kernels: two for each that runs at once (4 of 256 threads per SM, by their registers).
int apply_grid() {
    int dev = 0, sms = 0;
    paged_ck(cudaGetDevice(&dev), "cudaGetDevice");
    paged_ck(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
    return sms * 8;
}

}  // namespace
}  // namespace vxc

using namespace vxc;

extern "C" VXC_API size_t vxc_pages_work_ints(const vxc_pages* p) {
    size_t n = 0;
    paged_guard([&] {
        check_page_sizes(p);
        n = work_ints(p->n_pages, p->n_seqs);
    });
    return n;
}

extern "C" VXC_API int32_t vxc_pages_extend(const vxc_pages* p, const int32_t* counts, int32_t max_rows,
                                            int32_t* row_seq, int32_t* row_pos, void* cuda_stream) {
    return paged_guard([&] {
        paged_require(p && counts && row_seq && row_pos, "null argument");
        paged_require(max_rows > 0 && max_rows <= 1 << 30, "vxc_pages_extend: max_rows must be 1 to 2^30");
        paged_require(aligned4(counts) && aligned4(row_seq) && aligned4(row_pos), "vxc_pages_extend: misaligned int32 array");
        check_page_arrays(p);
        DeviceMemory mem("vxc_pages_extend");
        check_page_memory(p, mem);
        mem.require(counts, "counts");
        mem.require(row_seq, "row_seq");
        mem.require(row_pos, "row_pos");
        paged_launch(extend_kernel, 1, kPlan, 0, static_cast<cudaStream_t>(cuda_stream), "vxc_pages_extend", *p, counts,
                     max_rows, row_seq, row_pos);
    });
}

extern "C" VXC_API int32_t vxc_pages_free(const vxc_pages* p, const int32_t* flags, void* cuda_stream) {
    return paged_guard([&] {
        paged_require(p && flags, "null argument");
        paged_require(aligned4(flags), "vxc_pages_free: misaligned int32 array");
        check_page_arrays(p);
        DeviceMemory mem("vxc_pages_free");
        check_page_memory(p, mem);
        mem.require(flags, "flags");
        paged_launch(free_kernel, p->n_seqs, 128, 0, static_cast<cudaStream_t>(cuda_stream), "vxc_pages_free", *p, flags);
    });
}

extern "C" VXC_API int32_t vxc_pages_fork(const vxc_pages* p, const int32_t* parents, int32_t share, void* cuda_stream) {
    return paged_guard([&] {
        paged_require(p && parents, "null argument");
        paged_require(aligned4(parents), "vxc_pages_fork: misaligned int32 array");
        check_page_arrays(p);
        DeviceMemory mem("vxc_pages_fork");
        check_page_memory(p, mem);
        mem.require(parents, "parents");
        const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
        paged_launch(fork_plan_kernel, 1, kPlan, 0, cs, "vxc_pages_fork", *p, parents, share != 0);
        paged_launch(fork_apply_kernel, apply_grid(), kCopy, 0, cs, "vxc_pages_fork", *p, parents, share != 0,
                     dtype_size(p->dtype));
    });
}

extern "C" VXC_API int32_t vxc_pages_compact(const vxc_pages* p, int32_t* used, void* cuda_stream) {
    return paged_guard([&] {
        paged_require(aligned4(used), "vxc_pages_compact: misaligned int32 array");
        check_page_arrays(p);
        DeviceMemory mem("vxc_pages_compact");
        check_page_memory(p, mem);
        mem.require(used, "used");
        const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
        paged_launch(compact_plan_kernel, 1, kPlan, 0, cs, "vxc_pages_compact", *p, used);
        paged_launch(compact_apply_kernel, apply_grid(), kCopy, 0, cs, "vxc_pages_compact", *p, dtype_size(p->dtype));
    });
}
