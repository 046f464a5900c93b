// Moving pages of a KV pool on gfx950: copies, block-table renames, freed pages' marks.
//
// A pool is one or two regions of `layers` x `pages` runs of bytes (K and V together, K and V apart,
// or an 8-bit pool's data and its codes); a page is its run in every layer of every region. The page
// ids come from the host with the call and travel in the kernel arguments, up to kBatch pairs per
// launch, so a call makes no copy to the device and can be captured.
//
// The copies replace GpuKVBlockPool.copy_blocks (runtime/phase2/paged_kv_kernel.py:233-250), whose
// torch form gathers every page into a temporary and scatters it: twice the bytes.
#include <algorithm>
#include <vector>

#include "common.h"

namespace mx {
namespace pages {

constexpr int kBatch = 448;    // page pairs per launch: 3.5 KiB of the 4 KiB of kernel arguments
constexpr int kThreads = 256;
constexpr int kMaxPairs = 1 << 24;  // of one call: its lists are hashed on the host

struct Region {
    char* base;
    int64_t layer_stride, bytes;  // bytes between layers; bytes of one page in one layer
};

struct CopyParams {
    Region r[2];
    int layers;
    int slices;  // workgroups per (pair, layer)
    int move;    // sources are free afterwards: their marks go with the pages
    uint8_t* used;  // optional [pages]: 1 where a page was written
    int2 pair[kBatch];
};

// One workgroup copies its slice of one page in one layer, both regions; 16 bytes a thread and step
// where the page's size allows, else single bytes (an 8-bit pool's codes).
__device__ __forceinline__ void copy_run(const Region& r, int layer, int src, int dst, int slice, int slices) {
    if (r.bytes == 0) return;
    const char* s = r.base + layer * r.layer_stride + src * r.bytes;
    char* d = r.base + layer * r.layer_stride + dst * r.bytes;
    const int64_t step = (int64_t)slices * kThreads, first = (int64_t)slice * kThreads + threadIdx.x;
    if (r.bytes % 16 == 0) {
        for (int64_t i = first; i < r.bytes / 16; i += step)
            reinterpret_cast<uint4*>(d)[i] = reinterpret_cast<const uint4*>(s)[i];
    } else {
        for (int64_t i = first; i < r.bytes; i += step) d[i] = s[i];
    }
}

__global__ __launch_bounds__(kThreads) void copy_pages_kernel(CopyParams p) {
    const int slice = blockIdx.x, layer = blockIdx.y;
    const int2 pr = p.pair[blockIdx.z];
    if (p.used && slice == 0 && layer == 0 && threadIdx.x == 0) {
        p.used[pr.y] = p.move ? p.used[pr.x] : 1;
        if (p.move) p.used[pr.x] = 0;
    }
    copy_run(p.r[0], layer, pr.x, pr.y, slice, p.slices);
    copy_run(p.r[1], layer, pr.x, pr.y, slice, p.slices);
}

// The same for pairs whose pages depend on each other (a page that is read by one pair and written by
// another): every thread does all of them in the order given, on its own bytes of each page, so no
// order between threads is needed. pair {s, -1} keeps page s's bytes, {-1, d} writes the kept ones.
template <typename V>
__device__ __forceinline__ void copy_ordered(const CopyParams& p, const Region& r, int n, int layer, int slice) {
    char* base = r.base + layer * r.layer_stride;
    const int64_t step = (int64_t)p.slices * kThreads, first = (int64_t)slice * kThreads + threadIdx.x;
    for (int64_t i = first; i < r.bytes / (int64_t)sizeof(V); i += step) {
        V kept{};
        for (int k = 0; k < n; ++k) {
            const int2 pr = p.pair[k];
            V v = kept;
            if (pr.x >= 0) v = reinterpret_cast<const V*>(base + pr.x * r.bytes)[i];
            if (pr.y >= 0) reinterpret_cast<V*>(base + pr.y * r.bytes)[i] = v;
            else kept = v;
        }
    }
}

__global__ __launch_bounds__(kThreads) void copy_ordered_kernel(CopyParams p, int n) {
    if (p.used && blockIdx.x == 0 && blockIdx.y == 0)
        for (int k = threadIdx.x; k < n; k += kThreads)
            if (p.pair[k].y >= 0) p.used[p.pair[k].y] = 1;
    for (int i = 0; i < 2; ++i) {
        if (p.r[i].bytes % 16 == 0) copy_ordered<uint4>(p, p.r[i], n, blockIdx.y, blockIdx.x);
        else copy_ordered<uint8_t>(p, p.r[i], n, blockIdx.y, blockIdx.x);
    }
}

struct RenameParams {
    const int32_t* in;
    int32_t* out;
    int64_t in_sb, out_sb;
    int rows, width, n;
    int2 pair[kBatch];  // ascending by x
};

// Block tables with every id of the list renamed, the others as they are. A thread finds its id by
// bisection in the sorted list (at most 9 steps over the kernel argument's copy in LDS).
__global__ __launch_bounds__(kThreads) void rename_kernel(RenameParams p) {
    __shared__ int2 list[kBatch];
    for (int i = threadIdx.x; i < p.n; i += kThreads) list[i] = p.pair[i];
    __syncthreads();
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= (int64_t)p.rows * p.width) return;
    const int64_t b = i / p.width, c = i - b * p.width;
    const int id = p.in[b * p.in_sb + c];
    int lo = 0, hi = p.n;  // the first entry not below id
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (list[mid].x < id) lo = mid + 1;
        else hi = mid;
    }
    p.out[b * p.out_sb + c] = lo < p.n && list[lo].x == id ? list[lo].y : id;
}

struct ClearParams {
    Region r;       // bytes to zero (an 8-bit pool's codes); bytes = 0: none
    int layers;
    uint8_t* used;  // optional [pages]: marks to zero
    int n;
    int id[2 * kBatch];
};
static_assert(sizeof(CopyParams) < 4000 && sizeof(RenameParams) < 4000 && sizeof(ClearParams) < 4000,
              "kernel arguments");

__global__ __launch_bounds__(kThreads) void clear_kernel(ClearParams p) {
    const int id = p.id[blockIdx.x];
    if (p.used && threadIdx.x == 0) p.used[id] = 0;
    const int64_t total = p.r.bytes * p.layers;
    for (int64_t i = threadIdx.x; i < total; i += kThreads) {
        const int64_t layer = i / p.r.bytes;
        p.r.base[layer * p.r.layer_stride + id * p.r.bytes + (i - layer * p.r.bytes)] = 0;
    }
}

// Page id -> number, for n ids: open addressing over at least 4 n slots (a call's host work is a few
// microseconds where sorts of the lists took 25 for 384 pairs).
class IdMap {
   public:
    explicit IdMap(size_t n) {
        while (((size_t)1 << bits_) < 4 * n) ++bits_;
        slots_.assign((size_t)1 << bits_, int2{-1, -1});
    }
    void set(int id, int value) { *find(id) = int2{id, value}; }
    int get(int id) const {
        const int2* s = const_cast<IdMap*>(this)->find(id);
        return s->x == id ? s->y : -1;
    }

   private:
    int2* find(int id) {
        for (size_t i = ((uint32_t)id * 2654435761u) >> (32 - bits_);; i = (i + 1) & (slots_.size() - 1))
            if (slots_[i].x == id || slots_[i].x == -1) return &slots_[i];
    }
    int bits_ = 3;
    std::vector<int2> slots_;
};

// The pairs of (src, dst) that copy something, of several with one dst the last, split into independent
// ones and an ordered list for copy_ordered: a pair that reads a page comes before the one that writes
// it, a cycle is opened by keeping one page.
static void order_pairs(const int32_t* src, const int32_t* dst, int n, std::vector<int2>& free_pairs,
                        std::vector<int2>& ordered) {
    IdMap writer(n), reader(n);  // a page's last pair in the lists; whether a counted pair reads it
    for (int i = 0; i < n; ++i) writer.set(dst[i], i);
    auto counts = [&](int i) { return src[i] != dst[i] && writer.get(dst[i]) == i; };
    for (int i = 0; i < n; ++i)
        if (counts(i)) reader.set(src[i], 1);
    std::vector<int2> rest;
    for (int i = 0; i < n; ++i) {
        if (!counts(i)) continue;
        const int w = writer.get(src[i]);
        const bool tied = (w >= 0 && counts(w)) || reader.get(dst[i]) >= 0;
        (tied ? rest : free_pairs).push_back(int2{src[i], dst[i]});
    }
    if (rest.empty()) return;
    IdMap of(rest.size());  // page -> the pair of rest that writes it
    for (size_t i = 0; i < rest.size(); ++i) of.set(rest[i].y, (int)i);
    std::vector<int> readers(rest.size(), 0), ready;  // readers: pairs not yet done that read the pair's dst
    std::vector<char> done(rest.size(), 0);
    for (const int2& p : rest) {
        const int w = of.get(p.x);
        if (w >= 0) ++readers[w];
    }
    for (size_t i = 0; i < rest.size(); ++i)
        if (readers[i] == 0) ready.push_back((int)i);
    while (!ready.empty()) {
        const int i = ready.back();
        ready.pop_back();
        ordered.push_back(rest[i]);
        done[i] = 1;
        const int w = of.get(rest[i].x);  // the pair that overwrites what was just read
        if (w >= 0 && --readers[w] == 0) ready.push_back(w);
    }
    // What is left are cycles, each page read once: a1 <- a0, a2 <- a1, ..., a0 <- ak.
    for (size_t i = 0; i < rest.size(); ++i) {
        if (done[i]) continue;
        const int kept = rest[i].y;
        ordered.push_back(int2{kept, -1});
        int w = (int)i;
        while (rest[w].x != kept) {  // write a page, then the one that was just read
            ordered.push_back(rest[w]);
            done[w] = 1;
            w = of.get(rest[w].x);
        }
        ordered.push_back(int2{-1, rest[w].y});
        done[w] = 1;
    }
}

static int check_region(const char* what, const Region& r, bool required) {
    if (!r.base) return required ? fail(MX_ERR_NULL, "%s: null pointer", what) : MX_OK;
    if (r.bytes < 1) return fail(MX_ERR_INVALID, "%s: a page must have bytes", what);
    if (r.bytes % 16 == 0 && (!aligned(r.base, 16) || r.layer_stride % 16))
        return fail(MX_ERR_ALIGNMENT, "%s: pages must be 16-byte aligned", what);
    return MX_OK;
}

}  // namespace pages
}  // namespace mx

using namespace mx;

extern "C" int mx_kv_copy_pages(void* base, int64_t page_bytes, int64_t layer_stride, void* base2,
                                int64_t page_bytes2, int64_t layer_stride2, int32_t layers, int32_t num_pages,
                                const int32_t* src, const int32_t* dst, int32_t n, uint8_t* used, int32_t move,
                                void* stream) {
    const char* what = "mx_kv_copy_pages";
    if (n < 0) return fail(MX_ERR_INVALID, "%s: n must be >= 0", what);
    if (n == 0) return MX_OK;
    if (!src || !dst) return fail(MX_ERR_NULL, "%s: null pointer", what);
    if (layers < 1 || layers > 65535 || num_pages < 1) return fail(MX_ERR_INVALID, "%s: layers or pages out of range", what);
    if (n > pages::kMaxPairs) return fail(MX_ERR_UNSUPPORTED, "%s: more than %d pairs", what, pages::kMaxPairs);
    pages::CopyParams p{};
    p.r[0] = {static_cast<char*>(base), layer_stride, page_bytes};
    p.r[1] = {static_cast<char*>(base2), layer_stride2, base2 ? page_bytes2 : 0};
    int rc = pages::check_region(what, p.r[0], true);
    if (rc == MX_OK) rc = pages::check_region(what, p.r[1], false);
    if (rc != MX_OK) return rc;
    for (int i = 0; i < n; ++i)
        if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages)
            return fail(MX_ERR_INVALID, "%s: page id out of range: %d -> %d", what, src[i], dst[i]);
    try {
        std::vector<int2> ordered, free_pairs;
        pages::order_pairs(src, dst, n, free_pairs, ordered);
        if (move && free_pairs.size() != (size_t)n)
            return fail(MX_ERR_INVALID, "%s: a moved page occurs twice in the lists", what);
        if (move) {
            pages::IdMap seen(n);
            for (int i = 0; i < n; ++i) {
                if (seen.get(src[i]) >= 0) return fail(MX_ERR_INVALID, "%s: page %d is moved twice", what, src[i]);
                seen.set(src[i], 1);
            }
        }
        if (ordered.size() > (size_t)pages::kBatch)
            return fail(MX_ERR_UNSUPPORTED, "%s: more than %d copies depend on each other", what, pages::kBatch);
        p.layers = layers;
        p.used = used;
        p.move = move != 0;
        const int64_t most = std::max(p.r[0].bytes / (p.r[0].bytes % 16 ? 1 : 16), p.r[1].bytes / (p.r[1].bytes % 16 ? 1 : 16));
        p.slices = (int)std::min<int64_t>(std::max<int64_t>(ceil_div(most, pages::kThreads * 4), 1), 64);
        for (size_t i = 0; i < free_pairs.size(); i += pages::kBatch) {
            const size_t m = std::min<size_t>(pages::kBatch, free_pairs.size() - i);
            std::copy(free_pairs.begin() + i, free_pairs.begin() + i + m, p.pair);
            hipLaunchKernelGGL(pages::copy_pages_kernel, dim3(p.slices, layers, m), dim3(pages::kThreads), 0,
                               as_stream(stream), p);
        }
        if (!ordered.empty()) {
            std::copy(ordered.begin(), ordered.end(), p.pair);
            hipLaunchKernelGGL(pages::copy_ordered_kernel, dim3(p.slices, layers), dim3(pages::kThreads), 0,
                               as_stream(stream), p, (int)ordered.size());
        }
    } catch (...) {
        return fail(MX_ERR_INVALID, "%s: out of host memory", what);
    }
    return check_launch(what);
}

extern "C" int mx_kv_rename_pages(const int32_t* tables, int64_t in_stride, int32_t* out, int64_t out_stride,
                                  int32_t rows, int32_t width, const int32_t* from, const int32_t* to, int32_t n,
                                  void* stream) {
    const char* what = "mx_kv_rename_pages";
    if (rows < 0 || width < 0 || n < 0) return fail(MX_ERR_INVALID, "%s: sizes must be >= 0", what);
    if (rows == 0 || width == 0) return MX_OK;
    if (!tables || !out || (n > 0 && (!from || !to))) return fail(MX_ERR_NULL, "%s: null pointer", what);
    if ((int64_t)rows * width >= ((int64_t)1 << 31)) return fail(MX_ERR_UNSUPPORTED, "%s: tables too large", what);
    if (n > pages::kMaxPairs) return fail(MX_ERR_UNSUPPORTED, "%s: more than %d pairs", what, pages::kMaxPairs);
    try {
        std::vector<int2> list(n);
        pages::IdMap old(n);
        for (int i = 0; i < n; ++i) {
            if (from[i] < 0) return fail(MX_ERR_INVALID, "%s: id %d", what, from[i]);
            if (old.get(from[i]) >= 0) return fail(MX_ERR_INVALID, "%s: id %d twice", what, from[i]);
            old.set(from[i], 1);
            list[i] = int2{from[i], to[i]};
        }
        // Lists longer than a launch holds go one after another: no new name may be an old one.
        for (int i = 0; i < n; ++i)
            if (to[i] >= 0 && old.get(to[i]) >= 0)
                return fail(MX_ERR_INVALID, "%s: id %d is both renamed and a new name", what, to[i]);
        auto below = [](int2 a, int2 b) { return a.x < b.x; };
        if (!std::is_sorted(list.begin(), list.end(), below)) std::sort(list.begin(), list.end(), below);
        pages::RenameParams p{tables, out, in_stride, out_stride, rows, width, 0, {}};
        int i = 0;
        do {
            p.n = std::min(pages::kBatch, n - i);
            std::copy(list.begin() + i, list.begin() + i + p.n, p.pair);
            hipLaunchKernelGGL(pages::rename_kernel, dim3((unsigned)ceil_div((int64_t)rows * width, pages::kThreads)),
                               dim3(pages::kThreads), 0, as_stream(stream), p);
            p.in = out;
            p.in_sb = out_stride;
            i += p.n;
        } while (i < n);
    } catch (...) {
        return fail(MX_ERR_INVALID, "%s: out of host memory", what);
    }
    return check_launch(what);
}

extern "C" int mx_kv_clear_pages(uint8_t* codes, int64_t page_bytes, int64_t layer_stride, int32_t layers,
                                 uint8_t* used, int32_t num_pages, const int32_t* ids, int32_t n, void* stream) {
    const char* what = "mx_kv_clear_pages";
    if (n < 0) return fail(MX_ERR_INVALID, "%s: n must be >= 0", what);
    if (n == 0) return MX_OK;
    if (!ids || (!codes && !used)) return fail(MX_ERR_NULL, "%s: null pointer", what);
    if (codes && (layers < 1 || page_bytes < 1)) return fail(MX_ERR_INVALID, "%s: layers and page_bytes must be >= 1", what);
    for (int i = 0; i < n; ++i)
        if (ids[i] < 0 || ids[i] >= num_pages) return fail(MX_ERR_INVALID, "%s: page id out of range: %d", what, ids[i]);
    pages::ClearParams p{{reinterpret_cast<char*>(codes), layer_stride, codes ? page_bytes : 0}, layers, used, 0, {}};
    for (int i = 0; i < n; i += p.n) {
        p.n = std::min(2 * pages::kBatch, n - i);
        std::copy(ids + i, ids + i + p.n, p.id);
        hipLaunchKernelGGL(pages::clear_kernel, dim3(p.n), dim3(pages::kThreads), 0, as_stream(stream), p);
    }
    return check_launch(what);
}
