// kv_pages.cu -- the paged cache's bookkeeping on the device: page tables, lengths and the number of
// holders of every page, forked, resized and compacted, and the pages copied that this takes, in all
// layers.  Nothing comes back to the host in between, so that a captured graph can hold a step's bookkeeping.
//
// Every call is two kernels.  The first, one block, decides: it reads the lengths and holders as they
// stand, finds the lowest free pages, and writes new lengths, a list of page copies and what the tables
// get.  The second, the whole GPU, rewrites the tables and copies the pages.  Lengths, holders and free
// pages are read as they were before the call, for all items: one that cuts inside a page takes a copy where
// others held it then, and what one item gives back serves no other of the call.  Only the free pages go round
// in the items' order, by a prefix sum over them; holders are counted in whole numbers, in any order.
//
// Both are launched early (kv_launch.h): a call's second kernel, and the next call's first, wait for the one before
// them on the GPU.
// Bound by: the copies' bytes (read once, written once) where there are many, or else two launches and
// the first kernel's walk over the holders.
//
// Measured in a graph: half of 96 conversations gone, 728 MB moved down in 8 layers 245 us (5.9 TB/s, 91 % of the copy
// rate); 144 forks of 9 prompts, 87 MB of partly filled pages in 12 layers with the children let go before and grown
// after 43 us (the copies 22); four forks in three layers, likewise three calls, 17 us.
#include "block_scan.cuh"
#include "kv_launch.h"

namespace hc {

namespace {

constexpr int kPlanThreads = 1024, kItems = HC_KV_SEQS, kWorkThreads = 256;
static_assert(kItems == 2 * kPlanThreads, "two items to a thread");

constexpr int kRun = 8;  // pages of a thread at a time

// The lowest `need` pages that nobody holds into p.free, in order; returns how many there are (at most
// `need`, or some more that the last stretch had).
__device__ int find_free(const PagesDev& p, long long need, long long* scratch) {
    int found = 0;
    for (int b = 0; b < p.n_pages && found < need; b += kPlanThreads * kRun) {
        const int first = b + threadIdx.x * kRun;
        int r[kRun], n = 0;
#pragma unroll
        for (int i = 0; i < kRun; ++i) r[i] = first + i < p.n_pages ? p.refs[first + i] : 1;
#pragma unroll
        for (int i = 0; i < kRun; ++i) n += r[i] <= 0;
        int total, at = block_scan(n, scratch, total);
        at += found;
#pragma unroll
        for (int i = 0; i < kRun; ++i)
            if (r[i] <= 0) p.free[at++] = first + i;
        found += total;
    }
    return found;
}

// Which of the call's items is the first with its slot: a table of places by slot, open addressing.
struct Claims {
    static constexpr int kSize = 2 * kItems;
    int key[kSize], first[kSize];
    __device__ void clear() {
        for (int i = threadIdx.x; i < kSize; i += kPlanThreads) key[i] = -1, first[i] = kItems;
        __syncthreads();
    }
    __device__ int find(int slot, bool add) {
        unsigned h = (unsigned)slot * 2654435761u >> 20;
        static_assert(kSize == 4096, "20 bits fewer");
        for (;;) {
            const int k = add ? atomicCAS(&key[h], -1, slot) : key[h];
            if (k == slot || k == -1) return (int)h;
            h = (h + 1) & (kSize - 1);
        }
    }
    __device__ void claim(int slot, int item) { atomicMin(&first[find(slot, true)], item); }
    __device__ bool mine(int slot, int item) { return first[find(slot, false)] == item; }
};

__device__ __forceinline__ int pages_of(const PagesDev& p, int len) { return p.by_page(len + p.page_size - 1); }

// Can a slot's table have so many tokens?
__device__ __forceinline__ bool len_fits(const PagesDev& p, int n) { return n >= 0 && n <= p.max_pages * p.page_size; }
__device__ __forceinline__ int* slot_table(const PagesDev& p, int slot) { return p.table + slot * p.stride; }

// An item as the first kernel leaves it to the second (PagesDev::item): the slots and pages it is about.
enum { kSlot, kFrom, kHad, kGet };

// fork: children get the parents' whole pages and a page of their own for the rest.
// resize: slots get new lengths.
template <bool FORK>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PagesDev p, const int* first, const int* second, int n) {
    __shared__ long long scratch[33];
    __shared__ int moves_s;
    __shared__ Claims claims;
    after_previous();
    let_next_start();
    if (threadIdx.x == 0) moves_s = 0;
    claims.clear();
    struct Item {
        int slot = -1, from = -1;  // the slot that changes; the one whose pages it gets
        int old = 0, len = 0, had = 0, get = 0, need = 0, keep = 0, part = -1;
    } it[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = 2 * threadIdx.x + e;
        if (i >= n) continue;
        const int a = first[i], b = second[i], slot = FORK ? b : a;
        const bool ok = (unsigned)slot < (unsigned)p.n_slots &&
                        (FORK ? (unsigned)a < (unsigned)p.n_slots : len_fits(p, b));
        if (!ok) {
            atomicOr(p.err, kErrKvRange);
            continue;
        }
        claims.claim(slot, i);
        it[e].slot = slot;
        it[e].from = FORK ? a : slot;
    }
    __syncthreads();
    long long need = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        Item& x = it[e];
        const int i = 2 * threadIdx.x + e;
        if (x.slot < 0) continue;
        bool ok = claims.mine(x.slot, i);
        int whole = 0;
        if (ok) {
            x.old = p.len[x.slot];
            x.len = FORK ? p.len[x.from] : second[i];
            ok = len_fits(p, x.old) && len_fits(p, x.len) && !(FORK && x.old);  // a child holds nothing
        }
        if (ok) {
            // the tokens kept, and the page that the last of them share with the next ones
            x.keep = FORK ? x.len : min(x.old, x.len);
            whole = p.by_page(x.keep);
            if (x.keep - whole * p.page_size) {
                const int page = slot_table(p, x.from)[whole];
                ok = (unsigned)page < (unsigned)p.n_pages;
                if (ok && (FORK || p.refs[page] > 1)) x.part = page;
            }
        }
        if (!ok) {
            atomicOr(p.err, kErrKvRange);
            x.slot = -1;
            continue;
        }
        x.had = FORK ? 0 : pages_of(p, x.old);
        x.get = FORK ? whole : pages_of(p, x.len);
        x.need = (FORK ? 0 : max(x.get - x.had, 0)) + (x.part >= 0);
        need += x.need;
    }
    long long total, at = block_scan(need, scratch, total);
    const int found = total ? find_free(p, total, scratch) : 0;
    __syncthreads();  // all that was to be read of lengths, holders and tables is read, and the free pages are written
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        Item& x = it[e];
        const int i = 2 * threadIdx.x + e;
        if (i >= n) continue;
        const long long mine = at;
        at += x.need;
        if (x.slot >= 0 && x.need && mine + x.need > found) {  // no pages left for it: it stays as it was
            atomicOr(p.err, kErrKvFull);
            x.slot = -1;
        }
        p.item[kSlot * kItems + i] = x.slot;
        if (x.slot < 0) continue;
        const bool part = x.part >= 0;
        if (part) {
            const int page = p.free[mine], whole = p.by_page(x.keep), m = atomicAdd(&moves_s, 1);
            slot_table(p, x.slot)[whole] = page;
            p.refs[page] = 1;
            if (!FORK) atomicSub(&p.refs[x.part], 1);
            p.src[m] = x.part;
            p.dst[m] = page;
            p.rows[m] = x.keep - whole * p.page_size;
        }
        p.len[x.slot] = x.len;
        p.item[kFrom * kItems + i] = FORK ? x.from : (int)mine + part;  // resize: its first page in the free ones
        p.item[kHad * kItems + i] = x.had;
        p.item[kGet * kItems + i] = x.get;
    }
    __syncthreads();
    if (threadIdx.x == 0) *p.moves = moves_s;
}

// Where compacting moves pages: those held of numbers `used` and more to the free ones below, both in order.
__global__ void __launch_bounds__(kPlanThreads) plan_compact_kernel(PagesDev p, int* moved) {
    __shared__ long long scratch[33];
    after_previous();
    let_next_start();
    int n = 0, used;
    for (int b = 0; b < p.n_pages; b += kPlanThreads * kRun)
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const int q = b + i * kPlanThreads + threadIdx.x;
            n += q < p.n_pages && p.refs[q] > 0;
        }
    block_scan(n, scratch, used);
    int holes = 0, movers = 0;
    for (int b = 0; b < p.n_pages; b += kPlanThreads * kRun) {
        const int first = b + threadIdx.x * kRun;
        int r[kRun], total, h = 0, m = 0;
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const int q = first + i;
            r[i] = q < p.n_pages ? p.refs[q] : 0;
            h += q < used && r[i] <= 0;
            m += q >= used && r[i] > 0;
        }
        int at = holes + block_scan(h, scratch, total);
        holes += total;
#pragma unroll
        for (int i = 0; i < kRun; ++i)
            if (first + i < used && r[i] <= 0) p.dst[at++] = first + i;
        at = movers + block_scan(m, scratch, total);  // (its barriers stand between the holes' numbers and their use)
        movers += total;
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const int q = first + i;
            if (q >= p.n_pages) continue;
            int to = q;
            if (q >= used && r[i] > 0) {
                to = p.dst[at];
                p.src[at++] = q;
                p.refs[to] = r[i];
                p.refs[q] = 0;
            }
            moved[q] = to;
        }
    }
    if (threadIdx.x == 0) *p.moves = movers;
}

enum Work { kForkWork, kResizeWork, kCompactWork, kCopyWork };

// The tables of the call's items, a block to 256 pages of one; then the copies, a warp to a head's rows of a
// page, of keys or values, of a layer.
template <int WORK>
__global__ void __launch_bounds__(kWorkThreads) work_kernel(PagesDev p, const __grid_constant__ KvLayers y, int n,
                                                            const int* moved) {
    after_previous();
    let_next_start();
    const int runs = (p.max_pages + kWorkThreads - 1) / kWorkThreads;
    if constexpr (WORK != kCopyWork)
        for (long long w = blockIdx.x; w < (long long)n * runs; w += gridDim.x) {
            const int i = (int)(w / runs), j = (int)(w - (long long)i * runs) * kWorkThreads + threadIdx.x;
            if constexpr (WORK == kCompactWork) {
                int* const t = slot_table(p, i);
                // of a length that does not fit, what the table can have: entries in use are not to name what has moved
                const int len = p.len[i], held = min(max(len, 0), p.max_pages * p.page_size);
                if (held != len) atomicOr(p.err, kErrKvRange);
                if (j >= pages_of(p, held)) continue;
                const int page = t[j];
                if ((unsigned)page < (unsigned)p.n_pages) {
                    const int to = moved[page];
                    if (to != page) t[j] = to;
                } else {
                    atomicOr(p.err, kErrKvRange);
                }
            } else {
                const int slot = p.item[kSlot * kItems + i];
                if (slot < 0) continue;
                const int from = p.item[kFrom * kItems + i], had = p.item[kHad * kItems + i], get = p.item[kGet * kItems + i];
                int* const t = slot_table(p, slot);
                if constexpr (WORK == kForkWork) {
                    if (j >= get) continue;
                    const int page = slot_table(p, from)[j];
                    t[j] = page;
                    if ((unsigned)page < (unsigned)p.n_pages)
                        atomicAdd(&p.refs[page], 1);
                    else
                        atomicOr(p.err, kErrKvRange);
                } else if (j >= had && j < get) {
                    const int page = p.free[from + j - had];
                    t[j] = page;
                    p.refs[page] = 1;
                } else if (j >= get && j < had) {
                    const int page = t[j];
                    if ((unsigned)page >= (unsigned)p.n_pages)
                        atomicOr(p.err, kErrKvRange);
                    else if (atomicSub(&p.refs[page], 1) <= 0) {  // nobody held it
                        atomicAdd(&p.refs[page], 1);
                        atomicOr(p.err, kErrKvRange);
                    }
                }
            }
        }
    const int cpr = y.row_bytes / 16, per = 2 * y.n_heads, ln = lane_id();
    const int shift = 31 - __clz(cpr);  // 4, 8 or 16
    const long long items = (long long)*p.moves * y.n * per;
    for (long long w = ((long long)blockIdx.x * kWorkThreads + threadIdx.x) >> 5; w < items;
         w += (long long)gridDim.x * (kWorkThreads / 32)) {
        const long long ml = w / per;
        const int hw = (int)(w - ml * per), v = hw >= y.n_heads, head = v ? hw - y.n_heads : hw;
        const int m = (int)(ml / y.n), layer = (int)(ml - (long long)m * y.n);
        const int src = p.src[m], dst = p.dst[m], rows = WORK == kCompactWork || !p.rows ? p.page_size : p.rows[m];
        uint8_t* const base = (v ? y.v : y.k)[layer];
        const uint8_t* const from = base + 64ull * ((uint32_t)src * y.page + (uint32_t)head * y.head);
        uint8_t* const to = base + 64ull * ((uint32_t)dst * y.page + (uint32_t)head * y.head);
        const int chunks = rows << shift;
        constexpr int U = 8;
        for (int c0 = ln; c0 < chunks; c0 += 32 * U) {
            uint4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + 32 * u;
                if (c < chunks)
                    x[u] = *reinterpret_cast<const uint4*>(from + 64ull * ((uint32_t)(c >> shift) * y.row) + (c & (cpr - 1)) * 16);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + 32 * u;
                if (c < chunks)
                    *reinterpret_cast<uint4*>(to + 64ull * ((uint32_t)(c >> shift) * y.row) + (c & (cpr - 1)) * 16) = x[u];
            }
        }
        float* const sc = (v ? y.vs : y.ks)[layer];
        if (sc) {
            const float* const sf = sc + src * y.spage + (long long)head * p.page_size;
            float* const st = sc + dst * y.spage + (long long)head * p.page_size;
            for (int r = ln; r < rows; r += 32) st[r] = sf[r];
        }
    }
}

// The second kernel for the first kMaxLayers layers, and the copies of the others.
template <int WORK>
cudaError_t work(const PagesDev& p, const KvLayers* layers, int groups, int n, const int* moved, int sms, cudaStream_t s) {
    for (int g = 0; g < groups; ++g) {
        const cudaError_t e = launch_early(g ? work_kernel<kCopyWork> : work_kernel<WORK>, sms * 8, kWorkThreads, 0, s, p,
                                           layers[g], g ? 0 : n, g ? (const int*)nullptr : moved);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_kv_fork(const PagesDev& p, const KvLayers* layers, int groups, int n, const int* parents,
                           const int* children, int sms, cudaStream_t s) {
    const cudaError_t e = launch_early(plan_kernel<true>, 1, kPlanThreads, 0, s, p, parents, children, n);
    return e != cudaSuccess ? e : work<kForkWork>(p, layers, groups, n, nullptr, sms, s);
}

cudaError_t launch_kv_resize(const PagesDev& p, const KvLayers* layers, int groups, int n, const int* slots,
                             const int* lens, int sms, cudaStream_t s) {
    const cudaError_t e = launch_early(plan_kernel<false>, 1, kPlanThreads, 0, s, p, slots, lens, n);
    return e != cudaSuccess ? e : work<kResizeWork>(p, layers, groups, n, nullptr, sms, s);
}

cudaError_t launch_kv_compact(const PagesDev& args, const KvLayers* layers, int groups, int* moved, int sms,
                              cudaStream_t s) {
    PagesDev p = args;
    if (!moved) moved = p.rows;  // whole pages are copied: their numbers of rows are not needed
    p.rows = nullptr;
    const cudaError_t e = launch_early(plan_compact_kernel, 1, kPlanThreads, 0, s, p, moved);
    return e != cudaSuccess ? e : work<kCompactWork>(p, layers, groups, p.n_slots, moved, sms, s);
}

}  // namespace hc
