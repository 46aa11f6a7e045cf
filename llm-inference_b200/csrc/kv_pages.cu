// Page operations of a paged KV cache for sm_100a: copying pages, and the
// bookkeeping that gives sequences their pages (truncate, fork, extend,
// compact), all on device memory, so that a scheduler's step is captured with
// the model's.
//
// State: a page table [rows][stride], the rows' lengths in tokens, and a
// reference count a page (0: free). A sequence of n tokens holds
// ceil(n / page_size) pages; forked sequences share pages. The pages given
// out are the free ones with the lowest numbers, in the order of the items,
// so a call's result depends on its inputs alone.
//
// truncate and fork are one launch each. Every CTA checks all items and does
// its share of the table entries and counts, which no check reads; the CTA that
// finishes last, when nobody reads the old lengths any more, writes the new
// ones.
//
// extend is one launch as well. The first CTA plans and writes the whole
// bookkeeping; the others wait for its word (bounded) and copy the shared last
// pages with it. Its word comes as soon as it is known that none is copied. A
// CTA whose wait runs out (other kernels kept the first CTA from an SM) leaves
// its share to the CTA that finishes last, which then copies all pages again.
//
// The contents move with 16-byte loads and streaming stores, four in flight a
// thread: HBM-bound, a page's bytes read once and written once. (Plain stores:
// 95 us against 90 for 480 pages of 72 planes of 32 KB brought together; 8 CTAs
// an SM that loop against 32 that mostly do not: 95.7 against 90; a ring of bulk
// copies through shared memory: 103.) 90 us is 6.05 TB/s; 24 pages of 72 planes
// of 16 KB are copied in 11.2 us. Bound by dependent launches: 64 sequences
// rolled back and extended 9.2 us; 4 prompts dropped, forked into 8 beams and
// extended 33.6 us, 13.5 of them the copies. Bound by one CTA that walks the
// counts: with 700 / 20,000 / 100,000 / 2,000,000 pages, 95% of them taken from
// the low end, an extend of 64 sequences 4 / 10 / 29 / 455 us, a compact with
// nothing to move 8.5 / 23 / 87 / 1,561.
#include <algorithm>

#include "paged.cuh"

namespace b2 {
namespace {

constexpr uint32_t kItems = 1024;          // items of a call, one a thread
constexpr uint32_t kPlanThreads = 1024;
constexpr uint32_t kCopyThreads = 256;
constexpr uint32_t kCopyUnroll = 4;
constexpr uint32_t kMaxPairs = 4096;       // pairs of a copy: each CTA looks through all of them
constexpr uint32_t kHash = 2 * kItems;     // open addressing, at most half full
constexpr size_t kMaxPages = 1u << 21;     // kItems * kMaxPages pages asked for at once fit 32 bits
constexpr int32_t kNone = -1;

struct Pool {
    uint4* base;
    uint64_t plane_stride, page_stride;  // 16-byte pieces
    uint32_t planes, num_pages;
    FastDiv vecs;  // 16-byte pieces of a page in one plane
};

struct Seqs {
    int32_t* table;
    uint64_t table_stride;
    int32_t* len;
    int32_t* ref;
    uint32_t rows, num_pages;
    uint32_t capacity;  // tokens a row can hold
    FastDiv page_size;
    __device__ __forceinline__ uint32_t pages(uint32_t tokens) const {
        uint32_t r;
        const uint32_t q = page_size.div(tokens, r);
        return q + (r != 0);
    }
};

__device__ __forceinline__ uint4 ld16(const uint4* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p)
                 : "memory");
    return r;
}

// Pieces [first, first + threads * kCopyUnroll) of page src's planes to page
// dst: the pieces of all planes are numbered through.
__device__ __forceinline__ void copy_piece(const Pool& p, uint32_t src, uint32_t dst, uint32_t first, uint32_t threads) {
    const uint32_t total = p.planes * p.vecs.d;
    uint4 w[kCopyUnroll];
    uint64_t at[kCopyUnroll];
#pragma unroll
    for (uint32_t u = 0; u < kCopyUnroll; ++u) {
        const uint32_t i = first + u * threads + threadIdx.x;
        uint32_t v;
        const uint32_t plane = p.vecs.div(i, v);
        at[u] = plane * p.plane_stride + v;
        if (i < total) w[u] = ld16(p.base + at[u] + src * p.page_stride);
    }
#pragma unroll
    for (uint32_t u = 0; u < kCopyUnroll; ++u)
        if (first + u * threads + threadIdx.x < total) __stcs(p.base + at[u] + dst * p.page_stride, w[u]);
}

__device__ __forceinline__ uint32_t pieces_of(const Pool& p, uint32_t threads) {
    return (p.planes * p.vecs.d + threads * kCopyUnroll - 1) / (threads * kCopyUnroll);
}

// What the workspace begins with, zero before its first use.
struct Header {
    uint32_t finished;  // CTAs of this launch that are done (kGaveUp apiece: and had copied nothing)
    uint32_t word;      // extend: 0, or 1 + the pages to copy
    uint32_t moves;     // pages that this compact moves
    uint32_t unused;
    int32_t lists[];    // [kItems] sources and [kItems] copies of extend, then compact's
};

// ---- copy ---------------------------------------------------------------------

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const Pool p, const int32_t* src, const int32_t* dst,
                                                                  uint32_t n) {
    pdl_wait_primary();
    pdl_launch_dependents();
    const uint32_t pieces = pieces_of(p, kCopyThreads);
    const uint64_t total = static_cast<uint64_t>(n) * pieces;
    uint32_t cur = 0xffffffffu;
    bool go = false;
    int32_t s = 0, d = 0;
    // consecutive pieces to a CTA, so that a pair is looked at once or twice
    const uint64_t per = (total + gridDim.x - 1) / gridDim.x;
    const uint64_t end = min(total, (blockIdx.x + 1) * per);
    for (uint64_t w = blockIdx.x * per; w < end; ++w) {
        const uint32_t i = static_cast<uint32_t>(w / pieces);
        if (i != cur) {
            cur = i;
            s = src[i];
            d = dst[i];
            const bool bad = s < 0 || d < 0 || static_cast<uint32_t>(s) >= p.num_pages ||
                             static_cast<uint32_t>(d) >= p.num_pages;
            bool clash = false, later = false;
            for (uint32_t j = threadIdx.x; j < n; j += kCopyThreads) {
                const int32_t sj = src[j], dj = dst[j];
                clash |= j != i && sj == d && sj != dj;
                later |= j > i && dj == d && sj != dj && sj >= 0 && static_cast<uint32_t>(sj) < p.num_pages;
            }
            // both are barriers: every thread takes them
            clash = __syncthreads_or(clash) != 0;
            later = __syncthreads_or(later) != 0;
            if (threadIdx.x == 0 && (bad || (clash && s != d))) atomicOr(&g_device_error, kErrBadPage);
            go = !bad && !clash && !later && s != d;
        }
        if (go)
            copy_piece(p, static_cast<uint32_t>(s), static_cast<uint32_t>(d),
                       static_cast<uint32_t>(w - static_cast<uint64_t>(i) * pieces) * kCopyThreads * kCopyUnroll,
                       kCopyThreads);
    }
}

// ---- what the plans are made with ------------------------------------------------

struct Scan {
    uint32_t warp[kPlanThreads / 32];
};

// Exclusive prefix sum over the block; total of all threads in `total`.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, Scan& sm, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
    }
    if (lane == 31) sm.warp[warp] = x;
    __syncthreads();
    if (warp == 0) {
        uint32_t w = sm.warp[lane];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, w, off);
            if (lane >= off) w += y;
        }
        sm.warp[lane] = w;
    }
    __syncthreads();
    const uint32_t before = warp ? sm.warp[warp - 1] : 0u;
    total = sm.warp[kPlanThreads / 32 - 1];
    __syncthreads();  // sm is used again
    return before + x - v;
}

struct Hash {
    int32_t key[kHash];
    uint32_t count[kHash];
    uint32_t first[kHash];  // lowest item with this key
};

__device__ __forceinline__ void hash_clear(Hash& h) {
    for (uint32_t i = threadIdx.x; i < kHash; i += kPlanThreads) {
        h.key[i] = kNone;
        h.count[i] = 0;
        h.first[i] = 0xffffffffu;
    }
    __syncthreads();
}

// The slot of key (>= 0), entered if it is new. At most kItems keys are
// entered into 2 * kItems slots, so a free one is always met.
__device__ __forceinline__ uint32_t hash_slot(Hash& h, int32_t key) {
    uint32_t s = (static_cast<uint32_t>(key) * 2654435761u) >> 21;  // 11 bits: kHash slots
    for (uint32_t i = 0; i < kHash; ++i) {
        const int32_t old = atomicCAS(&h.key[s], kNone, key);
        if (old == kNone || old == key) break;
        s = (s + 1) & (kHash - 1);
    }
    return s;
}
static_assert(kHash == 1u << 11, "hash_slot gives 11 bits");

constexpr uint32_t kGaveUp = 1u << 16;  // beside the count of CTAs

// In the CTA that comes last 1 + how many CTAs gave `mark` as kGaveUp, 0 in
// the others; the counter is then 0 again.
__device__ __forceinline__ uint32_t last_cta(uint32_t* counter, uint32_t* flag, uint32_t mark = 0u) {
    __syncthreads();
    if (gridDim.x == 1) return 1u;
    if (threadIdx.x == 0) {
        __threadfence();
        const uint32_t now = atomicAdd(counter, 1u + mark) + 1u + mark;
        const bool last = (now & (kGaveUp - 1)) == gridDim.x;
        *flag = last ? 1u + now / kGaveUp : 0u;
        if (last) *counter = 0u;
        __threadfence();
    }
    __syncthreads();
    return *flag;
}

// Which of this thread's four pages from page `base` on are free.
__device__ __forceinline__ uint32_t free_mask(const Seqs& q, uint32_t base) {
    const uint32_t p0 = base + 4 * threadIdx.x;
    uint32_t mask = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        if (p0 + i < q.num_pages && q.ref[p0 + i] == 0) mask |= 1u << i;
    return mask;
}

// Calls f(rank, page) for the free pages of rank < want, ranks by page number;
// returns how many there are (at most want). mask0: free_mask(q, 0), looked up
// ahead, so that small pools are not read again.
template <typename F>
__device__ __forceinline__ uint32_t free_pages(const Seqs& q, uint32_t mask0, uint32_t want, Scan& sm, F f) {
    uint32_t found = 0;
    for (uint32_t base = 0; base < q.num_pages && found < want; base += 4 * kPlanThreads) {
        const uint32_t mask = base == 0 ? mask0 : free_mask(q, base);
        uint32_t total;
        uint32_t r = found + block_scan(__popc(mask), sm, total);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (mask & (1u << i)) {
                if (r < want) f(r, base + 4 * threadIdx.x + i);
                ++r;
            }
        }
        found += total;
    }
    return min(found, want);
}

// One reference of `page` given back; a bad number or a page without
// references sets the error bit and changes nothing.
__device__ __forceinline__ void drop_ref(const Seqs& q, int32_t page) {
    if (page >= 0 && static_cast<uint32_t>(page) < q.num_pages) {
        if (atomicSub(&q.ref[page], 1) > 0) return;
        atomicAdd(&q.ref[page], 1);
    }
    atomicOr(&g_device_error, kErrBadPage);
}

struct Shared {
    Hash hash;
    Scan scan;
    int32_t row[kItems];
    uint32_t from[kItems];
    uint32_t base[kItems + 1];  // entries (pages) of the items before
    uint32_t flag;
};

// Item that has number r of what base counts: base[lo] <= r < base[lo + 1].
__device__ __forceinline__ uint32_t item_of(const uint32_t* base, uint32_t n, uint32_t r) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (base[mid] <= r) lo = mid;
        else hi = mid;
    }
    return lo;
}

// ---- truncate -------------------------------------------------------------------

__global__ void __launch_bounds__(kPlanThreads) truncate_kernel(const Seqs q, const int32_t* seqs, const int32_t* new_len,
                                                                uint32_t n, int32_t* status, Header* head) {
    __shared__ Shared sm;
    pdl_wait_primary();
    pdl_launch_dependents();
    const uint32_t i = threadIdx.x;
    int32_t s = kNone, want = 0;
    if (i < n) {
        s = seqs[i];
        want = new_len ? new_len[i] : 0;
    }
    hash_clear(sm.hash);
    uint32_t keep = 0, held = 0;
    bool bad = false;
    if (s >= 0) {
        bad = static_cast<uint32_t>(s) >= q.rows;
        if (!bad) {
            const int32_t old = q.len[s];
            bad = old < 0 || static_cast<uint32_t>(old) > q.capacity || want < 0 || want > old;
            if (!bad) {
                keep = q.pages(want);
                held = q.pages(old);
            }
            bad |= atomicAdd(&sm.hash.count[hash_slot(sm.hash, s)], 1u) != 0;  // twice in one call
        }
    }
    bad = __syncthreads_or(bad) != 0;
    if (!bad) {
        uint32_t total;
        const uint32_t base = block_scan(held - keep, sm.scan, total);
        if (i < n) {
            sm.row[i] = s;
            sm.from[i] = keep;
            sm.base[i] = base;
        }
        if (i == 0) sm.base[n] = total;
        __syncthreads();
        for (uint32_t e = blockIdx.x * kPlanThreads + i; e < total; e += gridDim.x * kPlanThreads) {
            const uint32_t c = item_of(sm.base, n, e);
            int32_t* t = q.table + static_cast<uint64_t>(sm.row[c]) * q.table_stride + sm.from[c] + (e - sm.base[c]);
            const int32_t page = *t;
            *t = kNone;
            drop_ref(q, page);
        }
    }
    if (!last_cta(&head->finished, &sm.flag)) return;
    if (!bad && s >= 0) q.len[s] = want;
    if (i == 0 && status) {
        status[0] = bad ? B2_PAGES_BAD_ITEM : B2_PAGES_OK;
        status[1] = 0;
    }
}

// ---- fork -----------------------------------------------------------------------

__global__ void __launch_bounds__(kPlanThreads) fork_kernel(const Seqs q, const int32_t* parents, const int32_t* children,
                                                            const int32_t* fork_len, uint32_t n, int32_t* status,
                                                            Header* head) {
    __shared__ Shared sm;
    pdl_wait_primary();
    pdl_launch_dependents();
    const uint32_t i = threadIdx.x;
    int32_t par = kNone, child = kNone, len = 0;
    if (i < n) {
        par = parents[i];
        child = children[i];
        len = fork_len ? fork_len[i] : 0;
    }
    hash_clear(sm.hash);
    bool bad = false;
    uint32_t share = 0;
    if (par < 0 || child < 0) {
        par = child = kNone;  // an idle item
    } else {
        bad = static_cast<uint32_t>(par) >= q.rows || static_cast<uint32_t>(child) >= q.rows || par == child;
        if (!bad) {
            const int32_t have = q.len[par], taken = q.len[child];
            if (!fork_len) len = have;
            bad = have < 0 || static_cast<uint32_t>(have) > q.capacity || len < 0 || len > have || taken != 0;
            bad |= atomicAdd(&sm.hash.count[hash_slot(sm.hash, child)], 1u) != 0;  // twice in one call
            if (!bad) share = q.pages(len);
        }
    }
    bad = __syncthreads_or(bad) != 0;
    if (!bad) {
        uint32_t total;
        const uint32_t base = block_scan(share, sm.scan, total);
        if (i < n) {
            sm.row[i] = child;
            sm.from[i] = static_cast<uint32_t>(par);
            sm.base[i] = base;
        }
        if (i == 0) sm.base[n] = total;
        __syncthreads();
        for (uint32_t e = blockIdx.x * kPlanThreads + i; e < total; e += gridDim.x * kPlanThreads) {
            const uint32_t c = item_of(sm.base, n, e), j = e - sm.base[c];
            const int32_t page = q.table[static_cast<uint64_t>(sm.from[c]) * q.table_stride + j];
            q.table[static_cast<uint64_t>(sm.row[c]) * q.table_stride + j] = page;
            if (page >= 0 && static_cast<uint32_t>(page) < q.num_pages)
                atomicAdd(&q.ref[page], 1);
            else
                atomicOr(&g_device_error, kErrBadPage);
        }
    }
    if (!last_cta(&head->finished, &sm.flag)) return;
    if (!bad && child >= 0) q.len[child] = len;
    if (i == 0 && status) {
        status[0] = bad ? B2_PAGES_BAD_ITEM : B2_PAGES_OK;
        status[1] = 0;
    }
}

// ---- extend ----------------------------------------------------------------------

constexpr uint32_t kFound = sizeof(Hash) / sizeof(int32_t);  // free pages kept by number, where the hash was

struct ExtendShared {
    Shared s;
    int32_t last[kItems];  // a shared last page that is copied, or -1
    uint32_t to[kItems];   // its copy
};

// The first CTA's word to the others: the pages to copy, listed before.
__device__ __forceinline__ void tell(Header* head, uint32_t copies) {
    asm volatile("st.release.gpu.u32 [%0], %1;" ::"l"(&head->word), "r"(copies + 1) : "memory");
}

__device__ __forceinline__ uint32_t told(const Header* head) {
    uint32_t word;
    asm volatile("ld.acquire.gpu.u32 %0, [%1];" : "=r"(word) : "l"(&head->word) : "memory");
    return word;
}

// Every `step`th piece of the listed copies, from piece `begin` on.
__device__ __forceinline__ void copy_listed(const Pool& p, const Header* head, uint32_t copies, uint32_t n,
                                            uint32_t begin, uint32_t step) {
    if (copies > n) copies = 0;  // a workspace that was not zero at first: nothing is followed
    const uint32_t pieces = pieces_of(p, kPlanThreads);
    for (uint64_t w = begin; w < static_cast<uint64_t>(copies) * pieces; w += step) {
        const uint32_t c = static_cast<uint32_t>(w / pieces);
        const uint32_t src = static_cast<uint32_t>(__ldcg(head->lists + c));
        const uint32_t dst = static_cast<uint32_t>(__ldcg(head->lists + kItems + c));
        if (src < p.num_pages && dst < p.num_pages)
            copy_piece(p, src, dst, static_cast<uint32_t>(w - static_cast<uint64_t>(c) * pieces) * kPlanThreads * kCopyUnroll,
                       kPlanThreads);
    }
}

// The whole bookkeeping of an extend, by one CTA. Returns the pages to copy, listed in head.
__device__ uint32_t extend_plan(ExtendShared& sm, const Seqs& q, const int32_t* seqs, const int32_t* new_tokens,
                                uint32_t n, int32_t* first, int32_t* status, Header* head) {
    const uint32_t i = threadIdx.x;
    int32_t s = kNone, old = 0, take = 0, last = kNone;
    if (i < n) {
        s = seqs[i];
        take = new_tokens[i];
    }
    const uint32_t mask0 = free_mask(q, 0);
    hash_clear(sm.s.hash);
    uint32_t held = 0, want = 0;
    int32_t refs = 0;
    bool bad = false;
    if (s >= 0) {
        bad = static_cast<uint32_t>(s) >= q.rows;
        if (!bad) {
            old = q.len[s];
            bad = old < 0 || take < 0 || static_cast<int64_t>(old) + take > static_cast<int64_t>(q.capacity);
            bad |= atomicAdd(&sm.s.hash.count[hash_slot(sm.s.hash, s)], 1u) != 0;  // twice in one call
        }
        if (!bad) {
            held = q.pages(old);
            want = q.pages(old + take);
            uint32_t part;
            (void)q.page_size.div(old, part);
            if (part != 0 && take > 0) {
                last = q.table[static_cast<uint64_t>(s) * q.table_stride + held - 1];
                bad = last < 0 || static_cast<uint32_t>(last) >= q.num_pages;
                if (!bad) refs = q.ref[last];
                bad |= refs <= 0;   // counted as free: it would be given out again
            }
        }
    }
    bad = __syncthreads_or(bad) != 0;
    // A last page that others hold too is copied, unless all its holders are
    // extended by this call, of whom the first item keeps it.
    bool cow = !bad && refs > 1;
    const bool any_cow = __syncthreads_or(cow) != 0;
    if (any_cow) {
        hash_clear(sm.s.hash);
        uint32_t slot = 0;
        if (last >= 0) {
            slot = hash_slot(sm.s.hash, last);
            atomicAdd(&sm.s.hash.count[slot], 1u);
            atomicMin(&sm.s.hash.first[slot], i);
        }
        __syncthreads();
        if (cow && sm.s.hash.count[slot] == static_cast<uint32_t>(refs) && sm.s.hash.first[slot] == i) cow = false;
    } else if (i == 0) {
        tell(head, 0);  // nothing for the others to do
    }
    // an item takes table_stride <= kMaxPages pages at most (a copied one held one before), so the sum fits 32 bits
    const uint32_t need = bad ? 0u : want - held + (cow ? 1u : 0u);
    uint32_t total, copies = 0, place = 0;
    const uint32_t base = block_scan(need, sm.s.scan, total);
    if (any_cow) place = block_scan(cow ? 1u : 0u, sm.s.scan, copies);
    if (i < n) {
        sm.s.base[i] = base;
        sm.last[i] = cow ? last : kNone;
        sm.s.row[i] = s;
        sm.s.from[i] = held;
    }
    if (i == 0) sm.s.base[n] = total;
    __syncthreads();
    // the free pages, by rank; the first kFound are kept, so that few are looked up twice
    uint32_t* found = reinterpret_cast<uint32_t*>(&sm.s.hash);
    auto keep = [&](uint32_t r, uint32_t page) {
        if (r < kFound) found[r] = page;
    };
    const bool room = !bad && total <= q.num_pages && free_pages(q, mask0, total, sm.s.scan, keep) == total;
    __syncthreads();
    if (room) {
        auto give = [&](uint32_t r, uint32_t page) {
            const uint32_t it = item_of(sm.s.base, n, r);
            const uint32_t k = r - sm.s.base[it], copied = sm.last[it] >= 0 ? 1u : 0u;
            // a copy takes the place of the last page, the others follow it
            const uint64_t j = static_cast<uint64_t>(sm.s.from[it]) + k - copied;
            q.table[static_cast<uint64_t>(sm.s.row[it]) * q.table_stride + j] = static_cast<int32_t>(page);
            q.ref[page] = 1;
            if (copied && k == 0) sm.to[it] = page;
        };
        if (total <= kFound) {
            for (uint32_t r = i; r < total; r += kPlanThreads) give(r, found[r]);
        } else {
            free_pages(q, mask0, total, sm.s.scan, give);
        }
        if (cow) atomicSub(&q.ref[last], 1);
        if (s >= 0) q.len[s] = old + take;
        if (any_cow) {
            __syncthreads();
            if (cow) {
                head->lists[place] = last;
                head->lists[kItems + place] = static_cast<int32_t>(sm.to[i]);
            }
        }
    }
    if (i < n && first) first[i] = room && s >= 0 ? old : kNone;
    if (i == 0 && status) {
        status[0] = bad ? B2_PAGES_BAD_ITEM : room ? B2_PAGES_OK : B2_PAGES_SHORT;
        status[1] = static_cast<int32_t>(min(total, 0x7fffffffu));
    }
    copies = room ? copies : 0u;
    __syncthreads();
    if (any_cow && i == 0) tell(head, copies);
    return copies;
}

__global__ void __launch_bounds__(kPlanThreads) extend_kernel(const Pool p, const Seqs q, const int32_t* seqs,
                                                              const int32_t* new_tokens, uint32_t n, int32_t* first,
                                                              int32_t* status, Header* head) {
    __shared__ ExtendShared sm;
    pdl_wait_primary();
    pdl_launch_dependents();
    uint32_t copies, gave_up = 0;
    if (blockIdx.x == 0) {
        copies = extend_plan(sm, q, seqs, new_tokens, n, first, status, head);
    } else {
        if (threadIdx.x == 0) {
            const uint64_t deadline = global_timer_ns() + kWaitBudgetNs;
            uint32_t word;
            do {
                word = told(head);
            } while (word == 0 && global_timer_ns() < deadline);
            sm.s.flag = word;
        }
        __syncthreads();
        copies = sm.s.flag ? sm.s.flag - 1 : 0u;
        gave_up = sm.s.flag ? 0u : kGaveUp;
    }
    copy_listed(p, head, copies, n, blockIdx.x, gridDim.x);
    // the last to have read the word takes it back for the next call
    const uint32_t last = last_cta(&head->finished, &sm.s.flag, gave_up);
    if (last == 0) return;
    if (last > 1) {
        __syncthreads();  // flag is read
        if (threadIdx.x == 0) sm.s.flag = told(head) - 1;
        __syncthreads();
        copy_listed(p, head, sm.s.flag, n, 0, 1);
    }
    if (threadIdx.x == 0) head->word = 0u;
}

// ---- compact ---------------------------------------------------------------------

struct Moves {
    uint32_t* count;
    int32_t* src;
    int32_t* dst;
    int32_t* refs;
    int32_t* map;  // [num_pages] where each page goes
};

// The moves: live pages numbered at or past the number of live pages, in
// order, to the free ones below it. ref_out may be ref.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const int32_t* ref, int32_t* ref_out, uint32_t pages,
                                                                    const Moves mv, int32_t* status) {
    __shared__ Scan sm;
    pdl_wait_primary();
    pdl_launch_dependents();
    uint32_t live = 0;
    for (uint32_t p = threadIdx.x; p < pages; p += kPlanThreads) live += ref[p] > 0;
    uint32_t total;
    block_scan(live, sm, total);
    live = total;
    uint32_t before = 0;  // sources in the high half word, destinations in the low one
    uint32_t n_src = 0, n_dst = 0;
    for (uint32_t base = 0; base < pages; base += kPlanThreads) {
        const uint32_t p = base + threadIdx.x;
        const int32_t r = p < pages ? ref[p] : 0;
        const bool is_src = p < pages && r > 0 && p >= live, is_dst = p < pages && r <= 0 && p < live;
        before = block_scan((is_src ? 0x10000u : 0u) + (is_dst ? 1u : 0u), sm, total);
        if (is_src) {
            const uint32_t k = n_src + (before >> 16);
            mv.src[k] = static_cast<int32_t>(p);
            mv.refs[k] = r;
        }
        if (is_dst) mv.dst[n_dst + (before & 0xffffu)] = static_cast<int32_t>(p);
        if (p < pages) {
            mv.map[p] = static_cast<int32_t>(p);
            ref_out[p] = p < live ? max(r, 0) : 0;
        }
        n_src += total >> 16;
        n_dst += total & 0xffffu;
    }
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < n_src; k += kPlanThreads) {
        const int32_t s = mv.src[k], d = mv.dst[k];
        mv.map[s] = d;
        ref_out[d] = mv.refs[k];
    }
    if (threadIdx.x == 0) {
        *mv.count = n_src;
        if (status) {
            status[0] = B2_PAGES_OK;
            status[1] = static_cast<int32_t>(live);
        }
    }
}

__global__ void __launch_bounds__(kCopyThreads) compact_apply_kernel(const Pool p, const Seqs q, int32_t* table_out,
                                                                     const Moves mv) {
    pdl_wait_primary();
    pdl_launch_dependents();
    const uint64_t entries = static_cast<uint64_t>(q.rows) * q.table_stride;
    for (uint64_t e = blockIdx.x * static_cast<uint64_t>(kCopyThreads) + threadIdx.x; e < entries;
         e += static_cast<uint64_t>(gridDim.x) * kCopyThreads) {
        const uint32_t row = static_cast<uint32_t>(e / q.table_stride);
        const uint32_t j = static_cast<uint32_t>(e - row * q.table_stride);
        const int32_t len = q.len[row];
        int32_t page = q.table[e];
        if (len > 0 && j < q.pages(static_cast<uint32_t>(len))) {
            if (page >= 0 && static_cast<uint32_t>(page) < q.num_pages)
                page = mv.map[page];
            else
                atomicOr(&g_device_error, kErrBadPage);
        }
        table_out[e] = page;
    }
    const uint32_t pieces = pieces_of(p, kCopyThreads);
    const uint64_t total = static_cast<uint64_t>(*mv.count) * pieces;
    for (uint64_t w = blockIdx.x; w < total; w += gridDim.x) {
        const uint32_t k = static_cast<uint32_t>(w / pieces);
        copy_piece(p, static_cast<uint32_t>(mv.src[k]), static_cast<uint32_t>(mv.dst[k]),
                   static_cast<uint32_t>(w - static_cast<uint64_t>(k) * pieces) * kCopyThreads * kCopyUnroll, kCopyThreads);
    }
}

// ---- host side -------------------------------------------------------------------

int pages_sms() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    return n;
}

int make_pool(Pool* out, void* pool, size_t planes, size_t plane_stride, size_t num_pages, size_t page_stride,
              size_t page_elems) {
    if (!pool || planes == 0 || num_pages == 0 || page_elems == 0) return B2_ERR_INVALID_ARG;
    if (num_pages > kMaxPages || planes > 0xffffu || page_elems / 8 * planes > 0x3fffffffull) return B2_ERR_UNSUPPORTED;
    if (page_stride == 0) page_stride = page_elems;
    if (plane_stride == 0) plane_stride = num_pages * page_stride;
    if (num_pages > 1 && page_stride < page_elems) return B2_ERR_INVALID_ARG;
    // a plane's pages together, or a page's planes together: no two overlap
    const bool by_plane = plane_stride >= (num_pages - 1) * page_stride + page_elems;
    const bool by_page = plane_stride >= page_elems && page_stride >= (planes - 1) * plane_stride + page_elems;
    if (planes > 1 && !by_plane && !by_page) return B2_ERR_INVALID_ARG;
    if (!aligned16(pool) || page_elems % 8 != 0 || page_stride % 8 != 0 || plane_stride % 8 != 0) return B2_ERR_ALIGNMENT;
    out->base = static_cast<uint4*>(pool);
    out->plane_stride = plane_stride / 8;
    out->page_stride = page_stride / 8;
    out->planes = static_cast<uint32_t>(planes);
    out->num_pages = static_cast<uint32_t>(num_pages);
    out->vecs = FastDiv::of(static_cast<uint32_t>(page_elems / 8));
    return B2_OK;
}

int make_seqs(Seqs* out, int32_t* table, size_t table_stride, size_t rows, size_t page_size, size_t num_pages,
              int32_t* len, int32_t* ref) {
    if (!table || !len || !ref || table_stride == 0 || rows == 0 || page_size == 0 || num_pages == 0)
        return B2_ERR_INVALID_ARG;
    // (kItems rows of kMaxPages entries at most: their sums fit 32 bits too)
    if (table_stride > kMaxPages || rows > 0x7fffffffull || page_size > 0x7fffffffull || num_pages > kMaxPages)
        return B2_ERR_UNSUPPORTED;
    const uint64_t cap = static_cast<uint64_t>(table_stride) * page_size;
    out->table = table;
    out->table_stride = table_stride;
    out->len = len;
    out->ref = ref;
    out->rows = static_cast<uint32_t>(rows);
    out->num_pages = static_cast<uint32_t>(num_pages);
    out->capacity = static_cast<uint32_t>(cap > 0x7fffffffull ? 0x7fffffffull : cap);
    out->page_size = FastDiv::of(static_cast<uint32_t>(page_size));
    return B2_OK;
}

// CTAs of truncate and fork: one for up to eight entries a thread (by the
// rows' length; the counter of several costs about a microsecond), else more.
uint32_t items_grid(size_t items, size_t table_stride) {
    const uint64_t entries = static_cast<uint64_t>(items) * table_stride;
    if (entries <= 8 * kPlanThreads) return 1;
    return static_cast<uint32_t>(std::min<uint64_t>((entries + kPlanThreads - 1) / kPlanThreads, pages_sms()));
}

// Workspace: the header, extend's copies, then compact's moves.
size_t moves_words(size_t num_pages) { return 3 * (num_pages / 2 + 1) + num_pages; }

size_t pages_ws_bytes(size_t num_pages) {
    return (sizeof(Header) + (2 * kItems + moves_words(num_pages)) * 4 + 255) / 256 * 256;
}

int check_ws(const void* ws, size_t bytes, size_t num_pages) {
    if (!ws) return B2_ERR_INVALID_ARG;
    if (reinterpret_cast<uintptr_t>(ws) % 4 != 0) return B2_ERR_ALIGNMENT;
    return bytes < pages_ws_bytes(num_pages) ? B2_ERR_WORKSPACE : B2_OK;
}

}  // namespace

unsigned int device_error_pages() {
    unsigned int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(v)) != cudaSuccess) return 0;
    return v;
}

int clear_device_error_pages() {
    const unsigned int zero = 0;
    return cuda_status(cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero)));
}

}  // namespace b2

using namespace b2;

extern "C" size_t b2_kv_pages_workspace_bytes(size_t num_pages) {
    if (num_pages == 0 || num_pages > kMaxPages) return 0;
    return pages_ws_bytes(num_pages);
}

extern "C" int b2_launch_kv_pages_copy(void* d_pool, size_t num_planes, size_t plane_stride, size_t num_pages,
                                       size_t page_stride, size_t page_elems, const int32_t* d_src_pages,
                                       const int32_t* d_dst_pages, size_t num_pairs, b2_stream_t stream) {
    if (num_pairs == 0) return B2_NOTHING_TO_DO;
    if (!d_src_pages || !d_dst_pages) return B2_ERR_INVALID_ARG;
    if (num_pairs > kMaxPairs) return B2_ERR_UNSUPPORTED;
    Pool p{};
    const int st = make_pool(&p, d_pool, num_planes, plane_stride, num_pages, page_stride, page_elems);
    if (st != B2_OK) return st;
    const uint64_t pieces = (static_cast<uint64_t>(p.planes) * p.vecs.d + kCopyThreads * kCopyUnroll - 1) /
                            (kCopyThreads * kCopyUnroll);
    const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>(num_pairs * pieces, 32ull * pages_sms()));
    return launch_pdl(copy_pages_kernel, dim3(grid), dim3(kCopyThreads), 0, reinterpret_cast<cudaStream_t>(stream), p,
                      d_src_pages, d_dst_pages, static_cast<uint32_t>(num_pairs));
}

extern "C" int b2_launch_kv_pages_truncate(int32_t* d_page_table, size_t table_stride, size_t table_rows,
                                           size_t page_size, size_t num_pages, int32_t* d_seq_len,
                                           int32_t* d_ref_count, const int32_t* d_seqs, const int32_t* d_new_len,
                                           size_t num_items, int32_t* d_status, void* d_workspace,
                                           size_t workspace_bytes, b2_stream_t stream) {
    if (num_items == 0) return B2_NOTHING_TO_DO;
    if (!d_seqs) return B2_ERR_INVALID_ARG;
    if (num_items > kItems) return B2_ERR_UNSUPPORTED;
    Seqs q{};
    int st = make_seqs(&q, d_page_table, table_stride, table_rows, page_size, num_pages, d_seq_len, d_ref_count);
    if (st == B2_OK) st = check_ws(d_workspace, workspace_bytes, num_pages);
    if (st != B2_OK) return st;
    return launch_pdl(truncate_kernel, dim3(items_grid(num_items, table_stride)), dim3(kPlanThreads), 0, reinterpret_cast<cudaStream_t>(stream), q,
                      d_seqs, d_new_len, static_cast<uint32_t>(num_items), d_status,
                      static_cast<Header*>(d_workspace));
}

extern "C" int b2_launch_kv_pages_fork(int32_t* d_page_table, size_t table_stride, size_t table_rows, size_t page_size,
                                       size_t num_pages, int32_t* d_seq_len, int32_t* d_ref_count,
                                       const int32_t* d_parents, const int32_t* d_children, const int32_t* d_fork_len,
                                       size_t num_items, int32_t* d_status, void* d_workspace, size_t workspace_bytes,
                                       b2_stream_t stream) {
    if (num_items == 0) return B2_NOTHING_TO_DO;
    if (!d_parents || !d_children) return B2_ERR_INVALID_ARG;
    if (num_items > kItems) return B2_ERR_UNSUPPORTED;
    Seqs q{};
    int st = make_seqs(&q, d_page_table, table_stride, table_rows, page_size, num_pages, d_seq_len, d_ref_count);
    if (st == B2_OK) st = check_ws(d_workspace, workspace_bytes, num_pages);
    if (st != B2_OK) return st;
    return launch_pdl(fork_kernel, dim3(items_grid(num_items, table_stride)), dim3(kPlanThreads), 0, reinterpret_cast<cudaStream_t>(stream), q,
                      d_parents, d_children, d_fork_len, static_cast<uint32_t>(num_items), d_status,
                      static_cast<Header*>(d_workspace));
}

extern "C" int b2_launch_kv_pages_extend(void* d_pool, size_t num_planes, size_t plane_stride, size_t num_pages,
                                         size_t page_stride, size_t page_elems, int32_t* d_page_table,
                                         size_t table_stride, size_t table_rows, size_t page_size, int32_t* d_seq_len,
                                         int32_t* d_ref_count, const int32_t* d_seqs, const int32_t* d_new_tokens,
                                         size_t num_items, int32_t* d_pos, int32_t* d_status, void* d_workspace,
                                         size_t workspace_bytes, b2_stream_t stream) {
    if (num_items == 0) return B2_NOTHING_TO_DO;
    if (!d_seqs || !d_new_tokens) return B2_ERR_INVALID_ARG;
    if (num_items > kItems) return B2_ERR_UNSUPPORTED;
    Pool p{};
    Seqs q{};
    int st = make_pool(&p, d_pool, num_planes, plane_stride, num_pages, page_stride, page_elems);
    if (st == B2_OK)
        st = make_seqs(&q, d_page_table, table_stride, table_rows, page_size, num_pages, d_seq_len, d_ref_count);
    if (st == B2_OK) st = check_ws(d_workspace, workspace_bytes, num_pages);
    if (st != B2_OK) return st;
    return launch_pdl(extend_kernel, dim3(pages_sms()), dim3(kPlanThreads), 0, reinterpret_cast<cudaStream_t>(stream), p,
                      q, d_seqs, d_new_tokens, static_cast<uint32_t>(num_items), d_pos, d_status,
                      static_cast<Header*>(d_workspace));
}

extern "C" int b2_launch_kv_pages_compact(void* d_pool, size_t num_planes, size_t plane_stride, size_t num_pages,
                                          size_t page_stride, size_t page_elems, const int32_t* d_page_table,
                                          int32_t* d_page_table_out, size_t table_stride, size_t table_rows,
                                          size_t page_size, const int32_t* d_seq_len, const int32_t* d_ref_count,
                                          int32_t* d_ref_count_out, int32_t* d_status, void* d_workspace,
                                          size_t workspace_bytes, b2_stream_t stream_handle) {
    if (!d_page_table_out || !d_ref_count_out) return B2_ERR_INVALID_ARG;
    Pool p{};
    Seqs q{};
    int st = make_pool(&p, d_pool, num_planes, plane_stride, num_pages, page_stride, page_elems);
    if (st == B2_OK)
        st = make_seqs(&q, const_cast<int32_t*>(d_page_table), table_stride, table_rows, page_size, num_pages,
                       const_cast<int32_t*>(d_seq_len), const_cast<int32_t*>(d_ref_count));
    if (st == B2_OK) st = check_ws(d_workspace, workspace_bytes, num_pages);
    if (st != B2_OK) return st;
    Header* head = static_cast<Header*>(d_workspace);
    const size_t half = num_pages / 2 + 1;
    Moves mv{};
    mv.count = &head->moves;
    mv.src = head->lists + 2 * kItems;
    mv.dst = mv.src + half;
    mv.refs = mv.dst + half;
    mv.map = mv.refs + half;
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_handle);
    st = launch_pdl(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, static_cast<const int32_t*>(q.ref),
                    d_ref_count_out, q.num_pages, mv, d_status);
    if (st != B2_OK) return st;
    return launch_pdl(compact_apply_kernel, dim3(32 * pages_sms()), dim3(kCopyThreads), 0, stream, p, q,
                      d_page_table_out, mv);
}
