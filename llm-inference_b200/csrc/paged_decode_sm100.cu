// Decode attention over a paged KV cache for sm_100a, the tiled kernel
// (head_dim 128, 1 / 2 / 4 / 8 KV heads, up to 8 query heads a KV head): the
// decode of paged_decode.cu with K/V streamed by tensor copies and multiplied
// on the tensor cores.
//
// HBM-bound: 512 bytes a token and KV head, each read once for all query heads
// of its group.
//
// * A tile is 16 tokens of one page (the last of a page may hold fewer). The
//   batch's work is numbered through, a few units for beginning a sequence and
//   one a tile, and each CTA gets an even range of the numbers; its part of one
//   sequence is a segment. The cut depends on the lengths alone, so a call's
//   result does too. (Half of the work in ranges and the rest claimed in ever
//   smaller ones was slower at every size: 64 sequences of 512 to 16K tokens 123
//   us against 112, one of 64K 41 against 28, for the partials it makes.)
// * A producer warp (one CTA an SM) reads the page table 32 tiles ahead and
//   copies each tile's rows of all KV heads by a 4-D tensor map {64 fp16, row,
//   column block, page} (128-byte swizzle) into a ring of stages, and each
//   segment's Q row (with its rotation tables' rows) into one of two slots. In
//   the decode step it stores the new K/V row before the tile that holds it.
// * Eight consumer warps (KV head x eight / KV heads) take the tiles with the
//   MMA tile math of decode_tile.cuh, rotate Q in registers, and join their
//   states at a segment's end through shared memory, pair by pair. A segment
//   that is a whole sequence writes the output; others write one partial.
// * paged_join_kernel joins the partials of the sequences that were cut.
//
// Measured, a call in a graph: 64 sequences of 512 to 16K tokens, 16 heads over
// 4, 111.4 us (6.45 TB/s, the copy peak 6.55); one of 64K 27.7 us (4.8 TB/s: 3.5
// until the first tile, 5 for flush and join); 256 of one KV head 19.6; a step
// of 48 with 8 KV heads 78.2 (6.1 TB/s); one of 300 tokens 7.0.
//
// The weights go to the tensor cores as two 16-bit numbers each (kWide of
// tile_softmax_pv: off by 2^-22 of a weight, or by 2^-32 of the largest);
// scores, sums, maxima and O stay in 32 bits. Against one 16-bit number the
// eight more products a tile cost 0.1 to 0.3 us where latency counts (one of
// 300 tokens 7.15 us instead of 7.05, one of 64K 27.4 instead of 27.0, 256 of
// one KV head 19.6 instead of 19.3) and nothing where HBM does (64 ragged 111.5
// and 111.6).
#include <math.h>

#include <algorithm>
#include <atomic>

#include "decode_tile.cuh"
#include "paged_decode.h"
#include "slot_pair.h"
#include "tcgen05.cuh"

namespace b2 {
namespace {

constexpr int kPtConsumers = 8;
constexpr int kPtThreads = (kPtConsumers + 1) * 32;
constexpr uint32_t kPtMaxSeqs = 1024;   // 32 a lane of the producer warp; 32 * 32 for its search
constexpr uint32_t kPtMaxCtas = 160;
// Smaller pages leave most of a 16-token tile empty. 64 sequences of 1 to 4096 tokens, lengths spread over
// their logarithm, 4 query heads a KV head and 1 / 2 / 4 / 8 KV heads: pages of 2 tokens 34 / 50 / 81 / 138 us
// here and 28 / 31 / 55 / 101 with the split kernel, of 3 tokens 25 / 36 / 57 / 95 and 28 / 31 / 54 / 99, of 4
// tokens 21 / 29 / 44 / 74 and 28 / 31 / 54 / 97.
constexpr uint32_t kPtMinPage = 4;
constexpr uint32_t kPtSmemLimit = 226 * 1024;
constexpr uint32_t kPtMaxStages = 16;
constexpr uint32_t kNoSeg = 0xffffffffu;
// The maximum before any score: below every finite one (a product of 16-bit rows stays within 2^40)
// and finite itself, so that a score of -infinity (an infinity in K) weighs 0 from the first tile on.
constexpr float kNoMax = -1e30f;
// flags kept with a sequence's table row
constexpr uint32_t kRowBits = 0x0fffffffu, kRowRotate = 1u << 28, kRowAppend = 1u << 29, kRowCapped = 1u << 30;

__host__ __device__ constexpr uint32_t pt_npar(uint32_t kvh) { return kPtConsumers / kvh; }  // warps of a KV head
__host__ __device__ constexpr uint32_t pt_sub(uint32_t kvh) { return kvh < 4 ? 4 / kvh : 1; }  // tiles of a stage
__host__ __device__ constexpr uint32_t pt_spar(uint32_t kvh) { return pt_npar(kvh) / pt_sub(kvh); }
// What starting and ending a segment costs, in tiles: about two stages' time. 256 slots of 1 to 4099 tokens
// (lengths spread over their logarithm, a fifth idle) with 0 / 1 / 2 / 3 / 4 stages: 27.6 / 22.7 / 20.0 / 20.1
// / 21.1 us with one KV head, 32.6 / 30.0 / 26.5 / 25.2 / 26.1 with 2, 47.3 / 44.8 / 43.4 / 43.5 / 43.9 with 4,
// 81.2 / 80.5 / 80.4 / 81.5 / 81.7 with 8: the CTA with the most short sequences is last. 64 long ones do not
// notice it from 2 on.
__host__ __device__ constexpr uint32_t pt_begin(uint32_t kvh) { return 2 * pt_sub(kvh); }

// The cut of `total` units into a range for each CTA: the first `odd` CTAs get
// per + 1 units, the others per.
struct Cut {
    uint32_t per, odd;
    __device__ __forceinline__ static Cut of(uint32_t total, FastDiv ctas) {
        Cut c;
        c.per = ctas.div(total, c.odd);
        return c;
    }
    __device__ __forceinline__ uint32_t begin(uint32_t cta) const { return cta * per + min(cta, odd); }
    __device__ __forceinline__ uint32_t cta_of(uint32_t unit) const {
        const uint32_t head = odd * (per + 1);
        return unit < head ? unit / (per + 1) : odd + (unit - head) / per;
    }
};

struct TiledArgs {
    PagedArgs p;
    FastDiv tiles_per_page;
    FastDiv ctas;      // CTAs the cut is made for
    uint32_t stages;
    uint32_t off_q, off_comb, off_tab, off_bar, qslot_bytes;  // shared memory
    float* po;         // [P][H][128], unnormalised
    float* pm;         // [H][P], log2 units
    float* pl;
    uint32_t parts;    // P
    uint2* cuts;       // [B] first partial and number of segments of each sequence, for the join
};

__device__ __forceinline__ uint32_t tiles_of(const TiledArgs& a, uint32_t len) {
    uint32_t r;
    const uint32_t j = a.p.pv.page_size.div(len, r);
    return j * a.tiles_per_page.d + (r + kTile - 1) / kTile;
}

// ---- joining two warps' states through shared memory --------------------------
// A lane's state (32 values of o, then m and l of two heads) lies together,
// 144 bytes a lane: 16-byte accesses without bank conflicts on either side.
// Lanes of heads past the group are left out.
constexpr uint32_t kStateFloats = 36;

__device__ __forceinline__ void state_dump(const WarpState& st, float* at) {
    float4* w = reinterpret_cast<float4*>(at);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = make_float4(st.o[i][0], st.o[i][1], st.o[i][2], st.o[i][3]);
    w[8] = make_float4(st.m0, st.m1, st.l0, st.l1);
}

__device__ __forceinline__ void join_factors(float& ma, float mb, float& fa, float& fb) {
    const float m = fmaxf(ma, mb);
    fa = ex2(ma - m);
    fb = ex2(mb - m);
    ma = m;
}

__device__ __forceinline__ void state_join(WarpState& st, const float* at) {
    const float4* r = reinterpret_cast<const float4*>(at);
    const float4 ml = r[8];
    float fa0, fb0, fa1, fb1;
    join_factors(st.m0, ml.x, fa0, fb0);
    join_factors(st.m1, ml.y, fa1, fb1);
    st.l0 = st.l0 * fa0 + ml.z * fb0;
    st.l1 = st.l1 * fa1 + ml.w * fb1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float4 x = r[i];
        st.o[i][0] = st.o[i][0] * fa0 + x.x * fb0;
        st.o[i][1] = st.o[i][1] * fa1 + x.y * fb1;
        st.o[i][2] = st.o[i][2] * fa0 + x.z * fb0;
        st.o[i][3] = st.o[i][3] * fa1 + x.w * fb1;
        if (i == 3) asm volatile("" ::: "memory");  // four loads in flight, not eight (registers)
    }
}

// 128 registers a thread, 168 without the limit: more leave the SM fewer for the join's CTAs, which then do not
// stand ready. One sequence of 64K tokens with 1 / 2 / 4 / 8 KV heads: 12.4 / 15.7 / 24.8 / 48.2 us with 128,
// 13.8 / 17.1 / 27.4 / 48.0 with 168 (144: 12.3 / 15.7 / 27.4 / 48.2). The limit costs 256 slots of one KV head
// 19.3 us against 19.0 and nothing on 64 long sequences (110.6 and 110.6); with 8 KV heads it spills 10 to 20
// bytes, without a trace in the times.
template <uint32_t KVH, bool kStep>
__global__ void __maxnreg__(128)
    paged_tiled_kernel(const TiledArgs t, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v) {
    constexpr uint32_t npar = pt_npar(KVH), kSub = pt_sub(KVH), spar = pt_spar(KVH);
    constexpr uint32_t sub_bytes = KVH * 2 * kTile * 128;    // a tile's K (or V) rows of all heads
    constexpr uint32_t stage_bytes = 2 * kSub * sub_bytes;
    constexpr uint32_t kBegin = pt_begin(KVH);
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t st_valid[kPtMaxStages][kSub], st_last[kPtMaxStages];
    const PagedArgs& a = t.p;
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* ring = base;
    uint8_t* qslots = base + t.off_q;
    float* comb = reinterpret_cast<float*>(base + t.off_comb);
    const uint32_t B = a.num_seqs, stages = t.stages;
    uint32_t* prefix = reinterpret_cast<uint32_t*>(base + t.off_tab);  // [B + 1] units before each sequence
    uint32_t* lens = prefix + B + 1;
    uint32_t* rows = lens + B;
    uint64_t* full = reinterpret_cast<uint64_t*>(base + t.off_bar);
    uint64_t* empty = full + stages;
    uint64_t* qfull = empty + stages;
    uint64_t* qempty = qfull + 2;
    uint64_t* cfull = qempty + 2;   // [8] states dumped (a slot a warp)
    uint64_t* cempty = cfull + 8;   // [8] and joined
    uint64_t* tables = cempty + 8;  // the tables are written
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 256) {
        for (uint32_t s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], KVH * kSub);
        }
        for (uint32_t s = 0; s < 2; ++s) {
            mbar_init(&qfull[s], 1);
            mbar_init(&qempty[s], kPtConsumers);
        }
        for (uint32_t s = 0; s < 8; ++s) {
            mbar_init(&cfull[s], 1);
            mbar_init(&cempty[s], 1);
        }
        mbar_init(tables, 1);
        fence_mbarrier_init();
        tc::prefetch_tensormap(&map_k);
        tc::prefetch_tensormap(&map_v);
    }
    __syncthreads();
    pdl_wait_primary();  // lengths, tables, Q and the pages may come from the previous kernel
    pdl_launch_dependents();

    bool ok = true;
    if (warp == kPtConsumers) {
        // ---- producer
        // the sequences' lengths and the units before each, a run of sequences a lane
        const uint32_t run = (B + 31) / 32, b0 = min(lane * run, B), b1 = min(b0 + run, B);
        uint32_t units = 0;
        for (uint32_t bb = b0; bb < b1; bb += 8) {
            int32_t row8[8], len8[8];   // eight entries' loads in flight
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                const uint32_t b = min(bb + k, b1 - 1);
                row8[k] = paged_row(a.pv, b);
                len8[k] = a.kv_len[b];
            }
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                const uint32_t b = bb + k;
                if (b >= b1) break;
                const uint32_t len = paged_tokens(a, row8[k], len8[k]);
                uint32_t word = row8[k] < 0 ? 0u : static_cast<uint32_t>(row8[k]);
                if constexpr (kStep) {
                    const int32_t p = len8[k];
                    if (row8[k] >= 0 && p >= 0) {
                        const bool in_table = static_cast<uint32_t>(p) < a.rope_rows;
                        const bool in_row = static_cast<uint32_t>(p) < a.pv.capacity;
                        if (a.rotate && in_table) word |= kRowRotate;
                        if (a.rotate && !in_table && blockIdx.x == 0) atomicOr(&g_device_error, kErrBadPosition);
                        if (a.k_new != nullptr && in_row && (!a.rotate || in_table)) word |= kRowAppend;
                        if (!in_row) word |= kRowCapped;
                    }
                }
                const uint32_t tiles = tiles_of(t, len);
                lens[b] = len;
                rows[b] = word;
                prefix[b] = units;
                units += tiles ? tiles + kBegin : 0u;
            }
        }
        uint32_t before = units;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t n = __shfl_up_sync(0xffffffffu, before, off);
            if (lane >= off) before += n;
        }
        const uint32_t total = __shfl_sync(0xffffffffu, before, 31);
        before -= units;
        for (uint32_t b = b0; b < b1; ++b) prefix[b] += before;
        if (lane == 0) prefix[B] = total;
        __syncwarp();
        if (lane == 0) mbar_arrive(tables);
        const Cut cut = Cut::of(total, t.ctas);
        const uint64_t policy = l2_evict_first_policy();
        uint32_t i = 0;               // stages so far
        SlotPair q_rows;              // the segments' Q rows
        uint32_t s = 0, round = 0;    // i % stages, i / stages
        uint32_t at = cut.begin(blockIdx.x);
        const uint32_t end = cut.begin(blockIdx.x + 1);
        uint32_t seg_ahead = kNoSeg;  // sequence whose first pages are looked up ahead
        int32_t page_ahead = -1;
        if (at < end) {
            // prefix[b] <= at < prefix[b + 1]: 32 places of the table at a time
            uint32_t b = 0;
            for (uint32_t stride = B > 32 ? 32u : 1u;;) {
                const uint32_t q = b + lane * stride;
                const uint32_t ge = __ballot_sync(0xffffffffu, q < B && prefix[q] <= at);
                b += (31 - __clz(ge)) * stride;   // lane 0 always votes
                if (stride == 1) break;
                stride = 1;
            }
            while (at < end && ok) {
                while (prefix[b + 1] <= at) ++b;   // sequences without tokens
                const uint32_t u0 = prefix[b], u1 = prefix[b + 1], stop = min(end, u1);
                const uint32_t first = at > u0 + kBegin ? at - u0 - kBegin : 0u;
                const uint32_t nt = (stop > u0 + kBegin ? stop - u0 - kBegin : 0u) - first;
                at = stop;
                if (nt == 0) continue;
                const bool tail = stop == u1, whole = tail && first == 0;
                const uint32_t len = lens[b], word = rows[b];
                const int32_t* trow = a.pv.table + static_cast<uint64_t>(word & kRowBits) * a.pv.table_stride;
                // a lane looks up tile x0 + lane of the segment, 32 at a time: its page (of the
                // next 32 as well; of the next sequence's first, while this one is under way)
                auto look = [&](uint32_t x) {
                    return x < nt ? trow[t.tiles_per_page.div(first + x)] : -1;
                };
                int32_t page = seg_ahead == b ? page_ahead : look(lane), next = look(32 + lane);
                seg_ahead = kNoSeg;
                if (at < end) {
                    uint32_t bn = b + 1;
                    while (prefix[bn + 1] <= at) ++bn;
                    seg_ahead = bn;
                    // from its first tile on (entries past its pages are not used)
                    const uint32_t ahead = min(prefix[bn + 1] - prefix[bn] - kBegin, 32u);
                    if (static_cast<uint32_t>(lane) < ahead)
                        page_ahead = a.pv.table[static_cast<uint64_t>(rows[bn] & kRowBits) * a.pv.table_stride +
                                                t.tiles_per_page.div(lane)];
                }
                // ... its first row there and its tokens (none: no tile, or a bad page)
                uint32_t r0, valid;
                auto measure = [&](uint32_t x) {
                    const uint32_t pg = t.tiles_per_page.div(first + x, r0);
                    r0 *= kTile;
                    const uint32_t tok = pg * a.pv.page_size.d + r0;
                    valid = x < nt ? min(static_cast<uint32_t>(kTile), min(a.pv.page_size.d - r0, len - tok)) : 0u;
                    if (valid && (page < 0 || static_cast<uint32_t>(page) >= a.pv.num_pages)) {
                        atomicOr(&g_device_error, kErrBadPage);
                        valid = 0;
                    }
                };
                measure(lane);
                bool w_ok = true;
                const uint32_t nst = ((nt + kSub - 1) / kSub + spar - 1) / spar * spar;
                for (uint32_t j = 0; j < nst; ++j) {
                    const uint32_t x0 = j * kSub, own = x0 & 31;
                    if (own == 0 && j != 0) {
                        page = next;
                        next = look(x0 + 32 + lane);
                        measure(x0 + lane);
                    }
                    if (lane == 0 && round > 0) w_ok = mbar_wait(&empty[s], (round - 1) & 1);
                    if (!__shfl_sync(0xffffffffu, w_ok ? 1 : 0, 0)) {
                        ok = false;
                        break;
                    }
                    const uint32_t sub = static_cast<uint32_t>(lane) - own;  // this lane's tile of the stage, if < kSub
                    const bool copies = sub < kSub && valid != 0;
                    if constexpr (kStep) {
                        if ((word & kRowAppend) && tail && x0 < nt && x0 + kSub >= nt) {
                            // the new row, before the tile that holds it (the segment's last) is
                            // copied: stored by all lanes, each of which fences the async proxy
                            const uint32_t owner = own + (nt - 1 - x0);
                            const int32_t pg = __shfl_sync(0xffffffffu, valid != 0 ? page : -1, owner);
                            if (pg >= 0) {
                                uint32_t r;
                                (void)a.pv.page_size.div(len - 1, r);
                                const uint64_t to = static_cast<uint64_t>(pg) * a.pv.page_stride + static_cast<uint64_t>(r) * (KVH * 128);
                                const __half* kn = a.k_new + static_cast<uint64_t>(b) * a.kv_new_stride;
                                const __half* vn = a.v_new + static_cast<uint64_t>(b) * a.kv_new_stride;
                                for (uint32_t gi = lane; gi < KVH * 8; gi += 32) {
                                    const uint32_t e = (gi >> 3) * 128 + (gi & 7) * 8;
                                    uint4 lo = *reinterpret_cast<const uint4*>(kn + e);
                                    uint4 hi4 = *reinterpret_cast<const uint4*>(kn + e + 64);
                                    const uint4 v0 = *reinterpret_cast<const uint4*>(vn + e);
                                    const uint4 v1 = *reinterpret_cast<const uint4*>(vn + e + 64);
                                    if (a.rotate) {
                                        const uint64_t ti = static_cast<uint64_t>(len - 1) * 64 + (gi & 7) * 8;
                                        rot8_pairs(lo, hi4, *reinterpret_cast<const uint4*>(a.cos + ti),
                                                   *reinterpret_cast<const uint4*>(a.sin + ti));
                                    }
                                    *reinterpret_cast<uint4*>(a.pv.k + to + e) = lo;
                                    *reinterpret_cast<uint4*>(a.pv.k + to + e + 64) = hi4;
                                    *reinterpret_cast<uint4*>(a.pv.v + to + e) = v0;
                                    *reinterpret_cast<uint4*>(a.pv.v + to + e + 64) = v1;
                                }
                            }
                            asm volatile("fence.proxy.async.global;" ::: "memory");
                            __syncwarp();
                        }
                    }
                    const uint32_t count = __popc(__ballot_sync(0xffffffffu, copies));
                    if (sub < kSub) st_valid[s][sub] = valid;
                    if (sub == 0) st_last[s] = j + spar >= nst;
                    __syncwarp();
                    if (sub == 0) {
                        if (count) mbar_arrive_expect_tx(&full[s], count * 2 * sub_bytes);
                        else mbar_arrive(&full[s]);
                    }
                    __syncwarp();
                    if (copies) {
                        uint8_t* stg = ring + s * stage_bytes + sub * sub_bytes;
                        tc::tma_load_4d_hint(stg, &map_k, 0, static_cast<int32_t>(r0), 0, page, &full[s], policy);
                        tc::tma_load_4d_hint(stg + kSub * sub_bytes, &map_v, 0, static_cast<int32_t>(r0), 0, page,
                                             &full[s], policy);
                    }
                    ++i;
                    if (++s == stages) {
                        s = 0;
                        ++round;
                    }
                    if (j == 0) {
                        // behind the first tiles: the segment's Q row and where its result goes
                        if (lane == 0 && q_rows.in_use()) ok = mbar_wait(&qempty[q_rows.next()], q_rows.free_parity());
                        const uint32_t qs = q_rows.begin();
                        if (lane == 0 && ok) {
                            uint8_t* slot = qslots + qs * t.qslot_bytes;
                            const uint32_t q_bytes = a.num_heads * 256;
                            uint32_t* meta = reinterpret_cast<uint32_t*>(slot + q_bytes + 256);
                            meta[0] = b;
                            meta[1] = whole ? kNoSeg : blockIdx.x + b;   // the partial's number
                            meta[2] = word;
                            meta[3] = nt;
                            const bool rot = kStep && (word & kRowRotate) != 0;
                            mbar_arrive_expect_tx(&qfull[qs], q_bytes + (rot ? 256u : 0u));
                            bulk_g2s_plain(slot, a.q + static_cast<uint64_t>(b) * a.q_stride, q_bytes, &qfull[qs]);
                            if (rot) {
                                const uint64_t p = (word & kRowCapped) ? static_cast<uint64_t>(a.kv_len[b]) : len - 1u;
                                bulk_g2s_plain(slot + q_bytes, a.cos + p * 64, 128, &qfull[qs]);
                                bulk_g2s_plain(slot + q_bytes + 128, a.sin + p * 64, 128, &qfull[qs]);
                            }
                        }
                        if (!__shfl_sync(0xffffffffu, ok ? 1 : 0, 0)) {
                            ok = false;
                            q_rows.withdraw();
                            break;
                        }
                    }
                }
            }
        }
        // the end, for every stage parity
        for (uint32_t e = 0; e < spar && ok; ++e) {
            bool w_ok = true;
            if (lane == 0 && round > 0) w_ok = mbar_wait(&empty[s], (round - 1) & 1);
            if (!__shfl_sync(0xffffffffu, w_ok ? 1 : 0, 0)) {
                ok = false;
                break;
            }
            if (lane == 0) {
                st_last[s] = kNoSeg;
                mbar_arrive(&full[s]);
            }
            ++i;
            if (++s == stages) {
                s = 0;
                ++round;
            }
        }
        // never leave the CTA with copies in flight into its shared memory
        if (lane == 0) {
            for (uint32_t j = i > stages ? i - stages : 0; j < i; ++j) (void)mbar_wait(&full[j % stages], (j / stages) & 1);
            for (uint32_t j = q_rows.oldest(); j < q_rows.issued(); ++j)
                (void)mbar_wait(&qfull[SlotPair::slot(j)], SlotPair::parity(j));
        }
    } else {
        // ---- consumers: KV head warp % KVH; tile `sub` of the stages of parity `par`
        const uint32_t kvh = warp % KVH, jw = warp / KVH, sub = jw % kSub, par = jw / kSub;
        const int g = lane >> 2, tt = lane & 3;
        const uint32_t live_t = (a.group + 1) / 2;    // lanes with tt below it hold heads of the group
        const bool dumps = static_cast<uint32_t>(tt) < live_t;
        float* const my_comb = comb + (static_cast<uint32_t>(tt) * 8 + g) * kStateFloats;
        const uint32_t slot_floats = 8 * live_t * kStateFloats;
        WarpState st;
        uint32_t qf[8][2];
        uint32_t seg = 0, seq = 0, part = 0, tiles = 0;
        uint32_t dumped = 0, joined[3] = {0u, 0u, 0u};  // fills of its slot, and of those that it reads
        bool fresh = true;
        if (blockIdx.x == 0) {
            // one CTA's consumers, which have nothing to do yet, tell the join where the partials will lie
            ok = mbar_wait(tables, 0);
            const Cut cut = Cut::of(prefix[B], t.ctas);
            for (uint32_t b = threadIdx.x; ok && b < B; b += kPtConsumers * 32) {
                const uint32_t u0 = prefix[b], u1 = prefix[b + 1];
                uint2 c = make_uint2(0u, 0u);
                if (u1 > u0) {
                    const uint32_t c0 = cut.cta_of(u0 + kBegin);
                    c = make_uint2(c0 + b, cut.cta_of(u1 - 1) - c0 + 1);
                }
                t.cuts[b] = c;
            }
        }
        for (uint32_t s = par, round = 0;; s += spar) {
            if (s >= stages) {  // (a multiple of spar)
                s -= stages;
                ++round;
            }
            if (!mbar_wait(&full[s], round & 1)) {
                ok = false;
                break;
            }
            const uint32_t last = st_last[s];
            if (last == kNoSeg) break;
            if (fresh) {
                fresh = false;
                state_init(st);
                st.m0 = st.m1 = kNoMax;
                const uint32_t qs = seg & 1;
                if (!mbar_wait(&qfull[qs], (seg >> 1) & 1)) {
                    ok = false;
                    break;
                }
                const uint8_t* slot = qslots + qs * t.qslot_bytes;
                const uint8_t* tail = slot + a.num_heads * 256;
                const uint32_t* meta = reinterpret_cast<const uint32_t*>(tail + 256);
                seq = meta[0];
                part = meta[1];
                tiles = meta[3];
                if (static_cast<uint32_t>(g) < a.group) {
                    const uint8_t* qrow = slot + (kvh * a.group + g) * 256;
                    uint4 w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = lds128(qrow + (32 * j + 8 * tt) * 2);
                    if (kStep && (meta[2] & kRowRotate)) {
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            rot8_pairs(w[j], w[j + 2], lds128(tail + (32 * j + 8 * tt) * 2),
                                       lds128(tail + 128 + (32 * j + 8 * tt) * 2));
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        qf[2 * j][0] = w[j].x;
                        qf[2 * j][1] = w[j].y;
                        qf[2 * j + 1][0] = w[j].z;
                        qf[2 * j + 1][1] = w[j].w;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) qf[j][0] = qf[j][1] = 0u;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&qempty[qs]);
            }
            const uint32_t valid = st_valid[s][sub];
            if (valid != 0) {
                const uint8_t* kt = ring + s * stage_bytes + sub * sub_bytes + kvh * (2 * kTile * 128);
                const uint8_t* vt = kt + kSub * sub_bytes;
                float sc[4];
                uint4 va[4][2];
                if (valid == kTile) {
                    uint4 ka[4], kb[4];
                    load_k_frags_sw<false>(kt, g, tt, valid, ka, kb);
                    tile_scores<false>(sc, ka, kb, qf, tile_token(g), valid, a.scale_log2);
                    load_v_frags_sw<false>(vt, g, tt, valid, va);
                } else {
                    uint4 ka[4], kb[4];
                    load_k_frags_sw<true>(kt, g, tt, valid, ka, kb);
                    tile_scores<true>(sc, ka, kb, qf, tile_token(g), valid, a.scale_log2);
                    load_v_frags_sw<true>(vt, g, tt, valid, va);
                }
                tile_softmax_pv<true>(st, sc, va, g, tt);
                // (released as soon as the rows were in registers, a stage made 64 ragged sequences
                // 112.9 us instead of 111.1)
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[s]);
            } else {
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[s]);
            }
            if (!last) continue;
            // ---- the segment's end: join the KV head's warps, pair by pair: at
            // level 1, 2, 4 the warps jw with that lowest bit set leave their state to
            // jw - level, each in a slot of its own. Warp jw has tiles of the segment
            // if it has more than jw; the others are left out, so that short segments
            // take few steps.
            fresh = true;
            state_finish(st);
            bool mine = jw == 0;
#pragma unroll
            for (uint32_t l = 0; (1u << l) < npar; ++l) {
                const uint32_t level = 1u << l;
                if (jw & level) {
                    if (jw < tiles) {
                        const uint32_t id = kvh * (npar - 1) + jw - 1;
                        if (dumped > 0 && !mbar_wait(&cempty[id], (dumped - 1) & 1)) ok = false;
                        if (dumps) state_dump(st, my_comb + id * slot_floats);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&cfull[id]);
                        ++dumped;
                    }
                    break;
                }
                if (jw + level >= tiles) continue;
                const uint32_t id = kvh * (npar - 1) + jw + level - 1;
                if (!mbar_wait(&cfull[id], joined[l] & 1)) ok = false;
                if (dumps) state_join(st, my_comb + id * slot_floats);
                __syncwarp();
                if (lane == 0) mbar_arrive(&cempty[id]);
                ++joined[l];
            }
            ++seg;
            if (!ok) break;
            if (!mine) continue;
#pragma unroll
            for (int hs = 0; hs < 2; ++hs) {
                const uint32_t hh = 2 * tt + hs;
                if (hh >= a.group) continue;
                const uint32_t head = kvh * a.group + hh;
                const float m = hs ? st.m1 : st.m0, l = hs ? st.l1 : st.l0;
                if (part == kNoSeg) {
                    const float inv = l != 0.f ? 1.f / l : 0.f;
                    __half* o = a.out + static_cast<uint64_t>(seq) * a.out_stride + head * 128;
#pragma unroll
                    for (int mt = 0; mt < 8; ++mt)
                        *reinterpret_cast<__half2*>(o + 64 * (mt >> 2) + 8 * g + 2 * (mt & 3)) =
                            __floats2half2_rn(st.o[mt][hs] * inv, st.o[mt][hs + 2] * inv);
                } else {
                    float* o = t.po + (static_cast<uint64_t>(part) * a.num_heads + head) * 128;
#pragma unroll
                    for (int mt = 0; mt < 8; ++mt)
                        *reinterpret_cast<float2*>(o + 64 * (mt >> 2) + 8 * g + 2 * (mt & 3)) =
                            make_float2(st.o[mt][hs], st.o[mt][hs + 2]);
                    if (g == 0) {
                        t.pm[static_cast<uint64_t>(head) * t.parts + part] = m;
                        t.pl[static_cast<uint64_t>(head) * t.parts + part] = l;
                    }
                }
            }
        }
    }
    if (!ok) atomicOr(&g_device_error, kErrWaitTimeout);
}

// Joins the partials of one (head, sequence) that was cut, 128 / kDims CTAs
// each for kDims output dims; sequences that one segment covered are done,
// those without tokens get zeros. The first kAhead rows of a thread are on
// their way while the weights are worked out (the partials lie in L2; latency
// is what this kernel spends). Its CTAs fit beside the tiled kernel's (registers
// and shared memory), so they stand ready when that ends; with 256 threads fewer
// do (64 ragged sequences 112.3 us against 110.6 in all, the step of 48 sequences
// 80.5 against 78.6). Joined by the tiled kernel itself, in the CTA that completes
// a sequence, 113.5 and 84.1: its successor's CTAs then start with nothing done.
constexpr int kJoinThreads = 128;

template <int kDims>
__global__ void __launch_bounds__(kJoinThreads, 8) paged_join_kernel(const TiledArgs t) {
    constexpr int kThreads = kJoinThreads;
    constexpr int kLanes = kDims / 4;                     // threads of a partial's row, four dims each
    constexpr int kRowsAtOnce = kThreads / kLanes;
    constexpr int kWarps = kThreads / 32;
    constexpr int kAhead = 6;
    __shared__ float wgt[kPtMaxCtas];
    __shared__ float red[2][kWarps];
    __shared__ float4 sums[kWarps][kLanes];
    pdl_wait_primary();
    pdl_launch_dependents();
    const PagedArgs& a = t.p;
    const uint32_t split = 128 / kDims;
    const uint32_t h = blockIdx.x / split, d0 = (blockIdx.x - h * split) * kDims, b = blockIdx.y, tid = threadIdx.x;
    const uint2 where = __ldcg(t.cuts + b);
    const uint32_t n = where.y;
    if (n > kPtMaxCtas || where.x + n > t.parts) return;  // the tiled kernel gave up before it wrote them
    __half* out = a.out + static_cast<uint64_t>(b) * a.out_stride + h * 128 + d0;
    if (n == 0) {
        if (tid < kDims / 2) reinterpret_cast<__half2*>(out)[tid] = __floats2half2_rn(0.f, 0.f);
        return;
    }
    if (n == 1) return;
    const uint64_t p0 = where.x;
    const uint32_t dl = tid % kLanes, r = tid / kLanes;
    const float* po = t.po + (p0 * a.num_heads + h) * 128 + d0 + dl * 4;
    const uint64_t step = static_cast<uint64_t>(a.num_heads) * 128;
    const float* pm = t.pm + static_cast<uint64_t>(h) * t.parts + p0;
    const float* pl = t.pl + static_cast<uint64_t>(h) * t.parts + p0;
    float4 x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
        const uint32_t i = r + k * kRowsAtOnce;
        x[k] = i < n ? __ldcg(reinterpret_cast<const float4*>(po + i * step)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const float l0 = tid < n ? __ldcg(pl + tid) : 0.f;
    float m = kNoMax;
    for (uint32_t i = tid; i < n; i += kThreads) {
        wgt[i] = __ldcg(pm + i);
        m = fmaxf(m, wgt[i]);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    if ((tid & 31) == 0) red[0][tid >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, red[0][w]);
    float l = 0.f;
    for (uint32_t i = tid; i < n; i += kThreads) {
        const float w = ex2(wgt[i] - m);
        wgt[i] = w;
        l = fmaf(w, i == tid ? l0 : __ldcg(pl + i), l);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    if ((tid & 31) == 0) red[1][tid >> 5] = l;
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) l += red[1][w];
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t i = r; i < n;) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const float w = i + k * kRowsAtOnce < n ? wgt[i + k * kRowsAtOnce] : 0.f;
            o.x = fmaf(w, x[k].x, o.x);
            o.y = fmaf(w, x[k].y, o.y);
            o.z = fmaf(w, x[k].z, o.z);
            o.w = fmaf(w, x[k].w, o.w);
        }
        i += kAhead * kRowsAtOnce;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const uint32_t j = i + k * kRowsAtOnce;
            x[k] = j < n ? __ldcg(reinterpret_cast<const float4*>(po + j * step)) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    // a warp's rows, then the warps'
#pragma unroll
    for (int off = 16; off >= kLanes; off >>= 1) {
        o.x += __shfl_xor_sync(0xffffffffu, o.x, off);
        o.y += __shfl_xor_sync(0xffffffffu, o.y, off);
        o.z += __shfl_xor_sync(0xffffffffu, o.z, off);
        o.w += __shfl_xor_sync(0xffffffffu, o.w, off);
    }
    if ((tid & 31) < kLanes) sums[tid >> 5][dl] = o;
    __syncthreads();
    if (tid < kLanes) {
        o = sums[0][tid];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            const float4 y = sums[w][tid];
            o.x += y.x;
            o.y += y.y;
            o.z += y.z;
            o.w += y.w;
        }
        const float inv = l != 0.f ? 1.f / l : 0.f;
        reinterpret_cast<__half2*>(out)[2 * tid] = __floats2half2_rn(o.x * inv, o.y * inv);
        reinterpret_cast<__half2*>(out)[2 * tid + 1] = __floats2half2_rn(o.z * inv, o.w * inv);
    }
}

int tiled_sms() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    return n;
}

bool tiled_kvh(size_t kvh) { return kvh == 1 || kvh == 2 || kvh == 4 || kvh == 8; }

struct TiledWorkspace {
    size_t po, pm, pl, cuts, total_bytes;
};

TiledWorkspace tiled_layout(size_t num_seqs, size_t num_heads) {
    TiledWorkspace w{};
    const size_t P = kPtMaxCtas + num_seqs;
    w.po = 0;
    w.pm = P * num_heads * 128;
    w.pl = w.pm + P * num_heads;
    w.cuts = (w.pl + P * num_heads + 1) / 2 * 2;
    w.total_bytes = ((w.cuts + 2 * num_seqs) * sizeof(float) + 255) / 256 * 256;
    return w;
}

template <uint32_t KVH, bool kStep>
int launch_tiled_kvh(const TiledArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, size_t smem, cudaStream_t stream) {
    static std::atomic<uint64_t> attr_done{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return B2_ERR_CUDA;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(attr_done.load() & bit)) {
        const int st = cuda_status(cudaFuncSetAttribute(paged_tiled_kernel<KVH, kStep>,
                                                        cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                        static_cast<int>(kPtSmemLimit)));
        if (st != B2_OK) return st;
        attr_done.fetch_or(bit);
    }
    return launch_pdl(paged_tiled_kernel<KVH, kStep>, dim3(a.ctas.d), dim3(kPtThreads), smem, stream, a, mk, mv);
}

}  // namespace

bool paged_tiled_fits(const PagedArgs& a) {
    if (a.head_dim != 128 || !tiled_kvh(a.num_kv_heads) || a.group > 8 || a.num_seqs > kPtMaxSeqs ||
        a.pv.page_size.d < kPtMinPage)
        return false;
    // table rows leave room for the flags; the whole batch's units fit 31 bits; strides fit a tensor map
    const uint64_t tiles = (static_cast<uint64_t>(a.pv.capacity) / a.pv.page_size.d + 1) *
                               ((a.pv.page_size.d + kTile - 1) / kTile) + pt_begin(a.num_kv_heads);
    return a.pv.table_rows <= kRowBits && tiles * a.num_seqs < (1ull << 31) && a.pv.page_stride < (1ull << 38) &&
           a.out_stride % 2 == 0 && reinterpret_cast<uintptr_t>(a.out) % 4 == 0;
}

size_t paged_tiled_workspace(size_t num_seqs, size_t num_heads, size_t num_kv_heads, size_t head_dim) {
    if (head_dim != 128 || !tiled_kvh(num_kv_heads) || num_heads / num_kv_heads > 8 || num_seqs > kPtMaxSeqs) return 0;
    return tiled_layout(num_seqs, num_heads).total_bytes;
}

int launch_paged_tiled(const PagedArgs& p, bool step, void* workspace, cudaStream_t stream) {
    const uint32_t kvh = p.num_kv_heads, H = p.num_heads, B = p.num_seqs;
    const TiledWorkspace w = tiled_layout(B, H);
    float* ws = static_cast<float*>(workspace);
    TiledArgs a{};
    a.p = p;
    a.tiles_per_page = FastDiv::of((p.pv.page_size.d + kTile - 1) / kTile);
    const uint32_t ctas = std::min<uint32_t>(static_cast<uint32_t>(tiled_sms()), kPtMaxCtas);
    a.ctas = FastDiv::of(ctas);
    a.po = ws + w.po;
    a.pm = ws + w.pm;
    a.pl = ws + w.pl;
    a.parts = kPtMaxCtas + B;
    a.cuts = reinterpret_cast<uint2*>(ws + w.cuts);
    // shared memory: the ring, two Q slots, the joins' states, the tables, the barriers
    const uint32_t stage = 2 * pt_sub(kvh) * kvh * 2 * kTile * 128;
    a.qslot_bytes = H * 256 + 256 + 128;
    const uint32_t comb = kvh * (pt_npar(kvh) - 1) * 8 * ((p.group + 1) / 2) * kStateFloats * 4;
    const uint32_t tab = ((3 * B + 1) * 4 + 15) / 16 * 16;
    const uint32_t fixed = 1024 + 2 * a.qslot_bytes + comb + tab + (2 * kPtMaxStages + 21) * 8;
    if (fixed >= kPtSmemLimit) return B2_ERR_UNSUPPORTED;
    // a multiple of the parities: each slot of the ring is one parity's, whose warps see all of its
    // barrier's phases (a wait for a phase two ahead would pass at once)
    a.stages = std::min((kPtSmemLimit - fixed) / stage, kPtMaxStages) / pt_spar(kvh) * pt_spar(kvh);
    if (a.stages < 2) return B2_ERR_UNSUPPORTED;
    a.off_q = a.stages * stage;
    a.off_comb = a.off_q + 2 * a.qslot_bytes;
    a.off_tab = a.off_comb + comb;
    a.off_bar = a.off_tab + tab;
    const size_t smem = 1024 + a.off_bar + (2 * a.stages + 21) * 8;
    CUtensorMap mk, mv;
    if (encode_token_rows_by_column_block_seqs(&mk, p.pv.k, p.pv.page_size.d, kvh * 256, p.pv.num_pages,
                                               p.pv.page_stride * 2, kTile) != 0 ||
        encode_token_rows_by_column_block_seqs(&mv, p.pv.v, p.pv.page_size.d, kvh * 256, p.pv.num_pages,
                                               p.pv.page_stride * 2, kTile) != 0)
        return B2_ERR_CUDA;
    int st;
    switch (kvh * 2 + (step ? 1 : 0)) {
        case 2: st = launch_tiled_kvh<1, false>(a, mk, mv, smem, stream); break;
        case 3: st = launch_tiled_kvh<1, true>(a, mk, mv, smem, stream); break;
        case 4: st = launch_tiled_kvh<2, false>(a, mk, mv, smem, stream); break;
        case 5: st = launch_tiled_kvh<2, true>(a, mk, mv, smem, stream); break;
        case 8: st = launch_tiled_kvh<4, false>(a, mk, mv, smem, stream); break;
        case 9: st = launch_tiled_kvh<4, true>(a, mk, mv, smem, stream); break;
        case 16: st = launch_tiled_kvh<8, false>(a, mk, mv, smem, stream); break;
        default: st = launch_tiled_kvh<8, true>(a, mk, mv, smem, stream); break;
    }
    if (st != B2_OK) return st;
    // at most a few CTAs an SM; the fewer (head, sequence) pairs, the finer each is shared out
    const uint32_t pairs = B * H;
    if (pairs * 4 <= ctas)
        return launch_pdl(paged_join_kernel<8>, dim3(16 * H, B), dim3(kJoinThreads), 0, stream, a);
    if (pairs <= ctas)
        return launch_pdl(paged_join_kernel<32>, dim3(4 * H, B), dim3(kJoinThreads), 0, stream, a);
    return launch_pdl(paged_join_kernel<128>, dim3(H, B), dim3(kJoinThreads), 0, stream, a);
}

unsigned int device_error_paged_tiled() {
    unsigned int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(v)) != cudaSuccess) return 0;
    return v;
}

int clear_device_error_paged_tiled() {
    const unsigned int zero = 0;
    return cuda_status(cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero)));
}

}  // namespace b2
