// Decode attention over a paged KV cache for sm_100a: one new query token for
// each of B sequences whose K/V rows lie in pages (paged.cuh). The algebra is
// the split-KV attention and chunk merge of the reference
// (src/kernels/causal_attention.hip.cpp:493-595, :719-819): a part of a
// sequence's tokens gives m = max score, l = sum e^(s - m) and o = sum
// e^(s - m) v; parts are joined with weights e^(m_i - m).
//
// head_dim 128 with up to 8 query heads a KV head runs the tiled kernel where it
// can (paged_decode_sm100.cu); paged_split_kernel runs every shape (head dims of
// whole 16-byte pieces up to 256, any number of heads, any page size): a CTA
// takes one part of one sequence for up to four query heads of a KV head.
// head_dim / 8 lanes read a token's row as 16-byte pieces and keep q and o in
// registers in 32 bits; paged_merge_kernel joins the parts. Each K/V byte is read once per four
// query heads. Bound by its instructions:
// 64 sequences of 4096 tokens take 207 us with 16 heads over 4 (2.6 TB/s), 383
// with 32 over 8 (2.8), 121 with 8 over 2 (2.2), 69 with 4 over 1 (2.0); 520 with
// 40 over 4 (1.0), whose rows are read three times; 64 of 1 to 4096 tokens,
// lengths spread over their logarithm, 54 us (1.5 TB/s), 96, 31, 28 and 123.
#include <math.h>

#include <algorithm>

#include "paged_append.h"
#include "paged_decode.h"

namespace b2 {
namespace {

constexpr uint32_t kPgMaxSeqs = 65535;      // a grid dimension
constexpr uint32_t kPgHeads = 4;            // query heads of a CTA of the split kernel
constexpr uint32_t kPgThreads = 128;
constexpr uint32_t kPgUnroll = 4;           // tokens of a lane group in flight
constexpr uint32_t kPgMaxSplits = 512;
// Tokens of a part at least. With 64 / 192 / 512, 16 heads over 4: one sequence of 300 tokens 12.6 / 17 / 23 us,
// one of 32K 62 / 46 / 59, 64 of 1 to 4096 tokens 58 / 54 / 58.
constexpr uint32_t kPgPart = 192;
constexpr uint32_t kPgMergeThreads = 256;
// The maximum before any score: below every finite one and finite itself, so that a score of -infinity
// weighs 0, and one that is NaN, which no maximum shows, still makes a NaN of the weight and the output.
constexpr float kPgNoMax = -1e30f;

struct SplitArgs {
    PagedArgs p;
    float* po;  // [B][H][splits][head_dim]
    float* pm;  // [B][H][splits], log2 units
    float* pl;
    uint32_t splits;
    uint32_t chunks;  // CTAs of a KV head's group: ceil(group / kPgHeads)
    uint32_t lanes;   // lanes of a token row: a power of two >= head_dim / 8
};

// Parts of a sequence of len tokens (those past them neither run nor are merged).
__device__ __forceinline__ uint32_t parts_of(const SplitArgs& t, uint32_t len) {
    return min(t.splits, max(1u, (len + kPgPart - 1) / kPgPart));
}

// Whether entry b's query is rotated: its position is in the tables (one past
// them sets the error bit).
__device__ __forceinline__ bool paged_rotates(const PagedArgs& a, uint32_t b, uint32_t& pos) {
    if (!a.rotate) return false;
    const int32_t p = a.kv_len[b];
    pos = static_cast<uint32_t>(p);
    if (p >= 0 && pos >= a.rope_rows) atomicOr(&g_device_error, kErrBadPosition);
    return p >= 0 && pos < a.rope_rows;
}

__device__ __forceinline__ void half8(const uint4& w, float (&x)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// 16 bytes that are read once (coherent: the append before may have written them).
__device__ __forceinline__ uint4 ld_once(const __half* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p)
                 : "memory");
    return r;
}

template <uint32_t G>
__global__ void __launch_bounds__(kPgThreads) paged_split_kernel(const SplitArgs t) {
    extern __shared__ float sm[];  // [slots][G][head_dim] o, then [slots][G] m and l
    pdl_wait_primary();
    pdl_launch_dependents();
    const PagedArgs& a = t.p;
    const uint32_t split = blockIdx.x, b = blockIdx.z;
    const uint32_t kvh = blockIdx.y / t.chunks, chunk = blockIdx.y - kvh * t.chunks;
    const uint32_t d = a.head_dim, d8 = d / 8;
    const uint32_t nheads = min(G, a.group - chunk * G);
    const uint32_t head0 = kvh * a.group + chunk * G;
    const int32_t row = paged_row(a.pv, b);
    const uint32_t len = paged_tokens(a, row, a.kv_len[b]);
    // an even share of the tokens
    const uint32_t parts = parts_of(t, len);
    if (split >= parts) return;
    const uint32_t per = (len + parts - 1) / parts;
    const uint32_t begin = min(split * per, len), end = min(begin + per, len);

    const uint32_t li = threadIdx.x % t.lanes, slot = threadIdx.x / t.lanes, slots = kPgThreads / t.lanes;
    const bool on = li < d8;
    float q[G][8], o[G][8], m[G], l[G];
#pragma unroll
    for (uint32_t g = 0; g < G; ++g) {
        m[g] = kPgNoMax;
        l[g] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) q[g][i] = o[g][i] = 0.f;
    }
    if (begin < end) {
        uint32_t pos = 0;
        const bool rot = paged_rotates(a, b, pos);
#pragma unroll
        for (uint32_t g = 0; g < G; ++g) {
            if (g >= nheads || !on) continue;
            const __half* qr = a.q + b * a.q_stride + static_cast<uint64_t>(head0 + g) * d;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t e = li * 8 + i, half = d / 2;
                float x = __half2float(qr[e]);
                if (rot) {
                    // the stored form of a rotated row: products and sum rounded apart, then 16 bits
                    const bool hi = e >= half;
                    const uint64_t ti = static_cast<uint64_t>(pos) * half + (hi ? e - half : e);
                    const float y = __half2float(qr[hi ? e - half : e + half]);
                    const float c = __half2float(a.cos[ti]), s = __half2float(a.sin[ti]);
                    x = hi ? __fadd_rn(__fmul_rn(x, c), __fmul_rn(y, s)) : __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
                    x = __half2float(__float2half_rn(x));
                }
                q[g][i] = x * a.scale_log2;
            }
        }
    }
    // every lane of a warp makes the same number of rounds (the shuffles below)
    for (uint32_t base = begin; base < end; base += slots * kPgUnroll) {
        uint4 kw[kPgUnroll], vw[kPgUnroll];
        bool in[kPgUnroll];
#pragma unroll
        for (uint32_t u = 0; u < kPgUnroll; ++u) {
            const uint32_t tok = base + u * slots + slot;
            kw[u] = vw[u] = make_uint4(0u, 0u, 0u, 0u);
            in[u] = false;
            if (tok < end) {
                uint32_t r;
                const uint32_t j = a.pv.page_size.div(tok, r);
                const int32_t page = paged_page(a.pv, row, j);
                if (page >= 0) {
                    in[u] = true;
                    if (on) {
                        const uint64_t at = static_cast<uint64_t>(page) * a.pv.page_stride +
                                            (static_cast<uint64_t>(r) * a.num_kv_heads + kvh) * d + li * 8;
                        kw[u] = ld_once(a.pv.k + at);
                        vw[u] = ld_once(a.pv.v + at);
                    }
                }
            }
        }
        float sc[kPgUnroll][G];
#pragma unroll
        for (uint32_t u = 0; u < kPgUnroll; ++u) {
            float k[8];
            half8(kw[u], k);
#pragma unroll
            for (uint32_t g = 0; g < G; ++g) {
                float x = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) x = fmaf(q[g][i], k[i], x);
                sc[u][g] = x;
            }
        }
        for (uint32_t off = 1; off < t.lanes; off <<= 1) {
#pragma unroll
            for (uint32_t u = 0; u < kPgUnroll; ++u)
#pragma unroll
                for (uint32_t g = 0; g < G; ++g) sc[u][g] += __shfl_xor_sync(0xffffffffu, sc[u][g], off);
        }
        // the running maximum moves once for these tokens
#pragma unroll
        for (uint32_t g = 0; g < G; ++g) {
            float mn = m[g];
#pragma unroll
            for (uint32_t u = 0; u < kPgUnroll; ++u)
                if (in[u]) mn = fmaxf(mn, sc[u][g]);
            const float c = exp2f(m[g] - mn);
            m[g] = mn;
            l[g] *= c;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[g][i] *= c;
#pragma unroll
            for (uint32_t u = 0; u < kPgUnroll; ++u) {
                sc[u][g] = in[u] ? exp2f(sc[u][g] - mn) : 0.f;
                l[g] += sc[u][g];
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < kPgUnroll; ++u) {
            float v[8];
            half8(vw[u], v);   // (zeros where there is no token)
#pragma unroll
            for (uint32_t g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < 8; ++i) o[g][i] = fmaf(sc[u][g], v[i], o[g][i]);
        }
    }
    // join the CTA's lane groups
    float* so = sm;
    float* s_m = so + slots * G * d;
    float* s_l = s_m + slots * G;
#pragma unroll
    for (uint32_t g = 0; g < G; ++g) {
        if (on) {
#pragma unroll
            for (int i = 0; i < 8; ++i) so[(slot * G + g) * d + li * 8 + i] = o[g][i];
        }
        if (li == 0) {
            s_m[slot * G + g] = m[g];
            s_l[slot * G + g] = l[g];
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < nheads * d; i += kPgThreads) {
        const uint32_t g = i / d, e = i - g * d;
        float M = kPgNoMax, L = 0.f, O = 0.f;
        for (uint32_t w = 0; w < slots; ++w) M = fmaxf(M, s_m[w * G + g]);
        for (uint32_t w = 0; w < slots; ++w) {
            const float c = exp2f(s_m[w * G + g] - M);
            L = fmaf(c, s_l[w * G + g], L);
            O = fmaf(c, so[(w * G + g) * d + e], O);
        }
        if (parts == 1) {
            a.out[b * a.out_stride + static_cast<uint64_t>(head0 + g) * d + e] =
                __float2half_rn(L != 0.f ? O / L : 0.f);
        } else {
            const uint64_t p = (static_cast<uint64_t>(b) * a.num_heads + head0 + g) * t.splits + split;
            t.po[p * d + e] = O;
            if (e == 0) {
                t.pm[p] = M;
                t.pl[p] = L;
            }
        }
    }
}

// Joins the parts of one (head, sequence): a thread four output dims of every
// few parts (a single part wrote the output itself).
__global__ void __launch_bounds__(kPgMergeThreads) paged_merge_kernel(const SplitArgs t) {
    __shared__ float red[2][kPgMergeThreads / 32];
    __shared__ float4 sums[kPgMergeThreads];
    pdl_wait_primary();
    pdl_launch_dependents();
    const PagedArgs& a = t.p;
    const uint32_t h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const uint32_t n = parts_of(t, paged_tokens(a, paged_row(a.pv, b), a.kv_len[b]));
    if (n == 1) return;
    const uint64_t p = (static_cast<uint64_t>(b) * a.num_heads + h) * t.splits;
    float m = kPgNoMax;
    for (uint32_t i = tid; i < n; i += kPgMergeThreads) m = fmaxf(m, t.pm[p + i]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    if ((tid & 31) == 0) red[0][tid >> 5] = m;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kPgMergeThreads / 32; ++w) m = fmaxf(m, red[0][w]);
    float l = 0.f;
    for (uint32_t i = tid; i < n; i += kPgMergeThreads) l = fmaf(exp2f(t.pm[p + i] - m), t.pl[p + i], l);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    if ((tid & 31) == 0) red[1][tid >> 5] = l;
    const uint32_t lanes = a.head_dim / 4, rows = kPgMergeThreads / lanes, r = tid / lanes, e = tid - r * lanes;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rows) {
#pragma unroll 4
        for (uint32_t i = r; i < n; i += rows) {
            const float c = exp2f(t.pm[p + i] - m);
            const float4 x = *reinterpret_cast<const float4*>(t.po + (p + i) * a.head_dim + e * 4);
            o.x = fmaf(c, x.x, o.x);
            o.y = fmaf(c, x.y, o.y);
            o.z = fmaf(c, x.z, o.z);
            o.w = fmaf(c, x.w, o.w);
        }
    }
    sums[tid] = o;
    __syncthreads();
    if (tid >= lanes) return;
    l = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < kPgMergeThreads / 32; ++w) l += red[1][w];
    for (uint32_t w = 1; w < rows; ++w) {
        const float4 x = sums[w * lanes + tid];
        o.x += x.x;
        o.y += x.y;
        o.z += x.z;
        o.w += x.w;
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    __half* out = a.out + b * a.out_stride + static_cast<uint64_t>(h) * a.head_dim + tid * 4;
    out[0] = __float2half_rn(o.x * inv);
    out[1] = __float2half_rn(o.y * inv);
    out[2] = __float2half_rn(o.z * inv);
    out[3] = __float2half_rn(o.w * inv);
}

// Most parts of a sequence for the split kernel: 16 CTAs an SM of 148 if all
// were as long as the longest. With 8 / 16 / 32, 16 heads over 4: 64 sequences of
// 1 to 4096 tokens (lengths spread over their logarithm) 73 / 54 / 51 us, 64 of
// 4096 tokens 213 / 208 / 222; 32 over 8: 126 / 96 / 84 and 383 / 384 / 389; 4
// over 1: 27.5 / 28 / 30 and 71 / 69 / 71.
uint32_t paged_splits(size_t num_seqs, size_t num_heads, size_t num_kv_heads) {
    const size_t group = num_heads / num_kv_heads;
    const size_t ctas = num_seqs * num_kv_heads * ((group + kPgHeads - 1) / kPgHeads);
    const size_t s = (16 * 148 + ctas - 1) / ctas;
    return static_cast<uint32_t>(s > kPgMaxSplits ? kPgMaxSplits : s);
}

struct PgWorkspace {
    size_t po, pm, pl, total_bytes;
};

PgWorkspace pg_layout(size_t num_seqs, size_t num_heads, size_t num_kv_heads, size_t head_dim) {
    PgWorkspace w{};
    const size_t parts = num_seqs * num_heads * paged_splits(num_seqs, num_heads, num_kv_heads);
    w.po = 0;
    w.pm = parts * head_dim;
    w.pl = w.pm + parts;
    w.total_bytes = ((w.pl + parts) * sizeof(float) + 255) / 256 * 256;
    // a call's strides decide between the kernels too: room for either
    w.total_bytes = std::max(w.total_bytes, paged_tiled_workspace(num_seqs, num_heads, num_kv_heads, head_dim));
    return w;
}

// Inputs of one paged decode, or of a decode step (step: the new rows are
// appended at position kv_len[b], bias 1).
struct PagedCall {
    const void* q;
    size_t q_stride;
    const void* k_pages;
    const void* v_pages;
    size_t page_stride, num_pages, page_size;
    const int32_t* table;
    size_t table_stride, table_rows;
    const int32_t* seqs;
    const int32_t* kv_len;
    int32_t bias;
    void* out;
    size_t out_stride;
    size_t num_seqs, num_heads, num_kv_heads, head_dim;
    void* workspace;
    size_t workspace_bytes;
    bool step;
    const void* k_new;
    const void* v_new;
    size_t kv_new_stride;
    const void* cos;
    const void* sin;
    size_t rope_rows;
    bool rotate;
};

int launch_paged(PagedCall c, cudaStream_t stream) {
    if (c.num_seqs == 0 || c.num_heads == 0 || c.num_kv_heads == 0 || c.head_dim == 0) return B2_NOTHING_TO_DO;
    if (c.num_heads % c.num_kv_heads != 0) return B2_NOTHING_TO_DO;
    if (!c.q || !c.kv_len || !c.out || !c.workspace) return B2_ERR_INVALID_ARG;
    if (c.step && (!c.k_new != !c.v_new)) return B2_ERR_INVALID_ARG;
    if (c.step && c.rotate && (!c.cos || !c.sin || c.rope_rows == 0)) return B2_ERR_INVALID_ARG;
    if (c.head_dim % 8 != 0 || (c.rotate && c.head_dim % 16 != 0) || c.head_dim > 256 || c.num_heads > 0xffffu ||
        c.num_seqs > kPgMaxSeqs || c.rope_rows > 0x7fffffffull)
        return B2_ERR_UNSUPPORTED;  // (num_kv_heads * ceil(group / 4) <= num_heads: a grid dimension)
    const size_t group = c.num_heads / c.num_kv_heads;
    const size_t kv_dim = c.num_kv_heads * c.head_dim, q_dim = c.num_heads * c.head_dim;
    if (c.q_stride == 0) c.q_stride = q_dim;
    if (c.out_stride == 0) c.out_stride = q_dim;
    if (c.kv_new_stride == 0) c.kv_new_stride = kv_dim;
    if (c.q_stride < q_dim || c.out_stride < q_dim || (c.k_new && c.kv_new_stride < kv_dim)) return B2_ERR_INVALID_ARG;
    PagedArgs a{};
    const int vst = make_paged_view(&a.pv, c.k_pages, c.v_pages, c.page_stride, c.num_pages, c.page_size, c.table,
                                    c.table_stride, c.table_rows, c.seqs, c.num_seqs, kv_dim);
    if (vst != B2_OK) return vst;
    if (!aligned16(c.q) || !aligned16(c.k_pages) || !aligned16(c.v_pages) || !aligned16(c.workspace) ||
        c.q_stride % 8 != 0 || a.pv.page_stride % 8 != 0)
        return B2_ERR_ALIGNMENT;
    if ((c.k_new && (!aligned16(c.k_new) || !aligned16(c.v_new) || c.kv_new_stride % 8 != 0)) ||
        (c.step && c.rotate && (!aligned16(c.cos) || !aligned16(c.sin))))
        return B2_ERR_ALIGNMENT;
    const PgWorkspace w = pg_layout(c.num_seqs, c.num_heads, c.num_kv_heads, c.head_dim);
    if (c.workspace_bytes < w.total_bytes) return B2_ERR_WORKSPACE;
    a.q = static_cast<const __half*>(c.q);
    a.q_stride = c.q_stride;
    a.kv_len = c.kv_len;
    a.bias = c.bias;
    a.out = static_cast<__half*>(c.out);
    a.out_stride = c.out_stride;
    a.num_seqs = static_cast<uint32_t>(c.num_seqs);
    a.num_heads = static_cast<uint32_t>(c.num_heads);
    a.num_kv_heads = static_cast<uint32_t>(c.num_kv_heads);
    a.group = static_cast<uint32_t>(group);
    a.head_dim = static_cast<uint32_t>(c.head_dim);
    a.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(c.head_dim));
    if (c.step) {
        a.rotate = c.rotate ? 1u : 0u;
        a.rope_rows = static_cast<uint32_t>(c.rope_rows);
        a.cos = static_cast<const __half*>(c.cos);
        a.sin = static_cast<const __half*>(c.sin);
        a.k_new = static_cast<const __half*>(c.k_new);
        a.v_new = static_cast<const __half*>(c.v_new);
        a.kv_new_stride = c.kv_new_stride;
    }
    if (paged_tiled_fits(a)) {
        const int st = launch_paged_tiled(a, c.step, c.workspace, stream);
        if (st != B2_ERR_UNSUPPORTED) return st;
    }
    if (c.step && c.k_new) {
        PagedAppend p{};
        p.k_new = c.k_new;
        p.v_new = c.v_new;
        p.k_pages = const_cast<void*>(c.k_pages);
        p.v_pages = const_cast<void*>(c.v_pages);
        p.page_stride = c.page_stride;
        p.num_pages = c.num_pages;
        p.page_size = c.page_size;
        p.table = c.table;
        p.table_stride = c.table_stride;
        p.table_rows = c.table_rows;
        p.seqs = c.seqs;
        p.cos = c.cos;
        p.sin = c.sin;
        p.rope_rows = c.rope_rows;
        p.num_tokens = c.num_seqs;
        p.num_kv_heads = c.num_kv_heads;
        p.head_dim = c.head_dim;
        p.k_stride = c.kv_new_stride;
        p.pos = c.kv_len;
        p.rotate = c.rotate;
        const int st = launch_append(p, stream);
        if (st != B2_OK) return st;
    }
    float* ws = static_cast<float*>(c.workspace);
    SplitArgs t{};
    t.p = a;
    t.po = ws + w.po;
    t.pm = ws + w.pm;
    t.pl = ws + w.pl;
    t.splits = paged_splits(c.num_seqs, c.num_heads, c.num_kv_heads);
    t.chunks = static_cast<uint32_t>((group + kPgHeads - 1) / kPgHeads);
    t.lanes = 1;
    while (t.lanes * 8 < a.head_dim) t.lanes <<= 1;
    const uint32_t slots = kPgThreads / t.lanes;
    const dim3 grid(t.splits, a.num_kv_heads * t.chunks, a.num_seqs);
    const size_t per = (a.head_dim + 2) * sizeof(float) * slots;
    int st;
    if (group == 1)
        st = launch_pdl(paged_split_kernel<1>, grid, dim3(kPgThreads), per, stream, t);
    else
        st = launch_pdl(paged_split_kernel<kPgHeads>, grid, dim3(kPgThreads), per * kPgHeads, stream, t);
    if (st != B2_OK || t.splits == 1) return st;
    return launch_pdl(paged_merge_kernel, dim3(a.num_heads, a.num_seqs), dim3(kPgMergeThreads), 0, stream, t);
}

}  // namespace

unsigned int device_error_paged() {
    unsigned int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(v)) != cudaSuccess) return 0;
    return v | device_error_paged_tiled();
}

int clear_device_error_paged() {
    const unsigned int zero = 0;
    const int st = cuda_status(cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero)));
    return st != B2_OK ? st : clear_device_error_paged_tiled();
}

}  // namespace b2

extern "C" size_t b2_decode_paged_workspace_bytes(size_t num_seqs, size_t num_heads, size_t num_kv_heads,
                                                  size_t head_dim) {
    if (num_seqs == 0 || num_seqs > b2::kPgMaxSeqs || num_kv_heads == 0 || num_heads == 0 ||
        num_heads % num_kv_heads != 0 || head_dim == 0 || head_dim > 256 || num_heads > 0xffffu)
        return 0;
    return b2::pg_layout(num_seqs, num_heads, num_kv_heads, head_dim).total_bytes;
}

extern "C" int b2_launch_causal_attention_decode_paged(
    const void* d_q, size_t q_seq_stride, const void* d_k_pages, const void* d_v_pages, size_t page_stride,
    size_t num_pages, size_t page_size, const int32_t* d_page_table, size_t table_stride, size_t table_rows,
    const int32_t* d_seqs, const int32_t* d_kv_len, int32_t kv_len_bias, void* d_out, size_t out_seq_stride,
    size_t num_seqs, size_t num_heads, size_t num_kv_heads, size_t head_dim, void* d_workspace,
    size_t workspace_bytes, b2_stream_t stream) {
    b2::PagedCall c{};
    c.q = d_q;
    c.q_stride = q_seq_stride;
    c.k_pages = d_k_pages;
    c.v_pages = d_v_pages;
    c.page_stride = page_stride;
    c.num_pages = num_pages;
    c.page_size = page_size;
    c.table = d_page_table;
    c.table_stride = table_stride;
    c.table_rows = table_rows;
    c.seqs = d_seqs;
    c.kv_len = d_kv_len;
    c.bias = kv_len_bias;
    c.out = d_out;
    c.out_stride = out_seq_stride;
    c.num_seqs = num_seqs;
    c.num_heads = num_heads;
    c.num_kv_heads = num_kv_heads;
    c.head_dim = head_dim;
    c.workspace = d_workspace;
    c.workspace_bytes = workspace_bytes;
    return b2::launch_paged(c, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int b2_launch_decode_step_paged_fused(
    const void* d_q, size_t q_seq_stride, const void* d_k_new, const void* d_v_new, size_t kv_new_stride,
    void* d_k_pages, void* d_v_pages, size_t page_stride, size_t num_pages, size_t page_size,
    const int32_t* d_page_table, size_t table_stride, size_t table_rows, const int32_t* d_seqs, const void* d_cos,
    const void* d_sin, size_t rope_rows, bool apply_rotation, const int32_t* d_pos, void* d_out,
    size_t out_seq_stride, size_t num_seqs, size_t num_heads, size_t num_kv_heads, size_t head_dim,
    void* d_workspace, size_t workspace_bytes, b2_stream_t stream) {
    b2::PagedCall c{};
    c.q = d_q;
    c.q_stride = q_seq_stride;
    c.k_pages = d_k_pages;
    c.v_pages = d_v_pages;
    c.page_stride = page_stride;
    c.num_pages = num_pages;
    c.page_size = page_size;
    c.table = d_page_table;
    c.table_stride = table_stride;
    c.table_rows = table_rows;
    c.seqs = d_seqs;
    c.kv_len = d_pos;
    c.bias = 1;
    c.out = d_out;
    c.out_stride = out_seq_stride;
    c.num_seqs = num_seqs;
    c.num_heads = num_heads;
    c.num_kv_heads = num_kv_heads;
    c.head_dim = head_dim;
    c.workspace = d_workspace;
    c.workspace_bytes = workspace_bytes;
    c.step = true;
    c.k_new = d_k_new;
    c.v_new = d_v_new;
    c.kv_new_stride = kv_new_stride;
    c.cos = d_cos;
    c.sin = d_sin;
    c.rope_rows = rope_rows;
    c.rotate = apply_rotation;
    return b2::launch_paged(c, reinterpret_cast<cudaStream_t>(stream));
}
