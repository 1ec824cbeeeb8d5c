// Rotary positions of packed rows, alone (b2_rope) or on the way of new keys and values into a paged cache
// (b2_kv_append).
//
// A head's first 2F values are F pairs; pair f of a token at position p turns by the angle p * inv_freq[f]:
//   a' = mscale (a cos - b sin),   b' = mscale (a sin + b cos)
// with (a, b) = (x[f], x[F + f]) in the half layout and (x[2f], x[2f + 1]) in the interleaved one; the values from 2F
// on pass through. The angle is formed and reduced to a quarter turn in 64 bits (a position of 10^6 times a frequency
// has only four bits of the turn's fraction left in 32), sine and cosine of the remainder in 32, and each result is
// rounded once, to the tensor's type.
//
// Bound by HBM: each value is read once and written once. A CTA takes one token, or four where there are many: their
// sines and cosines are computed once, a pair per thread, into shared memory, and every head's pairs use them. A thread's
// item is 16 bytes of a's and 16 bytes of b's (both layouts: the same F indices), the first one loaded before the angles
// are known. Measured on 16384 tokens of 32 heads of 128, bf16: 50.5 us, 5.3 TB/s (one token per CTA 59.6, two 55.1,
// eight 51.4); two items in flight per thread cost more occupancy than they bring (62.5). The bound of six CTAs per SM
// (40 registers) is the best for the append (58.9 us, 5.7 TB/s, for 15000 tokens of 32 + 2 x 8 heads; eight: 77). Rows off
// 16 bytes go value by value: the 16384 tokens into a given output take 123 us, by 16-byte items 45.
#include <cuda_bf16.h>

#include "common.cuh"
#include "host.hpp"

namespace b2 {
namespace {

__device__ unsigned int g_status;

constexpr int MAX_PAIRS = 512;

struct RopeArgs {
    // rows rotated from x to out: rope's tensor, or the queries beside appended keys
    const void* x;
    void* out;
    int64_t sxt, sxh, sot, soh;  // element strides of token and head
    int heads;
    // appended keys and values (kv_heads 0: none)
    const void *k, *v;
    void *k_cache, *v_cache;
    int64_t skt, skh, svt, svh, sc_page, sc_row, sc_head;
    int kv_heads;
    const int32_t *table, *cu_q, *lengths;
    int batch, table_ld, max_pages, num_pages, page_size;
    const int64_t* positions;  // null: the cache position
    const float* inv_freq;
    float mscale;
    int tokens, dim, pairs;
    int items;  // per token
    Divisor by_items, by_head;
};

template <class T>
__device__ __forceinline__ float to_f(T v) {
    return static_cast<float>(v);
}
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// V values as one load: 16 bytes (V * sizeof(T) == 16) or a single value.
template <class T, int V>
struct alignas(V == 1 ? sizeof(T) : 16) Vec {
    T e[V];
};

// The sequence of row r: the b with cu_q[b] <= r < cu_q[b + 1], or -1 (rows behind the last sequence). A warp looks at
// 32 borders at a time. All lanes return the same value.
__device__ __forceinline__ int find_sequence(const int32_t* cu_q, int batch, int r) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = batch;  // cu_q[lo] <= r is known (or lo = 0), cu_q[hi] > r is to be found
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int at = min(lo + (lane + 1) * step, hi);
        const unsigned past = __ballot_sync(0xffffffffu, cu_q[at] > r);
        if (!past) return -1;
        const int first = __ffs(past) - 1;
        hi = min(lo + (first + 1) * step, hi);
        lo = lo + first * step;
    }
    return (cu_q[lo] <= r && r < cu_q[lo + 1]) ? lo : -1;
}

constexpr int THREADS = 256;

template <class T, int V, bool INTER, int TOK>
__global__ void __launch_bounds__(THREADS, 6) rope_kernel(const __grid_constant__ RopeArgs a) {
    pdl_trigger();
    pdl_wait();
    __shared__ float s_cos[TOK][MAX_PAIRS], s_sin[TOK][MAX_PAIRS];
    __shared__ int64_t s_slot[TOK];  // element offset of the token's cache row; -1: dropped; -2: behind the last sequence
    using W = Vec<T, V>;
    const int t0 = blockIdx.x * TOK;
    const int per_head = a.dim / (2 * V);
    const int rot_items = a.pairs / V;
    const int total = min(TOK, a.tokens - t0) * a.items;

    struct Item {
        int tok, head, off_a, off_b, f;
        bool rotate;
    };
    auto item = [&](int i) {
        Item m;
        m.tok = TOK == 1 ? 0 : a.by_items.of(i);
        i -= m.tok * a.items;
        m.head = a.by_head.of(i);
        const int u = i - m.head * per_head;
        m.rotate = u < rot_items && m.head < a.heads + a.kv_heads;
        m.f = u * V;
        if (u < rot_items && !INTER) {
            m.off_a = u * V;
            m.off_b = a.pairs + u * V;
        } else {
            m.off_a = 2 * u * V;
            m.off_b = m.off_a + V;
        }
        return m;
    };
    auto load = [&](const Item& m, W& wa, W& wb) {
        const int64_t t = t0 + m.tok;
        const T* src;
        if (m.head < a.heads)
            src = static_cast<const T*>(a.x) + t * a.sxt + m.head * a.sxh;
        else if (m.head < a.heads + a.kv_heads)
            src = static_cast<const T*>(a.k) + t * a.skt + (m.head - a.heads) * a.skh;
        else
            src = static_cast<const T*>(a.v) + t * a.svt + (m.head - a.heads - a.kv_heads) * a.svh;
        wa = *reinterpret_cast<const W*>(src + m.off_a);
        wb = *reinterpret_cast<const W*>(src + m.off_b);
    };
    auto finish = [&](const Item& m, W& wa, W& wb) {
        const int64_t t = t0 + m.tok, slot = a.kv_heads ? s_slot[m.tok] : 0;
        if (slot == -2 || (slot < 0 && m.head >= a.heads)) return;
        if (m.rotate) {
            float x[2 * V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x[e] = to_f(wa.e[e]);
                x[V + e] = to_f(wb.e[e]);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float c = s_cos[m.tok][m.f + e], s = s_sin[m.tok][m.f + e];
                const int ia = INTER ? 2 * e : e, ib = INTER ? 2 * e + 1 : V + e;
                const float p = x[ia], q = x[ib];
                x[ia] = p * c - q * s;
                x[ib] = p * s + q * c;
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                wa.e[e] = from_f<T>(x[e]);
                wb.e[e] = from_f<T>(x[V + e]);
            }
        }
        T* dst;
        if (m.head < a.heads)
            dst = static_cast<T*>(a.out) + t * a.sot + m.head * a.soh;
        else if (m.head < a.heads + a.kv_heads)
            dst = static_cast<T*>(a.k_cache) + slot + (m.head - a.heads) * a.sc_head;
        else
            dst = static_cast<T*>(a.v_cache) + slot + (m.head - a.heads - a.kv_heads) * a.sc_head;
        *reinterpret_cast<W*>(dst + m.off_a) = wa;
        *reinterpret_cast<W*>(dst + m.off_b) = wb;
    };

    Item m;
    W wa, wb;
    int i = threadIdx.x;
    if (i < total) {
        m = item(i);
        load(m, wa, wb);
    }
    // Each token's position, cache row and angles, by the warps of its share of the CTA.
    constexpr int SHARE = THREADS / TOK;
    const int tok = threadIdx.x / SHARE, t = t0 + tok;
    if (t < a.tokens) {
        int64_t pos = 0;
        bool live = true;
        if (a.kv_heads) {
            int64_t slot = -1;
            const int b = find_sequence(a.cu_q, a.batch, t);
            live = b >= 0;
            if (live) {
                pos = (int64_t)a.lengths[b] - a.cu_q[b + 1] + t;
                if (pos >= 0) {  // below 2^31: t < cu_q[b + 1]
                    const int pi = (int)pos / a.page_size;
                    const int page = pi < a.max_pages ? a.table[(int64_t)b * a.table_ld + pi] : -1;
                    if (page >= 0 && page < a.num_pages)
                        slot = (int64_t)page * a.sc_page + ((int)pos - pi * a.page_size) * a.sc_row;
                }
            }
            if (threadIdx.x % SHARE == 0) {
                s_slot[tok] = live ? slot : -2;
                if (live && slot < 0) atomicOr(&g_status, B2_DEV_BAD_PAGE);
            }
        }
        if (a.positions) pos = a.positions[t];
        for (int f = threadIdx.x % SHARE; live && f < a.pairs; f += SHARE) {
            // turns = p * inv_freq / (2 pi), less its nearest quarter turn: |rest| <= 1/8
            const double turns = (double)pos * (double)a.inv_freq[f] * 0.15915494309189533577;
            const double frac = turns - rint(turns);
            const double quarter = rint(4.0 * frac);
            const int qn = (int)quarter & 3;
            float s, c;
            sincospif((float)(2.0 * (frac - 0.25 * quarter)), &s, &c);
            const float cc = (qn & 1) ? -s : c, ss = (qn & 1) ? c : s;  // one quarter turn: (cos, sin) -> (-sin, cos)
            s_cos[tok][f] = ((qn & 2) ? -cc : cc) * a.mscale;
            s_sin[tok][f] = ((qn & 2) ? -ss : ss) * a.mscale;
        }
    }
    __syncthreads();
    while (i < total) {
        finish(m, wa, wb);
        i += THREADS;
        if (i < total) {
            m = item(i);
            load(m, wa, wb);
        }
    }
}

template <class T, int V, bool INTER>
int launch_tok(RopeArgs& a, cudaStream_t s) {
    a.items = (a.heads + 2 * a.kv_heads) * (a.dim / (2 * V));
    a.by_items.set(a.items);
    a.by_head.set(a.dim / (2 * V));
    if (a.tokens >= 4 * sm_count())
        return launch_pdl(rope_kernel<T, V, INTER, 4>, dim3((a.tokens + 3) / 4), THREADS, 0, s, "rope_kernel", a);
    return launch_pdl(rope_kernel<T, V, INTER, 1>, dim3(a.tokens), THREADS, 0, s, "rope_kernel", a);
}

template <class T>
int launch(RopeArgs& a, bool wide, bool inter, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    if (wide) return inter ? launch_tok<T, V, true>(a, s) : launch_tok<T, V, false>(a, s);
    return inter ? launch_tok<T, 1, true>(a, s) : launch_tok<T, 1, false>(a, s);
}

int run(RopeArgs& a, int dtype, int inter, void* stream, const char* what) {
    if (a.dim <= 0 || a.dim % 2 || a.pairs < 0 || 2 * a.pairs > a.dim || a.pairs > MAX_PAIRS)
        return fail(B2_ERR_UNSUPPORTED, "%s: head dim %d with %d rotated pairs (dim even, 2 * pairs <= dim, pairs <= %d)", what,
                    a.dim, a.pairs, MAX_PAIRS);
    if (a.pairs && !a.inv_freq) return fail(B2_ERR_INVALID, "%s: null inv_freq", what);
    if (dtype < B2_F16 || dtype > B2_F32) return fail(B2_ERR_UNSUPPORTED, "%s: dtype code %d", what, dtype);
    const int size = dtype == B2_F32 ? 4 : 2;
    const int vec = 16 / size;
    // 16-byte items need every row and both halves of a pair on 16 bytes; any other shape goes value by value.
    bool wide = a.pairs % vec == 0 && a.dim % (2 * vec) == 0;
    if (a.heads) wide = wide && aligned16(a.x) && aligned16(a.out) && (a.sxt | a.sxh | a.sot | a.soh) % vec == 0;
    if (a.kv_heads)
        wide = wide && aligned16(a.k) && aligned16(a.v) && aligned16(a.k_cache) && aligned16(a.v_cache) &&
               (a.skt | a.skh | a.svt | a.svh | a.sc_page | a.sc_row | a.sc_head) % vec == 0;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == B2_F16) return launch<__half>(a, wide, inter != 0, s);
    if (dtype == B2_BF16) return launch<__nv_bfloat16>(a, wide, inter != 0, s);
    return launch<float>(a, wide, inter != 0, s);
}

}  // namespace

unsigned int read_status_rope() {
    unsigned int v = 0, zero = 0;
    cudaMemcpyFromSymbol(&v, g_status, sizeof(v));
    if (v) cudaMemcpyToSymbol(g_status, &zero, sizeof(zero));
    return v;
}

}  // namespace b2

using namespace b2;

extern "C" int b2_rope(const b2_rope_args* p, void* stream) {
    if (!p) return fail(B2_ERR_INVALID, "rope: null arguments");
    if (p->tokens < 0 || p->heads < 0) return fail(B2_ERR_INVALID, "rope: bad shape tokens=%d heads=%d", p->tokens, p->heads);
    if (p->tokens == 0 || p->heads == 0) return B2_OK;
    if (!p->x || !p->out || !p->positions) return fail(B2_ERR_INVALID, "rope: null pointer");
    RopeArgs a{};
    a.x = p->x;
    a.out = p->out;
    a.sxt = p->sxt;
    a.sxh = p->sxh;
    a.sot = p->sot;
    a.soh = p->soh;
    a.heads = p->heads;
    a.positions = p->positions;
    a.inv_freq = p->inv_freq;
    a.mscale = p->mscale;
    a.tokens = p->tokens;
    a.dim = p->dim;
    a.pairs = p->pairs;
    return run(a, p->dtype, p->interleaved, stream, "rope");
}

extern "C" int b2_kv_append(const b2_kv_append_args* p, void* stream) {
    if (!p) return fail(B2_ERR_INVALID, "kv_append: null arguments");
    if (p->tokens < 0 || p->heads < 0 || p->kv_heads <= 0 || p->batch < 0 || p->max_pages < 0 || p->num_pages < 0 ||
        p->page_size <= 0 || p->table_ld < 0)
        return fail(B2_ERR_INVALID, "kv_append: bad shape tokens=%d heads=%d kv_heads=%d batch=%d pages %d of %d, page size %d",
                    p->tokens, p->heads, p->kv_heads, p->batch, p->max_pages, p->num_pages, p->page_size);
    if (p->tokens == 0 || p->batch == 0) return B2_OK;
    if (!p->k || !p->v || !p->k_cache || !p->v_cache || !p->table || !p->cu_q || !p->lengths ||
        (p->heads && (!p->q || !p->q_out)))
        return fail(B2_ERR_INVALID, "kv_append: null pointer");
    RopeArgs a{};
    a.x = p->q;
    a.out = p->q_out;
    a.sxt = p->sqt;
    a.sxh = p->sqh;
    a.sot = p->sot;
    a.soh = p->soh;
    a.heads = p->heads;
    a.k = p->k;
    a.v = p->v;
    a.k_cache = p->k_cache;
    a.v_cache = p->v_cache;
    a.skt = p->skt;
    a.skh = p->skh;
    a.svt = p->svt;
    a.svh = p->svh;
    a.sc_page = p->s_page;
    a.sc_row = p->s_row;
    a.sc_head = p->s_head;
    a.kv_heads = p->kv_heads;
    a.table = p->table;
    a.table_ld = p->table_ld;
    a.max_pages = p->max_pages;
    a.num_pages = p->num_pages;
    a.page_size = p->page_size;
    a.cu_q = p->cu_q;
    a.lengths = p->lengths;
    a.batch = p->batch;
    a.positions = p->positions;
    a.inv_freq = p->inv_freq;
    a.mscale = p->mscale;
    a.tokens = p->tokens;
    a.dim = p->dim;
    a.pairs = p->pairs;
    return run(a, p->dtype, p->interleaved, stream, "kv_append");
}
