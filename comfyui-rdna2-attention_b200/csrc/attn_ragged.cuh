// What the two ragged attention kernels (attn_rows.cu, attn_tiles.cu) share: the problem, the visible keys of a row,
// and how the work is dealt to the CTAs.
//
// Sequence b has n new tokens (rows cu_q[b] .. cu_q[b + 1] of q) and len keys, the last n of them the tokens' own:
// token i sits at position pos = len - n + i. It sees the keys [lo, hi):
//   hi = len, or with the causal mask min(len, max(pos + 1, prefix[b]));   lo = max(0, pos - window + 1), or 0.
// The G = H / Hkv query heads of a kv head share its keys, so they are packed into rows: row r of (b, kv head) is token
// r / G, head r % G, and an item is ROWS consecutive rows. An item's keys are cut into units of UNIT keys (at least one
// unit, so that an item that sees nothing still writes its zeros).
//
// The lengths live on the device (a captured graph replays with other lengths), so the CTAs deal the work among
// themselves: all units, ordered by (sequence, kv head, row tile, key), are cut into gridDim.x runs of equal length,
// each CTA adds up the sequences' units and finds its run. A run holds whole items, and at its ends parts of items,
// which leave unnormalized results (O, and per row the maximum m and the sum l) in the CTA's two slots of the workspace:
// slot 2x for the part of an item that began in an earlier CTA, slot 2x + 1 for the head of an item that goes on in
// the next. merge_kernel joins each head with the parts that follow it, in CTA order, so results do not depend on timing.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"
#include "host.hpp"

namespace b2 {

constexpr float RAGGED_LOG2E = 1.4426950408889634f;

struct RaggedArgs {
    const void* q;
    int64_t sqt, sqh;
    void* out;
    int64_t sot, soh;
    float* lse;  // [tokens, heads], may be null
    const void *k, *v;
    int64_t s_page, s_row, s_head;  // packed keys: s_page unused
    const int32_t* table;           // null: packed keys
    int table_ld, max_pages, num_pages, page_size;
    const int32_t* cu_q;
    const int32_t* lengths;  // paged: keys per sequence; packed: cu_k
    const int32_t* prefix;   // null: none
    const float* slopes;     // null: none
    int batch, tokens, key_rows, heads, kv_heads, group;
    int causal, window;
    float scale, softcap;
    float cap_y;  // scale / softcap: tanh's argument per unit of q.k
    Divisor by_group, by_page;
    int box_rows;  // attn_tiles.cu: rows of a TMA box of keys
    int q_tma;     // and whether the queries come by TMA
    // workspace: partial O [slots][ROWS][D], (m, l) [slots][ROWS], item descriptor [CTAs][4]
    float* part_o;
    float2* part_ml;
    int4* desc;
};

struct Sequence {
    int q0, n, len, pos0, prefix;
    int64_t key0;  // packed keys: first row
};

__device__ __forceinline__ Sequence load_sequence(const RaggedArgs& a, int b) {
    Sequence s;
    s.q0 = min(max(a.cu_q[b], 0), a.tokens);
    s.n = max(min(a.cu_q[b + 1], a.tokens) - s.q0, 0);
    s.key0 = 0;
    if (a.table) {
        s.len = min(max(a.lengths[b], 0), 1 << 30);  // so that positions and units keep to 32 bits
        s.len = (int)min((int64_t)s.len, (int64_t)a.max_pages * a.page_size);  // no key lies behind the table
    } else {
        const int k0 = min(max(a.lengths[b], 0), a.key_rows);
        s.len = max(min(a.lengths[b + 1], a.key_rows) - k0, 0);
        s.key0 = k0;
    }
    s.pos0 = s.len - s.n;
    s.prefix = a.prefix ? min(max(a.prefix[b], 0), s.len) : 0;
    return s;
}

__device__ __forceinline__ int key_hi(const RaggedArgs& a, const Sequence& s, int tok) {
    return a.causal ? min(s.len, max(s.pos0 + tok + 1, s.prefix)) : s.len;
}
__device__ __forceinline__ int key_lo(const RaggedArgs& a, const Sequence& s, int tok) {
    return a.window ? max(0, s.pos0 + tok - a.window + 1) : 0;
}

// The first key that any row of row tile rt sees: its first row's.
template <int ROWS>
__device__ __forceinline__ int item_from(const RaggedArgs& a, const Sequence& s, int rt) {
    return key_lo(a, s, a.by_group.of(rt * ROWS));
}
// The units [u0, u1) of the keys that any row of row tile rt sees.
template <int ROWS, int UNIT>
__device__ __forceinline__ int2 item_units(const RaggedArgs& a, const Sequence& s, int rt) {
    const int tok1 = min(s.n - 1, a.by_group.of(rt * ROWS + ROWS - 1));
    const int hi = key_hi(a, s, tok1), lo = item_from<ROWS>(a, s, rt);
    if (hi <= lo) return make_int2(0, 1);
    return make_int2(lo / UNIT, (hi + UNIT - 1) / UNIT);
}
template <int ROWS>
__device__ __forceinline__ int row_tiles(const RaggedArgs& a, const Sequence& s) {
    return (s.n * a.group + ROWS - 1) / ROWS;
}
// Units of one kv head of each lane's sequence. A lane adds up a sequence of one or two row tiles by itself; the longer
// ones are taken one after another by the whole warp, a row tile per lane.
template <int ROWS, int UNIT>
__device__ __forceinline__ int64_t head_units(const RaggedArgs& a, const Sequence& s) {
    const int lane = threadIdx.x & 31;
    const int tiles = row_tiles<ROWS>(a, s);
    int64_t c = 0;
    if (tiles <= 2)
        for (int rt = 0; rt < tiles; ++rt) {
            const int2 u = item_units<ROWS, UNIT>(a, s, rt);
            c += u.y - u.x;
        }
    for (unsigned todo = __ballot_sync(0xffffffffu, tiles > 2); todo; todo &= todo - 1) {
        const int src = __ffs(todo) - 1;
        Sequence o{};
        o.n = __shfl_sync(0xffffffffu, s.n, src);
        o.len = __shfl_sync(0xffffffffu, s.len, src);
        o.pos0 = __shfl_sync(0xffffffffu, s.pos0, src);
        o.prefix = __shfl_sync(0xffffffffu, s.prefix, src);
        const int many = row_tiles<ROWS>(a, o);
        int64_t sum = 0;
        for (int rt = lane; rt < many; rt += 32) {
            const int2 u = item_units<ROWS, UNIT>(a, o, rt);
            sum += u.y - u.x;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == src) c = sum;
    }
    return c;
}

// The runs: run x is [begin(x), begin(x + 1)) of all units.
struct Runs {
    int64_t each;  // units of a run; the first `more` runs have one more
    int more, count;
    __device__ __forceinline__ int64_t begin(int x) const { return each * x + min(x, more); }
};

// A CTA's place in the work: item (b, kvh, rt) with units [u0, u1), the next one to do and how many are left in its run.
struct Cursor {
    Sequence s;
    int b, kvh, rt, u0, u1, unit;
    int64_t left;
    Runs runs;
};

// Finds the CTA's run with all of its threads (THREADS of them; smem: 40 int64). Every thread returns the same cursor.
template <int ROWS, int UNIT, int THREADS>
__device__ __forceinline__ Cursor find_run(const RaggedArgs& a, int64_t* smem, unsigned int* status) {
    constexpr int WARPS = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // A sequence longer than its row of the table is cut there, and reported.
    if (a.table && blockIdx.x == 0)
        for (int b = tid; b < a.batch; b += THREADS)
            if (a.lengths[b] > (int64_t)a.max_pages * a.page_size) atomicOr(status, B2_DEV_BAD_PAGE);
    auto units_of = [&](int b) -> int64_t {  // every lane of the warp calls it
        return head_units<ROWS, UNIT>(a, b < a.batch ? load_sequence(a, b) : Sequence{}) * a.kv_heads;
    };
    // Total, and each thread's count for the first THREADS sequences.
    const int64_t first = units_of(tid);
    int64_t sum = first;
    for (int b = THREADS; b < a.batch; b += THREADS) sum += units_of(b + tid);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) smem[warp] = sum;
    if (tid == 0) smem[34] = -1;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += smem[w];
    Cursor c;
    // Fewer units than CTAs: one each, the other CTAs have none.
    c.runs.count = (int)min((int64_t)gridDim.x, total);
    c.left = 0;
    c.b = c.kvh = c.rt = c.u0 = c.u1 = c.unit = 0;
    c.s = Sequence{};
    __syncthreads();
    if ((int)blockIdx.x >= c.runs.count) return c;
    if (total < (1ll << 32)) {
        c.runs.each = (uint32_t)total / (uint32_t)c.runs.count;
        c.runs.more = (uint32_t)total % (uint32_t)c.runs.count;
    } else {
        c.runs.each = total / c.runs.count;
        c.runs.more = (int)(total % c.runs.count);
    }
    const int64_t begin = c.runs.begin(blockIdx.x);
    c.left = c.runs.begin(blockIdx.x + 1) - begin;
    // The sequence that holds unit `begin`: prefix sums over THREADS sequences at a time.
    int64_t before = 0;
    for (int base = 0;; base += THREADS) {
        const int64_t mine = base == 0 ? first : units_of(base + tid);
        int64_t inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        if (lane == 31) smem[warp] = inc;
        __syncthreads();
        int64_t off = before;
        for (int w = 0; w < warp; ++w) off += smem[w];
        const int64_t lo = off + inc - mine;
        if (mine > 0 && lo <= begin && begin < lo + mine) {
            smem[34] = base + tid;
            smem[35] = begin - lo;
            smem[36] = mine;
        }
        for (int w = 0; w < WARPS; ++w) before += smem[w];
        __syncthreads();
        if (smem[34] >= 0 || base + THREADS >= a.batch) break;
    }
    c.b = (int)smem[34];
    int64_t rem = smem[35];
    if (c.b < 0) {  // not reached: begin < total
        c.left = 0;
        c.b = 0;
        return c;
    }
    c.s = load_sequence(a, c.b);
    const int64_t per_head = smem[36] < (1ll << 32) ? (uint32_t)smem[36] / (uint32_t)a.kv_heads : smem[36] / a.kv_heads;
    while (rem >= per_head) {
        rem -= per_head;
        ++c.kvh;
    }
    // The row tile: a tile per lane, prefix sums.
    for (int rt0 = 0;; rt0 += 32) {
        const int rt = rt0 + lane;
        const int2 u = rt < row_tiles<ROWS>(a, c.s) ? item_units<ROWS, UNIT>(a, c.s, rt) : make_int2(0, 0);
        int inc = u.y - u.x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, inc > rem);
        if (past) {
            const int src = __ffs(past) - 1;
            c.rt = rt0 + src;
            c.u0 = __shfl_sync(0xffffffffu, u.x, src);
            c.u1 = __shfl_sync(0xffffffffu, u.y, src);
            c.unit = c.u0 + (int)rem - __shfl_sync(0xffffffffu, inc, src) + c.u1 - c.u0;
            break;
        }
        rem -= __shfl_sync(0xffffffffu, inc, 31);
        if (rt0 + 32 >= row_tiles<ROWS>(a, c.s)) {  // not reached: rem < per_head
            c.left = 0;
            break;
        }
    }
    return c;
}

// Moves on by `done` units, to the next item where the current one is finished.
template <int ROWS, int UNIT>
__device__ __forceinline__ void advance(const RaggedArgs& a, Cursor& c, int done) {
    c.unit += done;
    c.left -= done;
    if (c.unit < c.u1 || c.left <= 0) return;
    if (++c.rt >= row_tiles<ROWS>(a, c.s)) {
        c.rt = 0;
        if (++c.kvh >= a.kv_heads) {
            c.kvh = 0;
            do {
                if (c.b + 1 >= a.batch) {  // not reached: units are left
                    c.left = 0;
                    return;
                }
                c.s = load_sequence(a, ++c.b);
            } while (c.s.n == 0);
        }
    }
    const int2 u = item_units<ROWS, UNIT>(a, c.s, c.rt);
    c.u0 = c.unit = u.x;
    c.u1 = u.y;
}

// How many of the next CTAs hold the rest of an item that this CTA's run ends inside (`end`: where this run stops in the
// item), 0 where it does not.
__device__ __forceinline__ int parts_after(const Cursor& c, int end) {
    if (end >= c.u1) return 0;
    const int64_t stop = c.runs.begin(blockIdx.x + 1) + (c.u1 - end);
    int n = 1;
    while (blockIdx.x + 1 + n < c.runs.count && c.runs.begin(blockIdx.x + 1 + n) < stop) ++n;
    return n;
}

// What the merge reads of an item whose head this CTA holds: parts after the head (below 2^16, as the CTAs are) and rows,
// q0, kv head, first row.
template <int ROWS>
__device__ __forceinline__ int4 describe(const RaggedArgs& a, const Sequence& s, int parts, int kvh, int rt) {
    return make_int4(parts | min(ROWS, s.n * a.group - rt * ROWS) << 16, s.q0, kvh, rt * ROWS);
}

// Element offset of a key row of the sequence in k and v (head 0), or -1 for a row that counts as zeros: behind the last
// key, before the first key `from` that the item sees (a sliding window's old pages may be gone), or on a page that does
// not exist (reported in *status).
__device__ __forceinline__ int64_t key_row_offset(const RaggedArgs& a, const Sequence& s, int b, int key, int from,
                                                  unsigned int* status) {
    if (key >= s.len || key < from) return -1;
    if (!a.table) return (s.key0 + key) * a.s_row;
    const int pi = a.by_page.of(key);
    const int page = a.table[(int64_t)b * a.table_ld + pi];
    if (page < 0 || page >= a.num_pages) {
        atomicOr(status, B2_DEV_BAD_PAGE);
        return -1;
    }
    return (int64_t)page * a.s_page + (int64_t)(key - pi * a.page_size) * a.s_row;
}

// 16 bytes into shared memory, zeros where !ok (nothing is read then).
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool ok) {
    const int n = ok ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// cap * tanh(s / cap) in the base-2 domain, y = s / cap: tanh(y) = 1 - 2 / (1 + 2^(2 y log2 e)). y2 = 2 y log2(e),
// cap2 = cap log2(e); saturates to +-cap2 when the power over- or underflows. The difference leaves an error of 3e-7 cap2,
// small against the score beyond the cap (|y| > 1); inside it tanh_poly keeps the digits.
__device__ __forceinline__ float capped(float y2, float cap2) {
    return fmaf(-2.f * cap2, rcp_approx(1.f + ex2_approx(y2)), cap2);
}
// tanh(y) = y P(y^2), |y| <= 1, P of degree 5 fitted to the smallest relative error (7e-7): y P(y^2) scale on a pair.
__device__ __forceinline__ uint64_t tanh_poly(uint64_t y, float scale) {
    const uint64_t u = mul2(y, y);
    uint64_t p = fma2(splat2(-0.0030670601408928633f * scale), u, splat2(0.016743114218115807f * scale));
    p = fma2(p, u, splat2(-0.051605671644210815f * scale));
    p = fma2(p, u, splat2(0.13281433284282684f * scale));
    p = fma2(p, u, splat2(-0.3332904279232025f * scale));
    p = fma2(p, u, splat2(0.9999994039535522f * scale));
    return mul2(y, p);
}
// Each of a pair by the form that is accurate for it, so that the relative error stays below 2^-20 whatever the cap is.
__device__ __forceinline__ uint64_t capped_pair(uint64_t y, float cap2) {
    const float2 f = upk2(y), p = upk2(tanh_poly(y, cap2));
    return pk2(fabsf(f.x) <= 1.f ? p.x : capped(f.x * (2.f * RAGGED_LOG2E), cap2),
               fabsf(f.y) <= 1.f ? p.y : capped(f.y * (2.f * RAGGED_LOG2E), cap2));
}

// The fp32 value before x >= 0, and 0 for 0.
__device__ __forceinline__ float below(float x) { return __uint_as_float(max(__float_as_uint(x), 1u) - 1u); }

template <class T>
struct Pair;  // two 16-bit values of T from fp32, rounded to nearest even
template <>
struct Pair<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return h2_as_u32(__floats2half2_rn(a, b)); }
    // a, b >= 0 as hi + lo, both positive where the weight is: hi is cut off below the value one fp32 step smaller. (A
    // remainder of zero or less would turn an infinite value of a visible key into NaN.)
    static __device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(below(b)), "f"(below(a)));
        const float2 h = __half22float2(u32_as_h2(hi));
        lo = pack(a - h.x, b - h.y);
    }
};
template <>
struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
        const uint32_t x = __float_as_uint(below(a)), y = __float_as_uint(below(b));
        hi = __byte_perm(x, y, 0x7632);
        lo = pack(a - __uint_as_float(x & 0xffff0000u), b - __uint_as_float(y & 0xffff0000u));
    }
};

// Natural logarithm of a row's sum of exponentials from its base-2 maximum and sum; -inf where nothing was seen.
__device__ __forceinline__ float log_sum(float m2, float l) {
    return l == 0.f ? -INFINITY : (m2 + log2f(l)) * 0.69314718055994531f;
}

// Joins the parts of every item that was cut: one warp per row, blockIdx.x = the CTA that holds the item's head.
//   M = max m_p, L = sum l_p 2^(m_p - M), out = sum O_p 2^(m_p - M) / L
template <class T, int D, int ROWS>
__global__ void __launch_bounds__(512) merge_kernel(const RaggedArgs a) {
    pdl_trigger();
    pdl_wait();
    const int x = blockIdx.x, lane = threadIdx.x & 31;
    const int row = blockIdx.y * 16 + (threadIdx.x >> 5);
    const int4 d = a.desc[x];  // parts after the head and rows, q0, kvh, first row: see describe
    const int parts = (d.x & 0xffff) + 1;
    if (parts == 1 || row >= d.x >> 16) return;
    auto slot = [&](int p) { return (int64_t)(p == 0 ? 2 * x + 1 : 2 * (x + p)) * ROWS + row; };
    constexpr int C = D / 32, BATCH = 8;
    float acc[C];
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = 0.f;
    float M = -INFINITY, L = 0.f;
    for (int p0 = 0; p0 < parts; p0 += 32) {
        // 32 parts' (m, l) a lane each, and O of eight of them at a time: the loads do not wait for the weights.
        const int here = min(32, parts - p0);
        const float2 ml = lane < here ? a.part_ml[slot(p0 + lane)] : make_float2(-INFINITY, 0.f);
        float w = 0.f;
        for (int b = 0; b < here; b += BATCH) {
            float v[BATCH][C];
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                const float* src = a.part_o + slot(p0 + min(b + k, here - 1)) * D + lane * C;
                if constexpr (C == 4)
                    *reinterpret_cast<float4*>(v[k]) = *reinterpret_cast<const float4*>(src);
                else
                    *reinterpret_cast<float2*>(v[k]) = *reinterpret_cast<const float2*>(src);
            }
            if (b == 0) {
                float m = fmaxf(M, ml.x);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                const float keep = M == -INFINITY ? 0.f : ex2_approx(M - m);
                M = m;
                L *= keep;
#pragma unroll
                for (int i = 0; i < C; ++i) acc[i] *= keep;
                w = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - M);
                if (w != 0.f) L += w * ml.y;
            }
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                const float wp = __shfl_sync(0xffffffffu, w, b + k);
                if (b + k < here && wp != 0.f) {  // a part that saw nothing may hold no O
#pragma unroll
                    for (int i = 0; i < C; ++i) acc[i] = fmaf(wp, v[k][i], acc[i]);
                }
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int r = d.w + row, t = a.by_group.of(r), tok = d.y + t, head = d.z * a.group + r - t * a.group;
    T* dst = static_cast<T*>(a.out) + (int64_t)tok * a.sot + (int64_t)head * a.soh + lane * C;
    uint32_t u[C / 2];
#pragma unroll
    for (int i = 0; i < C / 2; ++i) u[i] = Pair<T>::pack(acc[2 * i] * inv, acc[2 * i + 1] * inv);
    if constexpr (C == 4)
        *reinterpret_cast<uint2*>(dst) = make_uint2(u[0], u[1]);
    else
        *reinterpret_cast<uint32_t*>(dst) = u[0];
    if (a.lse && lane == 0) a.lse[(int64_t)tok * a.heads + head] = log_sum(M, L);
}

// ---------------------------------------------------------------- host
// Workspace of a launch of `ctas` CTAs: two slots each of ROWS rows of O and (m, l), and the descriptors.
inline int64_t ragged_workspace(int ctas, int rows, int dim) {
    return (int64_t)ctas * (2 * rows * (dim * 4 + 8) + 16);
}
inline void ragged_slots(RaggedArgs& a, void* workspace, int ctas, int rows, int dim) {
    unsigned char* w = static_cast<unsigned char*>(workspace);
    a.part_o = reinterpret_cast<float*>(w);
    w += (int64_t)ctas * 2 * rows * dim * 4;
    a.part_ml = reinterpret_cast<float2*>(w);
    w += (int64_t)ctas * 2 * rows * 8;
    a.desc = reinterpret_cast<int4*>(w);
}
// The two kernels' launchers (attn_rows.cu, attn_tiles.cu).
int64_t rows_workspace(int dim);
int attn_rows(RaggedArgs& a, int dim, bool bf16, void* workspace, cudaStream_t s);
int64_t tiles_workspace(int dim);
int attn_tiles(RaggedArgs& a, int dim, bool bf16, void* workspace, cudaStream_t s);

}  // namespace b2
