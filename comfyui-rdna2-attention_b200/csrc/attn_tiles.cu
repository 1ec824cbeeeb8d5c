// Ragged attention for many rows per kv head (chunks of prompts, packed documents): 256 rows per item on tcgen05.
//
// With 256 rows an item does 1024 D flops per key against 4 D bytes of keys and values, 256 per byte: just where the tensor
// cores become the bound (1654 TFLOP/s over 6.55 TB/s are 252), and well inside it as the other row tiles find the same
// keys in L2. Two pipelines A and B work in ping-pong: while the softmax warps of one work on its scores, the tensor core
// works for the other (S, P and O in TMEM, P written back over the consumed scores as the A operand of the second product).
// An item of more than 128 rows puts its first 128 on A and the others on B, each over the units that its own rows see. An
// item of up to 128 rows (short chunks, drafts being checked) puts its even units on A and the odd ones on B, and the two
// results are joined at the end.
//
// One CTA per SM walks its run of units (attn_ragged.cuh); every barrier's phase counts on across the items.
//   warps 0..3, 4..7  softmax of A and B: thread -> row, its 128 scores of a unit in registers
//   warp 8            TMA of keys and values (boxes of whole page parts) and queries
//   warps 8..10       instead, the rows gathered by cp.async where no box fits (odd page sizes, odd groups for queries)
//   warp 11           issues the products
//   warps 12..15      epilogue: O out of TMEM while the softmax warps are at the next item
// Rows of V behind a sequence's last key are zero in shared memory, so nothing stale is multiplied; rows of an item behind
// its last one and keys behind the end have no say in the warps' votes: the values that stand beside a sequence move no bit.
//
// Measured (32 query heads over 8 kv heads of 128, bf16): 2048 tokens over 65 000 keys 1.94 ms, 1106 TFLOP/s, 0.67 of the
// measured bf16 rate (2.3 ms where the power cap holds the clock near 1.4 GHz); 12 packed documents of 50 to 4000 tokens
// 572 us, 798 TFLOP/s (626 us where calls follow without a pause). A unit of the long chunk takes about 3300 cycles, its four
// products 2048, a pipeline's softmax 1950.
#include "attn_ragged.cuh"

namespace b2 {
namespace {

__device__ unsigned int g_status;

constexpr int TQ = 128, ROWS = 2 * TQ, UNIT = 128;
constexpr int LOADERS = 3, LOAD_WARP = 8, MMA_WARP = 11, EPI_WARP = 12;
constexpr int THREADS = 512;
constexpr int LIST = 48;  // items described in shared memory at a time
// Registers: 128 a thread at launch; 128 x (2 x 176 (softmax) + 80 (loads, products) + 80 (epilogue)) = 512 x 128, the
// split at which no role spills (200 / 56 / 56: packed documents 653 us against 577).
constexpr int REGS_SOFTMAX = 176, REGS_LOAD = 80, REGS_EPI = 80;

struct Item {
    int q0, n, len, pos0, prefix, b, kvh, rt, unit, end, slot;  // slot -1: the item is whole
    int ub[2], ue[2];  // units of A and B, counted from `unit` (two tiles: every one; one tile: every second one)
    int two;
    int64_t key0;
};

template <int D>
struct Cfg {
    static constexpr int TILE = 128 * D * 2;  // bytes of 128 rows (q, k or v)
    static constexpr int OFF_Q = 0;
    static constexpr int OFF_K = OFF_Q + 2 * TILE;
    static constexpr int OFF_V = OFF_K + 2 * TILE;
    static constexpr int OFF_ML = OFF_V + 2 * TILE;  // (m, l) of the rows of A and B
    static constexpr int OFF_LIST = OFF_ML + 2 * TQ * 8;
    static constexpr int OFF_RUN = OFF_LIST + LIST * (int)sizeof(Item);
    static constexpr int OFF_CUR = OFF_RUN + 40 * 8;
    static constexpr int OFF_BAR = (OFF_CUR + (int)sizeof(Cursor) + 15) / 16 * 16;
    static constexpr int SMEM = OFF_BAR + 256 + 1024;
};

template <int N>
__device__ __forceinline__ uint64_t get2(const uint32_t (&v)[N], int e) {
    return pk2(__uint_as_float(v[e]), __uint_as_float(v[e + 1]));
}
template <int N>
__device__ __forceinline__ void put2(uint32_t (&v)[N], int e, uint64_t x) {
    const float2 f = upk2(x);
    v[e] = __float_as_uint(f.x);
    v[e + 1] = __float_as_uint(f.y);
}

// A loading warp's copies in flight: up to three groups, each with the barrier it completes.
struct Pending {
    uint64_t* bar[3];
    int n = 0;
    __device__ __forceinline__ void pop() {
        // The copies have landed; make them visible to the tensor core before the arrival.
        fence_proxy_async_smem();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(bar[0]);
        bar[0] = bar[1];
        bar[1] = bar[2];
        --n;
    }
    __device__ __forceinline__ void drain(int keep) {
        if (n == 3 && keep < 3) {
            asm volatile("cp.async.wait_group 2;" ::: "memory");
            pop();
        }
        if (n == 2 && keep < 2) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            pop();
        }
        if (n == 1 && keep < 1) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            pop();
        }
    }
    __device__ __forceinline__ void push(uint64_t* b) {
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (n == 0) bar[0] = b;
        if (n == 1) bar[1] = b;
        if (n == 2) bar[2] = b;
        ++n;
        drain(2);
    }
};

// The CTA's next items into the list (one warp); returns their number, negative for the last list. An item of the
// cursor's sequence per lane, cut where the run ends.
__device__ __forceinline__ int fill_list(const RaggedArgs& a, Cursor* s_cur, Item* list) {
    Cursor cur = *s_cur;
    const int lane = threadIdx.x & 31;
    int n = 0;
    while (cur.left > 0 && n < LIST) {
        const int tiles = row_tiles<ROWS>(a, cur.s);
        const int f = cur.kvh * tiles + cur.rt + lane;  // items of the sequence: row tiles of kv head 0, of 1, ...
        const int kvh = tiles == 1 ? f : f / tiles, rt = f - kvh * tiles;
        const bool live = f < tiles * a.kv_heads;
        const int2 u = live ? item_units<ROWS, UNIT>(a, cur.s, rt) : make_int2(0, 0);
        const int start = lane == 0 ? cur.unit : u.x;
        int inc = u.y - start;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        const int64_t room = cur.left - (inc - (u.y - start));  // units of the run left for the lane's item
        const bool take = live && room > 0 && n + lane < LIST;
        const int end = (int)min((int64_t)u.y, start + room);
        if (take) {
            Item& it = list[n + lane];
            it.q0 = cur.s.q0;
            it.n = cur.s.n;
            it.len = cur.s.len;
            it.pos0 = cur.s.pos0;
            it.prefix = cur.s.prefix;
            it.key0 = cur.s.key0;
            it.b = cur.b;
            it.kvh = kvh;
            it.rt = rt;
            it.unit = start;
            it.end = end;
            it.slot = start == u.x && end == u.y ? -1 : 2 * (int)blockIdx.x + (start == u.x ? 1 : 0);
            it.two = cur.s.n * a.group - rt * ROWS > TQ;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                int2 w = it.two ? item_units<TQ, UNIT>(a, cur.s, 2 * rt + t) : make_int2(start, end);
                it.ub[t] = it.two ? min(max(w.x, start), end) - start : min(t, end - start);
                it.ue[t] = max(min(w.y, end) - start, it.ub[t]);
            }
            if (start == u.x && end < u.y) {
                cur.unit = start;  // for this lane's descriptor only
                cur.u1 = u.y;
                a.desc[blockIdx.x] = describe<ROWS>(a, cur.s, parts_after(cur, end), kvh, rt);
            }
        }
        const int taken = __popc(__ballot_sync(0xffffffffu, take));
        if (taken == 0) {  // not reached: units are left
            cur.left = 0;
            break;
        }
        const int used = __shfl_sync(0xffffffffu, inc, taken - 1);
        cur.left = cur.left > used ? cur.left - used : 0;
        n += taken;
        // On to the item after the last one taken.
        const int next = __shfl_sync(0xffffffffu, f, 0) + taken;
        cur.kvh = next / tiles;
        cur.rt = next - cur.kvh * tiles;
        if (cur.left > 0) {
            if (cur.kvh >= a.kv_heads) {
                cur.kvh = cur.rt = 0;
                do {
                    if (++cur.b >= a.batch) {  // not reached: units are left
                        cur.left = 0;
                        break;
                    }
                    cur.s = load_sequence(a, cur.b);
                } while (cur.s.n == 0);
            }
            if (cur.left > 0) cur.unit = item_units<ROWS, UNIT>(a, cur.s, cur.rt).x;
        }
    }
    __syncwarp();
    if (lane == 0) *s_cur = cur;
    return cur.left > 0 ? n : -n;
}

// Which of 32 keys from key0 on a row sees, its keys being [lo, hi).
__device__ __forceinline__ uint32_t seen_bits(int lo, int hi, int key0) {
    const int l = lo - key0, h = hi - key0;
    const uint32_t below = h >= 32 ? ~0u : h <= 0 ? 0u : (1u << h) - 1u;
    const uint32_t from = l <= 0 ? ~0u : l >= 32 ? 0u : ~0u << l;
    return below & from;
}

template <class T, int D, int MODE, bool TMA>
__global__ void __launch_bounds__(THREADS, 1)
    attn_tiles_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ RaggedArgs a) {
    using C = Cfg<D>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    uint64_t* q_full = bars + 0;   // one TMA phase, or 8 arrivals (row blocks of 32)
    uint64_t* q_empty = bars + 1;
    uint64_t* k_full = bars + 2;   // [2]: one TMA phase, or 4 arrivals (row blocks of 32)
    uint64_t* v_full = bars + 4;   // [2]
    uint64_t* k_empty = bars + 6;  // [2]
    uint64_t* v_empty = bars + 8;  // [2]
    uint64_t* s_full = bars + 10;  // [2] tiles
    uint64_t* p_half = bars + 12;  // [2] keys 0..63 of P
    uint64_t* p_full = bars + 14;  // [2]
    uint64_t* o_done = bars + 16;  // [2]
    uint64_t* o_free = bars + 18;  // [2]
    uint64_t* ml_full = bars + 20; // [2]
    uint64_t* drain = bars + 22;
    uint64_t* v_tail = bars + 23;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* list_len = abort_flag + 1;  // items in the list; negative: the last list
    Item* list = reinterpret_cast<Item*>(smem + C::OFF_LIST);
    float2* ml = reinterpret_cast<float2*>(smem + C::OFF_ML);

    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(q_full, a.q_tma ? 1 : 8);
        mbar_init(q_empty, 1);
        mbar_init(drain, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], TMA ? 1 : 4);
            mbar_init(&v_full[i], TMA ? 1 : 4);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_half[i], 4);  // one arrival per softmax warp of the tile
            mbar_init(&p_full[i], 4);
            mbar_init(&o_done[i], 1);
            mbar_init(&o_free[i], 4);  // one per epilogue warp
            mbar_init(&ml_full[i], 4);
        }
        mbar_init(v_tail, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == MMA_WARP) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    pdl_wait();
    // Warp LOAD_WARP lists the CTA's next items; the cursor waits in shared memory meanwhile (it would cost every role's
    // threads twenty registers).
    Cursor* s_cur = reinterpret_cast<Cursor*>(smem + C::OFF_CUR);
    {
        const Cursor found = find_run<ROWS, UNIT, THREADS>(a, reinterpret_cast<int64_t*>(smem + C::OFF_RUN), &g_status);
        if (threadIdx.x == 0) {
            *s_cur = found;
            a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
        }
    }
    __syncthreads();
    if (warp == LOAD_WARP) {
        const int n = fill_list(a, s_cur, list);
        if (lane == 0) *list_len = n;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    unsigned char* sQ = smem + C::OFF_Q;
    unsigned char* sK = smem + C::OFF_K;
    unsigned char* sV = smem + C::OFF_V;

    // Every role walks the list, then meets the others where warp LOAD_WARP writes the next one (false: there is none, or
    // a wait ran out). Phase counters run on across items and lists.
    auto next_list = [&](int count, bool writer) -> bool {
        if (count <= 0) return false;
        __syncthreads();
        if (writer && warp == LOAD_WARP) {
            const int n = fill_list(a, s_cur, list);
            if (lane == 0) *list_len = n;
        }
        __syncthreads();
        return !*abort_flag;
    };

    // Each role's code stands in the branch of its own register budget: behind a join the smaller one would hold.
    if (warp >= LOAD_WARP && warp < EPI_WARP) {
        regs_dec<REGS_LOAD>();
        if (warp < LOAD_WARP + LOADERS) {
            // With TMA warp 8 loads keys and values (and the queries, if a box can hold them); else all share all rows.
            constexpr uint32_t Q_LOADERS = TMA ? LOADERS - 1 : LOADERS;
            const uint32_t loader = warp - LOAD_WARP - (TMA ? 1 : 0);
            const bool tma_warp = TMA && warp == LOAD_WARP;
            uint32_t tails = 0, k_issued = 0, v_issued = 0, q_issued = 0;
            uint32_t items_done = 0, units_done = 0, job = 0;
            int count;
            do {
                count = *list_len;
                const int items = abs(count);
                Pending pend;
                bool ok = true;
                auto wait_free = [&](uint64_t* bar, uint32_t parity) {
                    if (mbar_try_wait(bar, parity)) return true;
                    pend.drain(0);  // what the waited-for consumer may itself be waiting for
                    return mbar_wait(bar, parity, abort_flag, &g_status, B2_DEV_TIMEOUT_PRODUCER);
                };
                // 32 rows of D values from the lanes' row offsets (negative: zeros) into rows 32 blk.. of a swizzled tile.
                auto copy_rows = [&](unsigned char* tile, int blk, const T* base, int64_t off) {
                    constexpr int CH = D / 8, PASS = 32 / CH;
                    const int ch = lane % CH;
                    const uint32_t dst = smem_u32(tile) + (ch >> 3) * (128 * 128);
#pragma unroll 8
                    for (int p = 0; p < 32 / PASS; ++p) {
                        const int r = p * PASS + lane / CH;
                        const int64_t o = __shfl_sync(0xffffffffu, off, r);
                        const int row = 32 * blk + r;
                        cp16(dst + row * 128 + (((ch & 7) ^ (row & 7)) << 4), base + (o < 0 ? 0 : o) + ch * 8, o >= 0);
                    }
                };
                for (int i = 0; i < items && ok; ++i, ++items_done) {
                    const Item& it = list[i];
                    Sequence s;
                    s.len = it.len;
                    s.key0 = it.key0;
                    s.pos0 = it.pos0;
                    const int from = item_from<ROWS>(a, s, it.rt);
                    const int units = it.end - it.unit, first = it.unit, b = it.b;
                    if (tma_warp) {
                        // Lane -> box: `rows` keys of one page, 64 of their columns.
                        const int rows = a.box_rows, boxes = UNIT / rows;
                        const int bi = lane & (boxes - 1), half = lane / boxes;
                        auto place = [&](int j) -> int2 {  // page and row in it of the lane's box of unit j
                            const int key = (first + j) * UNIT + bi * rows;
                            if (j >= units || key >= s.len) return make_int2(0, 0);
                            if (!a.table) return make_int2(0, (int)s.key0 + key);
                            // A box that the window has left behind may have no page any more.
                            if (key + rows <= from) return make_int2(a.num_pages, 0);  // outside the map: zeros
                            const int pi = a.by_page.of(key);
                            int page = a.table[(int64_t)b * a.table_ld + pi];
                            if (page < 0 || page >= a.num_pages) {
                                atomicOr(&g_status, B2_DEV_BAD_PAGE);
                                page = a.num_pages;
                            }
                            return make_int2(page, key - pi * a.page_size);
                        };
                        // Boxes past the last key are not loaded; returns the number of the unit's keys that are there.
                        auto load_unit = [&](const CUtensorMap* map, unsigned char* ring, uint64_t* full, uint64_t* empty,
                                             int j, int2 at, uint64_t* bar) -> int {
                            const uint32_t u = units_done + j;
                            const int st = u & 1;
                            const int keys = min(UNIT, s.len - (first + j) * UNIT);
                            const int live = keys <= 0 ? 0 : (keys + rows - 1) / rows;
                            if (!wait_free(&empty[st], ((u >> 1) & 1) ^ 1)) return -1;
                            uint64_t* to = bar ? bar : &full[st];
                            if (lane == 0) {
                                if (live)
                                    mbar_arrive_expect_tx(to, live * rows * (D * 2));
                                else
                                    mbar_arrive(to);
                            }
                            __syncwarp();
                            if (half < D / 64 && bi < live)
                                tma_load_4d(ring + st * C::TILE + half * (128 * 128) + bi * rows * 128, map, to, 64 * half, at.y,
                                            it.kvh, at.x);
                            return max(keys, 0);
                        };
                        int2 at = place(0);
                        ok = load_unit(&tmK, sK, k_full, k_empty, 0, at, nullptr) >= 0;
                        if (ok) ++k_issued;
                        if (ok && a.q_tma) {
                            // 128 rows are 128 / group tokens of group heads. A second tile without rows is not loaded.
                            ok = wait_free(q_empty, (items_done & 1) ^ 1);
                            const int tiles = it.two ? 2 : 1;
                            if (ok) {
                                if (lane == 0) mbar_arrive_expect_tx(q_full, tiles * C::TILE);
                                __syncwarp();
                                if (lane < tiles * (D / 64)) {
                                    const int t = lane / (D / 64), h = lane % (D / 64);
                                    tma_load_4d(sQ + t * C::TILE + h * (128 * 128), &tmQ, q_full, 64 * h, it.kvh * a.group,
                                                it.q0 + a.by_group.of(it.rt * ROWS + t * TQ), 0);
                                }
                                ++q_issued;
                            }
                        }
                        for (int j = 0; j < units && ok; ++j) {
                            const int2 next = place(j + 1);
                            if (j + 1 < units) {
                                ok = load_unit(&tmK, sK, k_full, k_empty, j + 1, next, nullptr) >= 0;
                                if (!ok) break;
                                ++k_issued;
                            }
                            const bool tail = (first + j + 1) * UNIT > s.len;
                            const int keys = load_unit(&tmV, sV, v_full, v_empty, j, at, tail ? v_tail : nullptr);
                            ok = keys >= 0;
                            if (ok && tail) {
                                // Rows behind the last key hold whatever the page or the stage held before; the product
                                // takes them times zero, so they must be finite.
                                ok = mbar_wait(v_tail, tails & 1, abort_flag, &g_status, B2_DEV_TIMEOUT_PRODUCER);
                                if (!ok && !mbar_wait_drain(v_tail, tails & 1, 100000000ull))
                                    atomicOr(&g_status, B2_DEV_TIMEOUT_DRAIN);
                                ++tails;
                                unsigned char* tile = sV + ((units_done + j) & 1) * C::TILE;
                                for (int c = keys * 8 + lane; c < UNIT * 8; c += 32)
#pragma unroll
                                    for (int h = 0; h < D / 64; ++h)
                                        *reinterpret_cast<uint4*>(tile + h * (128 * 128) + c * 16) = make_uint4(0, 0, 0, 0);
                                fence_proxy_async_smem();
                                __syncwarp();
                                if (lane == 0) mbar_arrive(&v_full[(units_done + j) & 1]);
                            }
                            if (ok) ++v_issued;
                            at = next;
                        }
                    } else if (!TMA || !a.q_tma) {
                        const T* kh = static_cast<const T*>(a.k) + it.kvh * a.s_head;
                        const T* vh = static_cast<const T*>(a.v) + it.kvh * a.s_head;
                        auto load_unit = [&](const T* base, unsigned char* ring, uint64_t* full, uint64_t* empty, int j) {
                            const uint32_t u = units_done + j;
                            const int st = u & 1;
                            bool waited = false;
                            for (int blk = 0; blk < 4; ++blk) {
                                if (job++ % Q_LOADERS != loader) continue;
                                const int64_t off = key_row_offset(a, s, b, (first + j) * UNIT + 32 * blk + lane, from, &g_status);
                                if (!waited && !wait_free(&empty[st], ((u >> 1) & 1) ^ 1)) return false;
                                waited = true;
                                copy_rows(ring + st * C::TILE, blk, base, off);
                                pend.push(&full[st]);
                            }
                            return true;
                        };
                        if (!TMA) ok = load_unit(kh, sK, k_full, k_empty, 0);
                        bool waited = false;
                        for (int blk = 0; blk < 8 && ok; ++blk) {
                            if (job++ % Q_LOADERS != loader) continue;
                            if (!waited) ok = wait_free(q_empty, (items_done & 1) ^ 1);
                            waited = true;
                            if (!ok) break;
                            // Query rows of the item: row r is token r / group, head r % group of the kv head's group.
                            const int r = it.rt * ROWS + 32 * blk + lane;
                            int64_t off = -1;
                            if (r < it.n * a.group) {
                                const int tok = a.by_group.of(r);
                                off = (int64_t)(it.q0 + tok) * a.sqt + (int64_t)(it.kvh * a.group + r - tok * a.group) * a.sqh;
                            }
                            copy_rows(sQ + (blk >> 2) * C::TILE, blk & 3, static_cast<const T*>(a.q), off);
                            pend.push(q_full);
                        }
                        for (int j = 0; !TMA && j < units && ok; ++j) {
                            if (j + 1 < units) ok = load_unit(kh, sK, k_full, k_empty, j + 1);
                            if (ok) ok = load_unit(vh, sV, v_full, v_empty, j);
                        }
                        pend.drain(0);
                    }
                    units_done += units;
                }
                if (tma_warp && !ok) {
                    // Given up: the copies in flight must land before the CTA ends.
                    if (q_issued && !mbar_wait_drain(q_full, (q_issued - 1) & 1, 100000000ull))
                        atomicOr(&g_status, B2_DEV_TIMEOUT_DRAIN);
                    for (uint32_t n = 1; n <= 2; ++n) {
                        if (k_issued >= n && !mbar_wait_drain(&k_full[(k_issued - n) & 1], ((k_issued - n) >> 1) & 1, 100000000ull))
                            atomicOr(&g_status, B2_DEV_TIMEOUT_DRAIN);
                        if (v_issued >= n && !mbar_wait_drain(&v_full[(v_issued - n) & 1], ((v_issued - n) >> 1) & 1, 100000000ull))
                            atomicOr(&g_status, B2_DEV_TIMEOUT_DRAIN);
                    }
                }
                pend.drain(0);
            } while (next_list(count, true));
        } else {
            // The products. The whole warp runs this role in step (waits by all lanes, their results voted, list entries
            // broadcast) and one elected lane issues, so that the descriptors stay in uniform registers: with a lone lane
            // in a divergent branch an issue took 70 to 100 cycles against the product's 64.
            constexpr uint32_t FMT = __is_same(T, __nv_bfloat16) ? 1 : 0;
            constexpr uint32_t idesc_qk = idesc_make(1, FMT, 0, 0, TQ, UNIT);
            constexpr uint32_t idesc_pv = idesc_make(1, FMT, 0, 1, TQ, D);
            const bool leader = elect_one();
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint64_t q_desc = sdesc_sw128(smem_u32(sQ), 16, 1024), k_desc = sdesc_sw128(smem_u32(sK), 16, 1024);
            const uint64_t v_desc = sdesc_sw128(smem_u32(sV), 128 * 128, 1024);
            uint32_t items_done = 0, units_done = 0;
            uint32_t pv_a = 0, pv_b = 0, items_a = 0, items_b = 0;  // units and items that A and B have done
            auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
                return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, &g_status, B2_DEV_TIMEOUT_MMA));
            };
            auto issue_s = [&](const int t, int q_tile, uint32_t st) {
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
                        mma_f16_ss(tm + t * UNIT, q_desc + q_tile * (C::TILE >> 4) + off, k_desc + st * (C::TILE >> 4) + off,
                                   idesc_qk, kk != 0);
                    }
                    tc_commit(&s_full[t]);
                }
            };
            // O of pipeline t += P V, for its n-th unit: the first 64 keys as soon as their P is there. At an item's first
            // unit O starts anew, once the epilogue has read the pipeline's previous item out of it.
            auto issue_pv = [&](const int t, uint32_t st, bool first, uint32_t n, uint32_t item) -> bool {
                if (!wait(&p_half[t], n & 1)) return false;
                if (first && !wait(&o_free[t], (item & 1) ^ 1)) return false;
                tc_fence_after();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h == 1) {
                        if (!wait(&p_full[t], n & 1)) return false;
                        tc_fence_after();
                    }
                    if (leader) {
#pragma unroll
                        for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
                            mma_f16_ts(tm + 256 + t * D, tm + t * UNIT + 8 * kk, v_desc + st * (C::TILE >> 4) + kk * (2048 >> 4),
                                       idesc_pv, kk == 0 ? (first ? 0u : 1u) : 1u);
                        if (h == 1) tc_commit(&o_done[t]);
                    }
                }
                return true;
            };
            int count;
            do {
                count = __shfl_sync(0xffffffffu, *list_len, 0);
                const int items = abs(count);
                bool ok = true;
                for (int i = 0; i < items && ok; ++i, ++items_done) {
                    const Item& it = list[i];
                    auto get = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
                    const int units = get(it.end - it.unit);
                    const bool two = get(it.two);
                    const int ab = get(it.ub[0]), ae = get(it.ue[0]), bb = get(it.ub[1]), be = get(it.ue[1]);
                    const uint32_t u0 = units_done;
                    auto stage = [&](int j) { return (u0 + j) & 1; };
                    auto wait_k = [&](int j) {
                        const bool there = wait(&k_full[stage(j)], ((u0 + j) >> 1) & 1);
                        tc_fence_after();
                        return there;
                    };
                    auto wait_v = [&](int j) { return wait(&v_full[stage(j)], ((u0 + j) >> 1) & 1); };
                    ok = wait(q_full, items_done & 1) && wait_k(0);
                    if (!ok) break;
                    if (two) {
                        if (ab == 0 && ae > 0) issue_s(0, 0, stage(0));
                        if (bb == 0 && be > 0) issue_s(1, 1, stage(0));
                        if (leader) {
                            tc_commit(&k_empty[stage(0)]);
                            if (units == 1) tc_commit(q_empty);
                        }
                        for (int j = 0; j < units; ++j) {
                            const bool more = j + 1 < units;
                            ok = wait_v(j);
                            if (ok && ab <= j && j < ae) ok = issue_pv(0, stage(j), j == ab, pv_a++, items_a);
                            if (ok && more) ok = wait_k(j + 1);
                            if (!ok) break;
                            if (ab <= j + 1 && j + 1 < ae) issue_s(0, 0, stage(j + 1));
                            if (bb <= j && j < be) ok = issue_pv(1, stage(j), j == bb, pv_b++, items_b);
                            if (!ok) break;
                            if (bb <= j + 1 && j + 1 < be) issue_s(1, 1, stage(j + 1));
                            if (leader) {
                                tc_commit(&v_empty[stage(j)]);
                                if (more) tc_commit(&k_empty[stage(j + 1)]);
                                if (j + 2 == units) tc_commit(q_empty);
                            }
                        }
                    } else {
                        issue_s(0, 0, stage(0));
                        if (leader) tc_commit(&k_empty[stage(0)]);
                        if (units > 1) {
                            ok = wait_k(1);
                            if (!ok) break;
                            issue_s(1, 0, stage(1));
                            if (leader) tc_commit(&k_empty[stage(1)]);
                        }
                        if (leader && units <= 2) tc_commit(q_empty);
                        // Unit j on pipeline j % 2, its next one after it.
                        auto step = [&](const int t, int j, uint32_t n, uint32_t item) -> bool {
                            if (!wait_v(j) || !issue_pv(t, stage(j), j == t, n, item)) return false;
                            if (leader) tc_commit(&v_empty[stage(j)]);
                            if (j + 2 < units) {
                                if (!wait_k(j + 2)) return false;
                                issue_s(t, 0, stage(j));
                                if (leader) {
                                    tc_commit(&k_empty[stage(j)]);
                                    if (j + 3 == units) tc_commit(q_empty);
                                }
                            }
                            return true;
                        };
                        for (int j = 0; j < units && ok; j += 2) {
                            ok = step(0, j, pv_a++, items_a);
                            if (ok && j + 1 < units) ok = step(1, j + 1, pv_b++, items_b);
                        }
                    }
                    units_done += units;
                    items_a += ae > ab;
                    items_b += be > bb;
                }
            } while (next_list(count, false));
            if (leader) {
                tc_commit(drain);
                if (!mbar_wait_drain(drain, 0, 100000000ull)) atomicOr(&g_status, B2_DEV_TIMEOUT_DRAIN);
            }
            __syncwarp();
        }
    } else if (warp >= EPI_WARP) {
        regs_dec<REGS_EPI>();
        // Epilogue: rows out of TMEM, lane quarter warp % 4 of both pipelines.
        const int row = (warp & 3) * 32 + lane;
        const uint32_t tO = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 256;
        uint32_t done[2] = {0, 0}, units_of[2] = {0, 0};  // items and units of A and B
        int count;
        do {
            count = *list_len;
            const int items = abs(count);
            bool ok = true;
            for (int i = 0; i < items && ok; ++i) {
                const Item& it = list[i];
                const int two = it.two;
                // m, l of pipeline t's part of the item; nothing seen where it has no units
                auto arrive_at = [&](int t, int c, float2& w) -> bool {
                    w = make_float2(-INFINITY, 0.f);
                    if (c == 0) return true;
                    units_of[t] += c;
                    if (!mbar_wait(&ml_full[t], done[t] & 1, abort_flag, &g_status, B2_DEV_TIMEOUT_EPILOGUE) ||
                        !mbar_wait(&o_done[t], (units_of[t] - 1) & 1, abort_flag, &g_status, B2_DEV_TIMEOUT_EPILOGUE))
                        return false;
                    w = ml[t * TQ + row];
                    ++done[t];
                    return true;
                };
                for (int p = 0; p <= two && ok; ++p) {  // two tiles: one after the other; one tile: both parts at once
                    const int rows = it.n * a.group - it.rt * ROWS - p * TQ;
                    const int ca = two ? it.ue[p] - it.ub[p] : (it.end - it.unit + 1) / 2;
                    const int cb = two ? 0 : (it.end - it.unit) / 2;
                    float2 wa, wb = make_float2(-INFINITY, 0.f);
                    ok = arrive_at(p, ca, wa) && (two || arrive_at(1, cb, wb));
                    if (!ok) break;
                    tc_fence_after();
                    const float M = fmaxf(wa.x, wb.x);
                    float fa = wa.x == -INFINITY ? 0.f : ex2_approx(wa.x - M), fb = wb.x == -INFINITY ? 0.f : ex2_approx(wb.x - M);
                    const float L = (ca ? wa.y * fa : 0.f) + (cb ? wb.y * fb : 0.f);
                    const bool live = row < rows;
                    const int r = it.rt * ROWS + p * TQ + row;
                    const int tr = a.by_group.of(r), tok = it.q0 + tr, head = it.kvh * a.group + r - tr * a.group;
                    const bool whole = it.slot < 0;
                    const int64_t srow = (int64_t)it.slot * ROWS + p * TQ + row;
                    if (whole) {
                        const float inv = L == 0.f ? 0.f : 1.f / L;
                        fa *= inv;
                        fb *= inv;
                    }
                    if (rows > (warp & 3) * 32) {  // some row of the warp's
                        T* dst = static_cast<T*>(a.out) + (int64_t)tok * a.sot + (int64_t)head * a.soh;
                        float* part = a.part_o + srow * D;
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            float x[16];
                            uint32_t o[16];
                            if (ca) tmem_ld16_wait(tO + p * D + c, o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) x[e] = ca ? __uint_as_float(o[e]) * fa : 0.f;
                            if (cb) {
                                tmem_ld16_wait(tO + D + c, o);
#pragma unroll
                                for (int e = 0; e < 16; ++e) x[e] = fmaf(__uint_as_float(o[e]), fb, x[e]);
                            }
                            if (live && whole) {
#pragma unroll
                                for (int e = 0; e < 16; e += 8)
                                    *reinterpret_cast<uint4*>(dst + c + e) =
                                        make_uint4(Pair<T>::pack(x[e], x[e + 1]), Pair<T>::pack(x[e + 2], x[e + 3]),
                                                   Pair<T>::pack(x[e + 4], x[e + 5]), Pair<T>::pack(x[e + 6], x[e + 7]));
                            } else if (live) {
#pragma unroll
                                for (int e = 0; e < 16; e += 4)
                                    *reinterpret_cast<float4*>(part + c + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                            }
                        }
                        if (live && whole && a.lse) a.lse[(int64_t)tok * a.heads + head] = log_sum(M, L);
                        if (live && !whole) a.part_ml[srow] = make_float2(M, L);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0 && ca) mbar_arrive(&o_free[p]);
                    if (lane == 0 && cb) mbar_arrive(&o_free[1]);
                }
            }
        } while (next_list(count, false));
    } else {
        regs_inc<REGS_SOFTMAX>();
        constexpr bool CAP = MODE & 1, SLOPE = MODE & 2, LARGE = MODE & 4;
        // Softmax of pipeline t = warp / 4.
        const int t = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + lane_base + t * UNIT, tO = tmem + lane_base + 256 + t * D;
        const float scale2 = a.scale * RAGGED_LOG2E;
        const float cap2 = a.softcap * RAGGED_LOG2E, cap_in = CAP ? 2.f * scale2 / a.softcap : 0.f;
        const float cap_y = CAP ? a.scale / a.softcap : 0.f;  // tanh's argument per unit of raw score
        uint32_t ucount = 0, icount = 0;
        int count;
        do {
            count = *list_len;
            const int items = abs(count);
            bool ok = true;
            for (int i = 0; i < items && ok; ++i) {
                const Item& it = list[i];
                const int two = it.two, step = two ? 1 : 2;
                const int begin = it.ub[t], stop = it.ue[t];
                if (begin >= stop) continue;
                const int rows = it.n * a.group - it.rt * ROWS - (two ? t * TQ : 0);  // valid rows of the tile
                const int first = it.unit;
                // The keys [x, y) the thread's row sees (all, where it is behind the last row), worked out again where a unit
                // is partly hidden rather than held in registers.
                auto row_keys = [&]() -> int2 {
                    if (row >= rows) return make_int2(0, 0x7fffffff);
                    const int pos = it.pos0 + a.by_group.of(it.rt * ROWS + (two ? t * TQ : 0) + row);
                    return make_int2(a.window ? max(0, pos - a.window + 1) : 0,
                                     a.causal ? min(it.len, max(pos + 1, it.prefix)) : it.len);
                };
                const float inside = row < rows ? a.softcap / a.scale : INFINITY;  // raw scores inside the cap; any for such a row
                int pos = 0;
                float slope = 0.f;
                if (SLOPE && row < rows) {
                    const int r = it.rt * ROWS + (two ? t * TQ : 0) + row;
                    const int tok = a.by_group.of(r);
                    pos = it.pos0 + tok;
                    slope = a.slopes[it.kvh * a.group + r - tok * a.group] * RAGGED_LOG2E;
                }
                const bool idle = rows <= (warp & 3) * 32;  // no row of the warp's: it only keeps the barriers' count
                const int2 keys = row_keys();
                const int lo_all = __reduce_max_sync(0xffffffffu, keys.x), hi_all = __reduce_min_sync(0xffffffffu, keys.y);
                // Keys a row may see behind its own position (their distance changes sign): first such key of the warp.
                const int ahead = SLOPE && (!a.causal || it.prefix > 0)
                                      ? __reduce_min_sync(0xffffffffu, row < rows ? pos : 0x7fffffff)
                                      : 0x7fffffff;
                // A row behind the last one holds another sequence's queries, or none, and sees keys behind the end: its maximum
                // starts where no score moves it, so that it has no say in when the warp's maxima move.
                float m = row < rows ? -INFINITY : INFINITY, l = 0.f;
                for (int j = begin; j < stop; j += step, ++ucount) {
                    if (!mbar_wait(&s_full[t], ucount & 1, abort_flag, &g_status, B2_DEV_TIMEOUT_EPILOGUE)) {
                        ok = false;
                        break;
                    }
                    if (idle) {
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(&p_half[t]);
                            mbar_arrive(&p_full[t]);
                        }
                        continue;
                    }
                    tc_fence_after();
                    const int key0 = (first + j) * UNIT;
                    const bool part = key0 < lo_all || key0 + UNIT > hi_all;
                    float mx;
                    uint32_t v[128];
                    if (MODE == 0) {
                        tmem_ld128_wait(tS, v);
                        if (part) {
                            const int2 seen_keys = row_keys();
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const uint32_t seen = seen_bits(seen_keys.x, seen_keys.y, key0 + 32 * c);
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (!(seen >> e & 1)) v[32 * c + e] = 0xff800000u;  // -inf
                            }
                        }
                        float mm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int e = 0; e < 128; e += 8)
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                mm[q] = max3(mm[q], __uint_as_float(v[e + 2 * q]), __uint_as_float(v[e + 2 * q + 1]));
                        mx = max3(mm[0], mm[1], fmaxf(mm[2], mm[3])) * scale2;  // scale2 > 0
                    } else {
                        // Cap, bias and mask, 32 scores at a time and back into TMEM as finished scores in the base-2 domain. A
                        // rolled loop: written out for 128 scores beside the exponentials below, the code was larger than
                        // the instruction cache next to the scheduler, and a unit took twice as long.
                        float mm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                        const int2 seen_keys = part ? row_keys() : make_int2(0, 0x7fffffff);
                        const int there = it.len - key0;  // keys of the unit; what stands behind them is masked below
#pragma unroll 1
                        for (int c = 0; c < 128; c += 32) {
                            uint32_t w[32];
                            tmem_ld32_wait(tS + c, w);
                            if (CAP && c < there) {
                                float am[2] = {0.f, 0.f};
#pragma unroll
                                for (int e = 0; e < 32; e += 4)
#pragma unroll
                                    for (int q = 0; q < 2; ++q)
                                        am[q] = max3(am[q], fabsf(__uint_as_float(w[e + 2 * q])),
                                                     fabsf(__uint_as_float(w[e + 2 * q + 1])));
                                // All inside the cap: the polynomial. Else exponential and reciprocal, or with a large cap
                                // each score by the form that is accurate for it. The choice moves a rounding, so where the end
                                // falls inside the chunk it is not the scores' (K cleared behind the end instead: 24 drafts over
                                // up to 9000 keys 3 % slower, as the loads wait for the last unit).
                                if (__all_sync(0xffffffffu, fmaxf(am[0], am[1]) <= (c + 32 <= there ? inside : -1.f))) {
#pragma unroll
                                    for (int e = 0; e < 32; e += 2)
                                        put2(w, e, tanh_poly(mul2(get2(w, e), splat2(cap_y)), cap2));
                                } else if (LARGE) {
#pragma unroll
                                    for (int e = 0; e < 32; e += 2)
                                        put2(w, e, capped_pair(mul2(get2(w, e), splat2(cap_y)), cap2));
                                } else {
#pragma unroll
                                    for (int e = 0; e < 32; ++e)
                                        w[e] = __float_as_uint(capped(__uint_as_float(w[e]) * cap_in, cap2));
                                }
                            }
                            if (SLOPE) {
                                const float dist = (float)(pos - key0 - c);  // of the chunk's first key
                                const uint64_t sc = splat2(CAP ? 1.f : scale2);
                                if (key0 + c + 31 <= ahead) {
                                    const uint64_t by = splat2(2.f * slope);
                                    uint64_t b2 = pk2(-slope * dist, slope * (1.f - dist));
#pragma unroll
                                    for (int e = 0; e < 32; e += 2) {
                                        put2(w, e, fma2(get2(w, e), sc, b2));
                                        b2 = add2(b2, by);
                                    }
                                } else {
#pragma unroll
                                    for (int e = 0; e < 32; ++e)
                                        w[e] = __float_as_uint(fmaf(-slope, fabsf(dist - (float)e),
                                                                    __uint_as_float(w[e]) * (CAP ? 1.f : scale2)));
                                }
                            }
                            if (part) {
                                const uint32_t seen = seen_bits(seen_keys.x, seen_keys.y, key0 + c);
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (!(seen >> e & 1)) w[e] = 0xff800000u;  // -inf
                            }
#pragma unroll
                            for (int e = 0; e < 32; e += 8)
#pragma unroll
                                for (int q = 0; q < 4; ++q)
                                    mm[q] = max3(mm[q], __uint_as_float(w[e + 2 * q]), __uint_as_float(w[e + 2 * q + 1]));
                            tmem_st32(tS + c, w);
                        }
                        mx = max3(mm[0], mm[1], fmaxf(mm[2], mm[3]));
                        tmem_wait_st();
                        tmem_ld128_wait(tS, v);
                    }
                    // The maximum moves only when a row's grew by more than 2^8: p stays below 2^8 (inside fp16) and O is
                    // rescaled rarely.
                    if (__any_sync(0xffffffffu, mx > m + 8.f)) {
                        const float mn = fmaxf(m, mx);
                        const float alpha = m == -INFINITY ? 0.f : ex2_approx(m - mn);
                        m = mn;
                        l *= alpha;
                        if (j > begin) {
                            // O holds the products of the previous units; they must be complete before the rescale.
                            if (!mbar_wait(&o_done[t], (ucount - 1) & 1, abort_flag, &g_status, B2_DEV_TIMEOUT_EPILOGUE)) {
                                ok = false;
                                break;
                            }
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D / 16; ++c) {
                                uint32_t o[16];
                                tmem_ld16_wait(tO + c * 16, o);
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                                tmem_st16(tO + c * 16, o);
                            }
                        }
                    }
                    // p = 2^(s - m); l sums the fp32 p; P, rounded to the inputs' type (half a step per key, averaged over
                    // the row), goes over the scores already read: 32 scores -> 16 columns.
                    const float nm = m == -INFINITY ? 0.f : -m;
                    const uint64_t nm2 = splat2(nm);
                    uint64_t l2 = splat2(0.f), l3 = splat2(0.f);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const uint64_t s2 = get2(v, c * 32 + 2 * e);
                            const float2 x = upk2(MODE == 0 ? fma2(s2, splat2(scale2), nm2) : add2(s2, nm2));
                            const float p0 = ex2_approx(x.x), p1 = ex2_approx(x.y);
                            if (e & 1)
                                l3 = add2(l3, pk2(p0, p1));
                            else
                                l2 = add2(l2, pk2(p0, p1));
                            pk[e] = Pair<T>::pack(p0, p1);
                        }
                        tmem_st16(tS + c * 16, pk);
                        if (c == 1) {
                            tmem_wait_st();
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&p_half[t]);
                        }
                    }
                    const float2 lf = upk2(add2(l2, l3));
                    l += lf.x + lf.y;
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[t]);
                }
                // m and l to the epilogue, once it has read the pipeline's previous item's.
                ok = ok && mbar_wait(&o_free[t], (icount & 1) ^ 1, abort_flag, &g_status, B2_DEV_TIMEOUT_EPILOGUE);
                if (!ok) break;
                ++icount;
                ml[t * TQ + row] = make_float2(m, l);
                __syncwarp();
                if (lane == 0) mbar_arrive(&ml_full[t]);
            }
        } while (next_list(count, false));
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
}

// Tensor map of the keys or values: [pages][heads][rows][D], or one page of all packed rows.
bool key_map(CUtensorMap* map, const void* base, const RaggedArgs& a, int dim, bool bf16) {
    const bool paged = a.table != nullptr;
    const uint64_t dims[4] = {(uint64_t)dim, (uint64_t)(paged ? a.page_size : a.key_rows), (uint64_t)a.kv_heads,
                              (uint64_t)(paged ? a.num_pages : 1)};
    const int64_t step[3] = {a.s_row * 2, a.s_head * 2, a.s_page * 2};
    uint64_t strides[3];
    for (int i = 0; i < 3; ++i) {
        if (dims[i + 1] == 0) return false;
        strides[i] = dims[i + 1] == 1 ? (uint64_t)dim * 2 : (uint64_t)step[i];  // a single row's stride is never used
        if (strides[i] == 0 || strides[i] >= (1ull << 40)) return false;
    }
    const uint32_t box[4] = {64, (uint32_t)a.box_rows, 1, 1};
    return make_map_4d(map, base, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, dims, strides,
                       box) == B2_OK;
}

// Tensor map of the queries, [tokens][heads][D] in boxes of 128 / group tokens of group heads.
bool query_map(CUtensorMap* map, const RaggedArgs& a, int dim, bool bf16) {
    if (TQ % a.group) return false;
    const uint64_t dims[4] = {(uint64_t)dim, (uint64_t)a.heads, (uint64_t)a.tokens, 1};
    const uint64_t strides[3] = {a.heads == 1 ? (uint64_t)dim * 2 : (uint64_t)a.sqh * 2,
                                 a.tokens == 1 ? (uint64_t)dim * 2 : (uint64_t)a.sqt * 2, (uint64_t)dim * 2};
    for (int i = 0; i < 2; ++i)
        if (strides[i] == 0 || strides[i] >= (1ull << 40)) return false;
    const uint32_t box[4] = {64, (uint32_t)a.group, (uint32_t)(TQ / a.group), 1};
    return make_map_4d(map, a.q, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, dims, strides,
                       box) == B2_OK;
}

template <class T, int D, int MODE, bool TMA>
int launch_tiles(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const RaggedArgs& a, cudaStream_t s) {
    static bool done[64] = {false};
    if (int rc = set_smem_once(attn_tiles_kernel<T, D, MODE, TMA>, Cfg<D>::SMEM, done)) return rc;
    const int ctas = sm_count();
    if (int rc = launch_pdl(attn_tiles_kernel<T, D, MODE, TMA>, dim3(ctas), THREADS, Cfg<D>::SMEM, s, "attn_tiles_kernel", tq, tk,
                            tv, a))
        return rc;
    return launch_pdl(merge_kernel<T, D, ROWS>, dim3(ctas, ROWS / 16), 512, 0, s, "merge_kernel", a);
}

}  // namespace

int64_t tiles_workspace(int dim) { return ragged_workspace(sm_count(), ROWS, dim); }

int attn_tiles(RaggedArgs& a, int dim, bool bf16, void* workspace, cudaStream_t s) {
    // 1: capped scores, 2: bias by distance, 4: a cap beyond 128, where the exponential's form of tanh is off by more than
    // 1e-4 inside the cap (capped). A variant of its own: the code for it beside the usual caps' made those 2 to 5 % slower
    // (three packed documents of 700 to 2100 tokens with a cap of 50: 128.5 us against 125.7).
    const int mode = (a.softcap > 0.f ? 1 : 0) | (a.slopes ? 2 : 0) | (a.softcap > 128.f ? 4 : 0);
    ragged_slots(a, workspace, sm_count(), ROWS, dim);
    // A TMA box is as many rows as divide both a page and a unit; below 8 rows it would cut the swizzle's pattern, and a
    // stride the map cannot hold has none: those caches are gathered by cp.async (2048 tokens over 15 000 keys, 32 heads over 8
    // of 128: pages of 64 by TMA 420 us, pages of 12 663, of 1 672). Queries of a group that does not divide 128 rows are gathered
    // too, beside keys by TMA: 24 heads over 8, 335 us.
    a.box_rows = a.table ? a.page_size & -a.page_size : UNIT;
    if (a.box_rows > UNIT) a.box_rows = UNIT;
    CUtensorMap tq{}, tk{}, tv{};
    const bool tma = a.box_rows >= 8 && key_map(&tk, a.k, a, dim, bf16) && key_map(&tv, a.v, a, dim, bf16);
    a.q_tma = tma && query_map(&tq, a, dim, bf16);
#define B2_TILES(T, D)                                                                                             \
    switch (mode) {                                                                                                \
        case 0: return tma ? launch_tiles<T, D, 0, true>(tq, tk, tv, a, s) : launch_tiles<T, D, 0, false>(tq, tk, tv, a, s); \
        case 1: return tma ? launch_tiles<T, D, 1, true>(tq, tk, tv, a, s) : launch_tiles<T, D, 1, false>(tq, tk, tv, a, s); \
        case 2: return tma ? launch_tiles<T, D, 2, true>(tq, tk, tv, a, s) : launch_tiles<T, D, 2, false>(tq, tk, tv, a, s); \
        case 3: return tma ? launch_tiles<T, D, 3, true>(tq, tk, tv, a, s) : launch_tiles<T, D, 3, false>(tq, tk, tv, a, s); \
        case 5: return tma ? launch_tiles<T, D, 5, true>(tq, tk, tv, a, s) : launch_tiles<T, D, 5, false>(tq, tk, tv, a, s); \
        default: return tma ? launch_tiles<T, D, 7, true>(tq, tk, tv, a, s) : launch_tiles<T, D, 7, false>(tq, tk, tv, a, s); \
    }
    if (dim == 128) {
        if (bf16) {
            B2_TILES(__nv_bfloat16, 128)
        }
        B2_TILES(__half, 128)
    }
    if (bf16) {
        B2_TILES(__nv_bfloat16, 64)
    }
    B2_TILES(__half, 64)
#undef B2_TILES
}

unsigned int read_status_attn_tiles() {
    unsigned int v = 0, zero = 0;
    cudaMemcpyFromSymbol(&v, g_status, sizeof(v));
    if (v) cudaMemcpyToSymbol(g_status, &zero, sizeof(zero));
    return v;
}

}  // namespace b2
