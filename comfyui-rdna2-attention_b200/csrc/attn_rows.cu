// Ragged attention for few rows per kv head (tokens being decoded): 16 rows per item on mma.sync m16n8k16.
//
// With r = tokens x G rows per kv head the work is 4 D r flops per key and kv head against 4 D bytes of keys and
// values, r flops per byte: 16 at 16 rows, where the tensor cores bound from 252 on, so HBM bounds it and the legacy tensor
// path (16-row tiles, operands in registers) is enough; a tcgen05 tile would be 128 rows of which at most 16 hold anything.
//
// A CTA is four warps, each its own pipeline: warp w takes keys [64 u + 16 w, + 16) of every unit u of the run, loads
// their K and V rows with cp.async (16 bytes a lane, rows gathered through the page table; rows behind the last key
// are zero-filled, so nothing stale reaches a product) into its own ring of stages, and keeps its own maximum, sum and
// O in registers. No barrier between warps until the item's end, where the four results meet in shared memory.
//
// Measured (32 query heads over 8 kv heads of 128): 96 sequences of one token over 500 to 16000 keys, bf16, 460 us, 6.5 TB/s,
// the copy rate; one token over 1024 keys 9.5 us, the latency of the deal, the page lookup, the keys and the merge.
#include "attn_ragged.cuh"
#include "host.hpp"

namespace b2 {
namespace {

__device__ unsigned int g_status;

constexpr int ROWS = 16, UNIT = 64, WARPS = 4, THREADS = 32 * WARPS, KEYS = 16;

template <int D>
struct Cfg {
    static constexpr int STAGES = D == 128 ? 3 : 4;
    static constexpr int TILE = KEYS * D * 2;                 // bytes of one stage's K (or V) rows
    static constexpr int WARP_BYTES = STAGES * 2 * TILE;      // >= ROWS * PITCH * 4, reused for O at the item's end
    static constexpr int PITCH = D + 4;                       // floats per O row in shared memory
    static constexpr int SMEM = WARPS * WARP_BYTES;
    static constexpr int CTAS = D == 128 ? 2 : 3;             // per SM
};

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Byte offset of 16-byte chunk c of row r in a [KEYS][D] tile: chunks are permuted by the row so that the eight rows
// an ldmatrix reads sit in different banks.
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return r * (D * 2) + ((c ^ (r & 7)) << 4);
}

template <class T, int D, bool BIAS>
__global__ void __launch_bounds__(THREADS, Cfg<D>::CTAS) attn_rows_kernel(const __grid_constant__ RaggedArgs a) {
    using C = Cfg<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int64_t s_run[40];
    __shared__ float s_m[WARPS][ROWS], s_l[WARPS][ROWS];
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t ring = smem_u32(smem) + warp * C::WARP_BYTES;
    float* o_smem = reinterpret_cast<float*>(smem + warp * C::WARP_BYTES);

    Cursor c = find_run<ROWS, UNIT, THREADS>(a, s_run, &g_status);
    int4 desc = make_int4(0, 0, 0, 0);
    while (c.left > 0) {
        const int end = (int)min((int64_t)c.u1, c.unit + c.left);
        const int units = end - c.unit;
        const Sequence& s = c.s;
        const int rows = s.n * a.group - c.rt * ROWS;  // valid rows of the item (>= 1, may exceed 16)

        // Loads of the run's i-th unit into stage i % STAGES. The lane's row (of 16) is found one unit ahead.
        const T* kh = static_cast<const T*>(a.k) + c.kvh * a.s_head;
        const T* vh = static_cast<const T*>(a.v) + c.kvh * a.s_head;
        const int from = item_from<ROWS>(a, s, c.rt);
        auto row_of = [&](int i) -> int64_t {
            return i < units ? key_row_offset(a, s, c.b, (c.unit + i) * UNIT + warp * KEYS + (lane & 15), from, &g_status) : -1;
        };
        int64_t next = row_of(0);
        auto load = [&](int i) {
            const int64_t mine = next;
            next = row_of(i + 1);
            if (i < units) {
                constexpr int CH = D / 8, PASS = 32 / CH;  // chunks per row, rows per pass
                const uint32_t dst = ring + (i % C::STAGES) * 2 * C::TILE;
                const int ch = lane % CH;
#pragma unroll
                for (int p = 0; p < KEYS / PASS; ++p) {
                    const int r = p * PASS + lane / CH;
                    const int64_t off = __shfl_sync(0xffffffffu, mine, r);
                    const bool ok = off >= 0;
                    const int64_t e = (ok ? off : 0) + ch * 8;
                    cp16(dst + chunk_at<D>(r, ch), kh + e, ok);
                    cp16(dst + C::TILE + chunk_at<D>(r, ch), vh + e, ok);
                }
            }
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < C::STAGES - 1; ++i) load(i);

        // The lane's two rows (of the mma fragments): query values, visible keys, position.
        uint32_t qf[D / 16][4];
        int lo[2], hi[2], pos[2];
        float slope[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = (lane >> 2) + 8 * h;
            const bool live = row < rows;
            const int r = c.rt * ROWS + (live ? row : 0);
            const int tok = a.by_group.of(r), head = c.kvh * a.group + r - tok * a.group;
            pos[h] = s.pos0 + tok;
            lo[h] = live ? key_lo(a, s, tok) : 0;
            hi[h] = live ? key_hi(a, s, tok) : 0x7fffffff;
            slope[h] = BIAS && a.slopes && live ? a.slopes[head] * RAGGED_LOG2E : 0.f;
            const T* src = static_cast<const T*>(a.q) + (int64_t)(s.q0 + tok) * a.sqt + (int64_t)head * a.sqh + (lane & 3) * 2;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                qf[k][h] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * k) : 0;
                qf[k][2 + h] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8) : 0;
            }
        }
        // Keys that every live row sees, and that any row sees.
        const int lo_all = __reduce_max_sync(0xffffffffu, max(lo[0], lo[1]));
        const int hi_all = __reduce_min_sync(0xffffffffu, min(hi[0], hi[1]));
        const float scale2 = a.scale * RAGGED_LOG2E;
        const float cap2 = a.softcap * RAGGED_LOG2E;

        float o[D / 8][4];
#pragma unroll
        for (int t = 0; t < D / 8; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][e] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

        for (int i = 0; i < units; ++i) {
            __syncwarp();  // every lane is done with the stage that is loaded next
            load(i + C::STAGES - 1);
            cp_wait<C::STAGES - 1>();
            __syncwarp();
            const int key0 = (c.unit + i) * UNIT + warp * KEYS;
            if (key0 >= s.len) continue;
            const uint32_t kt = ring + (i % C::STAGES) * 2 * C::TILE, vt = kt + C::TILE;
            // S = Q K^T, 16 rows x 16 keys
            float sc[2][4] = {};
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                uint32_t b[4];
                ldm4(b, kt + chunk_at<D>((lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
                mma16816<T>(sc[0], qf[k], b[0], b[1]);
                mma16816<T>(sc[1], qf[k], b[2], b[3]);
            }
            // Scores in the base-2 domain: element e of n-tile t is row (lane >> 2) + 8 (e >> 1), key 8 t + 2 (lane & 3) + (e & 1).
            float x[2][4];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    float2 y = make_float2(sc[t][e] * scale2, sc[t][e + 1] * scale2);
                    if (BIAS) {
                        if (a.softcap > 0.f) y = upk2(capped_pair(mul2(pk2(sc[t][e], sc[t][e + 1]), splat2(a.cap_y)), cap2));
                        const int key = key0 + 8 * t + 2 * (lane & 3);
                        y.x = fmaf(-slope[e >> 1], (float)abs(pos[e >> 1] - key), y.x);
                        y.y = fmaf(-slope[e >> 1], (float)abs(pos[e >> 1] - key - 1), y.y);
                    }
                    x[t][e] = y.x;
                    x[t][e + 1] = y.y;
                }
            if (key0 < lo_all || key0 + KEYS > hi_all) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + 8 * t + 2 * (lane & 3) + (e & 1);
                        if (key < lo[e >> 1] || key >= hi[e >> 1]) x[t][e] = -INFINITY;
                    }
            }
            float mx[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mx[h] = fmaxf(fmaxf(x[0][2 * h], x[0][2 * h + 1]), fmaxf(x[1][2 * h], x[1][2 * h + 1]));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
            }
            // The maximum moves only when some row's grew by more than 2^8: p stays below 2^8, well inside fp16, and
            // O is rescaled rarely. A row that has seen nothing keeps m = -inf.
            if (__any_sync(0xffffffffu, mx[0] > m[0] + 8.f || mx[1] > m[1] + 8.f)) {
                float al[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float mn = fmaxf(m[h], mx[h]);
                    al[h] = m[h] == -INFINITY ? 0.f : ex2_approx(m[h] - mn);
                    m[h] = mn;
                    l[h] *= al[h];
                }
#pragma unroll
                for (int t = 0; t < D / 8; ++t) {
                    o[t][0] *= al[0];
                    o[t][1] *= al[0];
                    o[t][2] *= al[1];
                    o[t][3] *= al[1];
                }
            }
            const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[t][e] = ex2_approx(x[t][e] - ref[e >> 1]);
                    l[e >> 1] += x[t][e];
                }
            // O += P V, each weight as the sum of two values of the inputs' type (16 bits of it with bf16, 22 with fp16), so that
            // the result is off by its own rounding only: 1.7e-3 of the values in the mean square with bf16, 2.3e-3 with weights
            // of one part. The second product costs nothing beside the keys' loads at dim 128 (96 tokens over 500 to 16000 keys
            // 461 us with and without it), 5 % at dim 64 (179, 169.5).
            uint32_t p[4], r[4];
#pragma unroll
            for (int f = 0; f < 4; ++f) Pair<T>::split(x[f >> 1][2 * (f & 1)], x[f >> 1][2 * (f & 1) + 1], p[f], r[f]);
#pragma unroll
            for (int t = 0; t < D / 16; ++t) {
                uint32_t b[4];
                ldm4t(b, vt + chunk_at<D>((lane & 7) + (((lane >> 3) & 1) << 3), 2 * t + (lane >> 4)));
                mma16816<T>(o[2 * t], p, b[0], b[1]);
                mma16816<T>(o[2 * t + 1], p, b[2], b[3]);
                mma16816<T>(o[2 * t], r, b[0], b[1]);
                mma16816<T>(o[2 * t + 1], r, b[2], b[3]);
            }
        }
        cp_wait<0>();

        // The four warps' results meet.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if ((lane & 3) == 0) {
                s_m[warp][(lane >> 2) + 8 * h] = m[h];
                s_l[warp][(lane >> 2) + 8 * h] = l[h];
            }
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = (lane >> 2) + 8 * h;
            float M = s_m[0][row];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) M = fmaxf(M, s_m[w][row]);
            const float f = m[h] == -INFINITY ? 0.f : ex2_approx(m[h] - M);
#pragma unroll
            for (int t = 0; t < D / 8; ++t)
                *reinterpret_cast<float2*>(o_smem + row * C::PITCH + 8 * t + 2 * (lane & 3)) =
                    make_float2(o[t][2 * h] * f, o[t][2 * h + 1] * f);
        }
        __syncthreads();
        const bool whole = c.unit == c.u0 && end == c.u1;
        const int slot = 2 * blockIdx.x + (c.unit == c.u0 ? 1 : 0);
        for (int i = threadIdx.x; i < ROWS * (D / 8); i += THREADS) {
            const int row = i / (D / 8), col = i % (D / 8) * 8;
            if (row >= rows) break;
            float v[8] = {};
            float M = s_m[0][row], L = 0.f;
#pragma unroll
            for (int w = 1; w < WARPS; ++w) M = fmaxf(M, s_m[w][row]);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float* src = reinterpret_cast<const float*>(smem + w * C::WARP_BYTES) + row * C::PITCH + col;
                const float4 lo4 = *reinterpret_cast<const float4*>(src), hi4 = *reinterpret_cast<const float4*>(src + 4);
                v[0] += lo4.x;
                v[1] += lo4.y;
                v[2] += lo4.z;
                v[3] += lo4.w;
                v[4] += hi4.x;
                v[5] += hi4.y;
                v[6] += hi4.z;
                v[7] += hi4.w;
                if (s_m[w][row] != -INFINITY) L += s_l[w][row] * ex2_approx(s_m[w][row] - M);
            }
            if (whole) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
                const int r = c.rt * ROWS + row;
                const int t = a.by_group.of(r), tok = s.q0 + t, head = c.kvh * a.group + r - t * a.group;
                *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (int64_t)tok * a.sot + (int64_t)head * a.soh + col) =
                    make_uint4(Pair<T>::pack(v[0] * inv, v[1] * inv), Pair<T>::pack(v[2] * inv, v[3] * inv),
                               Pair<T>::pack(v[4] * inv, v[5] * inv), Pair<T>::pack(v[6] * inv, v[7] * inv));
                if (a.lse && col == 0) a.lse[(int64_t)tok * a.heads + head] = log_sum(M, L);
            } else {
                float4* dst = reinterpret_cast<float4*>(a.part_o + ((int64_t)slot * ROWS + row) * D + col);
                dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                dst[1] = make_float4(v[4], v[5], v[6], v[7]);
                if (col == 0) a.part_ml[(int64_t)slot * ROWS + row] = make_float2(M, L);
            }
        }
        if (c.unit == c.u0) desc = describe<ROWS>(a, s, parts_after(c, end), c.kvh, c.rt);
        __syncthreads();  // shared memory is free for the next item
        advance<ROWS, UNIT>(a, c, units);
    }
    if (threadIdx.x == 0) a.desc[blockIdx.x] = desc;
}

template <class T, int D, bool BIAS>
int launch_rows(const RaggedArgs& a, cudaStream_t s) {
    static bool done[64] = {false};
    if (int rc = set_smem_once(attn_rows_kernel<T, D, BIAS>, Cfg<D>::SMEM, done)) return rc;
    const int ctas = Cfg<D>::CTAS * sm_count();
    if (int rc = launch_pdl(attn_rows_kernel<T, D, BIAS>, dim3(ctas), THREADS, Cfg<D>::SMEM, s, "attn_rows_kernel", a)) return rc;
    return launch_pdl(merge_kernel<T, D, ROWS>, dim3(ctas, ROWS / 16), 512, 0, s, "merge_kernel", a);
}

}  // namespace

int64_t rows_workspace(int dim) { return ragged_workspace((dim == 128 ? Cfg<128>::CTAS : Cfg<64>::CTAS) * sm_count(), ROWS, dim); }

int attn_rows(RaggedArgs& a, int dim, bool bf16, void* workspace, cudaStream_t s) {
    const bool bias = a.softcap > 0.f || a.slopes;
    ragged_slots(a, workspace, (dim == 128 ? Cfg<128>::CTAS : Cfg<64>::CTAS) * sm_count(), ROWS, dim);
#define B2_ROWS(T, D) return bias ? launch_rows<T, D, true>(a, s) : launch_rows<T, D, false>(a, s)
    if (dim == 128) {
        if (bf16) B2_ROWS(__nv_bfloat16, 128);
        B2_ROWS(__half, 128);
    }
    if (bf16) B2_ROWS(__nv_bfloat16, 64);
    B2_ROWS(__half, 64);
#undef B2_ROWS
}

unsigned int read_status_attn_rows() {
    unsigned int v = 0, zero = 0;
    cudaMemcpyFromSymbol(&v, g_status, sizeof(v));
    if (v) cudaMemcpyToSymbol(g_status, &zero, sizeof(zero));
    return v;
}

}  // namespace b2
