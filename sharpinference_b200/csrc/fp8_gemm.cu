// Products of block-scaled 8-bit operands on the 5th-generation tensor cores, dense or per expert:
//
//   C[m, n] = sum over blocks b of K of  sa[b, m] * sw[n / 128, b] * sum over k in b of  a[m, k] * w[n, k]
//
// a: e4m3 [rows, K], one float32 scale for 128 neighbours of a row; w: e4m3 [E, N, K], one for 128 x 128.  The tensor core
// adds the 128 products of a block in float32 (tcgen05.mma kind::f8f6f4, four instructions of K = 32); because the scale
// changes with every block the sum leaves tensor memory then and is multiplied and added in float32 registers (fma, one
// rounding a block).
//
// Layout.  A tile is 128 activation rows (the lanes of tensor memory) by TILES * 128 weight rows.  A stage holds 128 bytes
// of K (one swizzle row) of both operands.  Blocks go to two tensor-memory buffers in turn, so the tensor core works on
// one block while the block before it is read out.  Sixteen warps read: four groups of four (128 lanes), each with a
// quarter of the columns, 32 TILES sums a thread in registers; one warp issues the copies, one the MMAs, two multiply the
// scales of rows and weights into a ring in shared memory (a factor a row and weight tile), so the readers' loop is a load
// from tensor memory and paired multiply-adds.  The registers go where the sums are (setmaxnreg: 4 x 112 + 32).
// The grid is one CTA an SM (as many as there are tiles); a CTA walks tiles of all experts, those of one weight tile one
// after the other, and copies and MMAs of its next tile run while the last one's sums are written.
//
// Two epilogues:
//   MODE_STORE   C[out_row, n] = (or +=) s D + bias   float32 or bfloat16; out_row = out_rows[sorted row] or the sorted row,
//                s = row_scale[scale_rows[sorted row] or sorted row] or 1
//   MODE_SWIGLU  w holds gate rows [0, I) and up rows [I, 2 I), I a multiple of 128; h = silu(s g) * (s u) leaves in 8 bits:
//                a tile's 128 columns of h are one block of the next product's K
//
// Every mbarrier wait is bounded; on a timeout the kernel sets *status and winds down.
#include "fp8.cuh"
#include "sm100.cuh"
#include "tensor_map.cuh"

using namespace sm100;

namespace {

constexpr int BM = 128;              // activation rows of a tile (the M of the instruction)
constexpr int WN = 128;              // weight rows of a weight tile: one row of scale blocks
constexpr int BK = fp8::BLOCK;       // K bytes of a stage
constexpr int A_BOX = 32;            // rows of an activation copy: a tile with few rows asks for what it has
constexpr int READERS = 16;          // warps that read tensor memory
constexpr int THREADS = 32 * (READERS + 4);
constexpr int RING = 8;              // blocks of scale factors

enum Mode : int { MODE_STORE = 0, MODE_SWIGLU = 1 };

struct Params {
    const float* a_scale;            // [KB, rows]
    const float* w_scale;            // [E, NB, KB]
    const int* group_offsets;        // [E + 1]; null: one group of all rows
    const int* out_rows;             // MODE_STORE: nullable
    const float* row_scale;          // nullable
    const int* scale_rows;           // nullable
    const float* bias;               // MODE_STORE: [N], nullable
    void* out;                       // MODE_STORE: float or bf16 [*, N]; MODE_SWIGLU: e4m3 [rows, I]
    float* out_scale;                // MODE_SWIGLU: [I / 128, rows]
    int* status;                     // device word: 0 ok, else the code of the wait that gave up
    long long ldq;                   // MODE_SWIGLU: bytes between rows of out
    int rows, N, E, NB, KB;          // NB, KB: blocks of 128 along N and K
    int out_bf16, accumulate, vec;   // vec: rows of out start on 16 bytes
};

template <int TILES>
struct Cfg {
    static constexpr int A_BYTES = BM * BK;
    static constexpr int W_BYTES = WN * BK;
    static constexpr int STAGE = A_BYTES + TILES * W_BYTES;
    static constexpr int STAGES = 4;
    static constexpr int SCALES = TILES * BM * 4;                    // bytes of a ring entry
    static constexpr int STAGING = READERS * 1024;
    static constexpr int BARRIERS = 2 * STAGES + 4 + 2 * RING + 1;
    static constexpr int SMEM = STAGES * STAGE + RING * SCALES + STAGING + BARRIERS * 8 + 16 + 1024;
    static constexpr int COLS = 32 * TILES;                          // columns a reader holds
    static constexpr int BUF = TILES * WN;                           // tensor-memory columns of a buffer
};

__device__ __forceinline__ uint32_t instr_desc_e4m3(int m, int n) {  // e4m3 x e4m3 -> fp32, operands K-major
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void mma_e4m3_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
        "}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// (x, y) += (a, b) * s: the paired multiply-add, two roundings to the nearest as from two fma
__device__ __forceinline__ void fma2(float& x, float& y, uint32_t a, uint32_t b, float s) {
    asm("{\n\t"
        ".reg .b64 c, d, e;\n\t"
        "mov.b64 c, {%2, %3};\n\t"
        "mov.b64 d, {%4, %4};\n\t"
        "mov.b64 e, {%0, %1};\n\t"
        "fma.rn.f32x2 e, c, d, e;\n\t"
        "mov.b64 {%0, %1}, e;\n\t"
        "}"
        : "+f"(x), "+f"(y)
        : "r"(a), "r"(b), "f"(s));
}

// silu(g) * u with the exponential and the reciprocal as single instructions (relative error about 2^-21, before a
// rounding to 2^-4); a large negative g gives -0 * u.
__device__ __forceinline__ float silu_mul(float g, float u) {
    return g * rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * g)) * u;
}

struct Tile {
    int group;                       // -1: no more tiles
    int row0, row_end, nt;           // rows, index of the weight tile (pair)
};

// The tiles of a launch in order: group after group, in a group weight tile after weight tile, in those the row tiles.
// A warp asks for tiles in ascending order; lane l holds the bounds of group base + l.
struct Walk {
    int base, start, end, first, count, before;

    __device__ __forceinline__ void load(const Params& p, int n_tiles) {
        const int lane = threadIdx.x & 31, e = base + lane;
        start = end = 0;
        if (e < p.E) {
            start = p.group_offsets ? min(max(p.group_offsets[e], 0), p.rows) : 0;
            end = p.group_offsets ? min(p.group_offsets[e + 1], p.rows) : p.rows;
        }
        count = end > start ? (end - start + BM - 1) / BM * n_tiles : 0;
        int incl = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        first = before + incl - count;
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    __device__ __forceinline__ void begin(const Params& p, int n_tiles) {
        base = before = 0;
        load(p, n_tiles);
    }
    __device__ __forceinline__ Tile at(int t, const Params& p, int n_tiles) {
        while (t >= before && base + 32 < p.E) {
            base += 32;
            load(p, n_tiles);
        }
        const unsigned hit = __ballot_sync(0xffffffffu, t >= first && t < first + count);
        Tile r;
        r.group = -1;
        r.row0 = r.row_end = r.nt = 0;
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int s = __shfl_sync(0xffffffffu, start, src), f = __shfl_sync(0xffffffffu, first, src);
            r.row_end = __shfl_sync(0xffffffffu, end, src);
            const int row_tiles = (r.row_end - s + BM - 1) / BM;
            r.group = base + src;
            r.nt = (t - f) / row_tiles;
            r.row0 = s + (t - f - r.nt * row_tiles) * BM;
        }
        return r;
    }
};

template <int MODE, int TILES>
__global__ void __launch_bounds__(THREADS, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const Params p) {
    using C = Cfg<TILES>;
    static_assert(MODE == MODE_STORE || TILES == 2, "gate and up are two tiles");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* ring = reinterpret_cast<float*>(smem + C::STAGES * C::STAGE);                  // [RING][TILES][BM]
    uint8_t* staging = smem + C::STAGES * C::STAGE + RING * C::SCALES;
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + C::STAGING);
    uint64_t* empty = full + C::STAGES;
    uint64_t* acc_full = empty + C::STAGES;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* sc_full = acc_empty + 2;
    uint64_t* sc_empty = sc_full + RING;
    uint64_t* drained = sc_empty + RING;
    uint32_t* slot = reinterpret_cast<uint32_t*>(drained + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int I = p.N / 2;
    const int n_tiles = MODE == MODE_SWIGLU ? I / WN : (p.N + C::BUF - 1) / C::BUF;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], READERS);
        }
        for (int r = 0; r < RING; ++r) {
            mbar_init(&sc_full[r], 1);
            mbar_init(&sc_empty[r], READERS);
        }
        mbar_init(drained, 1);
        fence_barrier_init();
    }
    if (warp == READERS + 1) {
        tmem_alloc(slot, 2 * C::BUF);
        tmem_relinquish();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *slot;
    pdl_wait();

    Walk walk;
    if (warp >= READERS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
        walk.begin(p, n_tiles);
        int it = 0;                                                   // blocks of K so far, over all tiles
        bool ok = true;
        if (warp == READERS) {
            // ---- copies ----------------------------------------------------------------------
            for (int t = blockIdx.x; ok; t += gridDim.x) {
                const Tile tile = walk.at(t, p, n_tiles);
                if (tile.group < 0) break;
                const int n0 = tile.nt * (MODE == MODE_SWIGLU ? WN : C::BUF), n1 = MODE == MODE_SWIGLU ? I + n0 : n0 + WN;
                const int boxes = (min(BM, tile.row_end - tile.row0) + A_BOX - 1) / A_BOX;
                if (lane == 0) {
                    for (int kb = 0; kb < p.KB; ++kb, ++it) {
                        const int s = it % C::STAGES;
                        if (it >= C::STAGES) ok = mbar_wait(&empty[s], (it / C::STAGES - 1) & 1);
                        if (!ok) { atomicExch(p.status, 1); break; }
                        uint8_t* stage = smem + s * C::STAGE;
                        mbar_arrive_expect_tx(&full[s], boxes * (A_BOX * BK) + TILES * C::W_BYTES);
                        tma_load_3d(stage + C::A_BYTES, &map_w, &full[s], kb * BK, n0, tile.group);
                        if (TILES == 2) tma_load_3d(stage + C::A_BYTES + C::W_BYTES, &map_w, &full[s], kb * BK, n1, tile.group);
                        for (int b = 0; b < boxes; ++b)
                            tma_load_2d(stage + b * (A_BOX * BK), &map_a, &full[s], kb * BK, tile.row0 + b * A_BOX);
                    }
                }
                ok = __shfl_sync(0xffffffffu, (int)ok, 0);
            }
            if (!ok && lane == 0)                                     // let the copies that were started land
                for (int i = max(0, it - C::STAGES); i < it; ++i) mbar_wait(&full[i % C::STAGES], (i / C::STAGES) & 1, 1u << 16);
        } else if (warp == READERS + 1) {
            // ---- MMAs ------------------------------------------------------------------------
            const uint32_t idesc = instr_desc_e4m3(BM, C::BUF);
            for (int t = blockIdx.x; ok; t += gridDim.x) {
                const Tile tile = walk.at(t, p, n_tiles);
                if (tile.group < 0) break;
                if (lane == 0) {
                    for (int kb = 0; kb < p.KB; ++kb, ++it) {
                        const int s = it % C::STAGES, b = it & 1;
                        if (it >= 2) ok = mbar_wait(&acc_empty[b], (it / 2 - 1) & 1);
                        if (!ok) { atomicExch(p.status, 7); break; }
                        ok = mbar_wait(&full[s], (it / C::STAGES) & 1);
                        if (!ok) { atomicExch(p.status, 2); break; }
                        tcgen05_fence_after();
                        const uint8_t* stage = smem + s * C::STAGE;
#pragma unroll
                        for (int k = 0; k < BK / 32; ++k)
                            mma_e4m3_ss(tmem + b * C::BUF, smem_desc_k_sw128(stage, k * 32), smem_desc_k_sw128(stage + C::A_BYTES, k * 32),
                                        idesc, k != 0);
                        mma_commit(&empty[s]);
                        mma_commit(&acc_full[b]);
                    }
                    if (!ok) {                                        // tensor memory is given back when all MMAs are done
                        mma_commit(drained);
                        mbar_wait(drained, 0, 1u << 16);
                    }
                }
                ok = __shfl_sync(0xffffffffu, (int)ok, 0);
            }
        } else {
            // ---- scales: this warp the blocks of one parity --------------------------------------
            for (int t = blockIdx.x; ok; t += gridDim.x) {
                const Tile tile = walk.at(t, p, n_tiles);
                if (tile.group < 0) break;
                const int nb = tile.nt * (MODE == MODE_SWIGLU ? 1 : TILES);
                const float* w0 = p.w_scale + ((size_t)tile.group * p.NB + nb) * p.KB;
                // a weight tile behind the last row of weights has no scales (its sums are not stored)
                const float* w1 = p.w_scale + ((size_t)tile.group * p.NB + (MODE == MODE_SWIGLU ? nb + I / WN : min(nb + 1, p.NB - 1))) * p.KB;
                const float* a[BM / 32];
#pragma unroll
                for (int i = 0; i < BM / 32; ++i) a[i] = p.a_scale + min(tile.row0 + i * 32 + lane, tile.row_end - 1);
                const int skip = (it ^ (warp - READERS - 2)) & 1;
                for (int kb = skip; kb < p.KB; kb += 2) {
                    const int i = it + kb, r = i % RING;
                    float sa[BM / 32];
#pragma unroll
                    for (int j = 0; j < BM / 32; ++j) sa[j] = a[j][(size_t)kb * p.rows];
                    const float s0 = w0[kb], s1 = TILES == 2 ? w1[kb] : 0.0f;
                    if (i >= RING) ok = mbar_wait(&sc_empty[r], (i / RING - 1) & 1);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) { if (lane == 0) atomicExch(p.status, 8); break; }
#pragma unroll
                    for (int j = 0; j < BM / 32; ++j) {
                        float* dst = ring + r * TILES * BM + j * 32 + lane;
                        dst[0] = sa[j] * s0;
                        if (TILES == 2) dst[BM] = sa[j] * s1;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[r]);
                }
                it += p.KB;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
        // ---- readers: warp w has lanes 32 (w % 4) .. + 31 (a row a thread) and quarter w / 4 of the columns -------
        walk.begin(p, n_tiles);
        const int part = warp >> 2, at = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        int it = 0, turn = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok; t += gridDim.x, ++turn) {
            const Tile tile = walk.at(t, p, n_tiles);
            if (tile.group < 0) break;
            const int row = tile.row0 + at;
            const bool live = row < tile.row_end;
            float acc[C::COLS];
#pragma unroll
            for (int i = 0; i < C::COLS; ++i) acc[i] = 0.0f;
            for (int kb = 0; kb < p.KB; ++kb, ++it) {
                const int b = it & 1, r = it % RING;
                ok = mbar_wait(&sc_full[r], (it / RING) & 1);
                const float* f = ring + r * TILES * BM + at;
                // store: this part's 64 (32) columns in a run; SwiGLU: 32 of the gate's and 32 of the up tile
                const float s0 = f[MODE == MODE_STORE && TILES == 2 ? (part >> 1) * BM : 0];
                const float s1 = MODE == MODE_SWIGLU ? f[BM] : s0;
                ok = ok && mbar_wait(&acc_full[b], (it / 2) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) { if (lane == 0) atomicExch(p.status, 3); break; }
                tcgen05_fence_after();
                uint32_t v[32];
#pragma unroll
                for (int c = 0; c < TILES; ++c) {
                    const int col = MODE == MODE_SWIGLU ? c * WN + part * 32 : part * C::COLS + c * 32;
                    tmem_ld_32_nowait(lanes + b * C::BUF + col, v);
                    tmem_ld_wait();
                    if (c == TILES - 1) {                             // all read: the buffer is free
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(&acc_empty[b]);
                            mbar_arrive(&sc_empty[r]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 2) fma2(acc[c * 32 + i], acc[c * 32 + i + 1], v[i], v[i + 1], c == 0 ? s0 : s1);
                }
            }
            if (MODE == MODE_STORE && !ok) break;
            float rs = 1.0f;
            if (p.row_scale && live) rs = p.row_scale[p.scale_rows ? p.scale_rows[row] : row];
            uint8_t* mine = staging + warp * 1024;
            if constexpr (MODE == MODE_SWIGLU) {
                // 32 columns of h a thread; the block's maximum over the four parts
                float* peak = reinterpret_cast<float*>(mine) + (turn & 1) * 32;
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    acc[i] = silu_mul(acc[i] * rs, acc[32 + i] * rs);
                    m = max(m, fp8::abs_bits(acc[i]));
                }
                peak[lane] = __uint_as_float(m);
                ok = named_barrier_all(1 + (warp & 3), 128, ok);      // a part that gave up takes the other three along
                if (!ok) break;
#pragma unroll
                for (int o = 0; o < 4; ++o)
                    m = max(m, __float_as_uint(reinterpret_cast<const float*>(staging + (o * 4 + (warp & 3)) * 1024)[(turn & 1) * 32 + lane]));
                const float s = fp8::scale_of(m), inv = 1.0f / s;
                if (live) {
                    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + (size_t)row * p.ldq + tile.nt * WN + part * 32);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            w[j] = fp8::pack4(acc[i * 16 + j * 4] * inv, acc[i * 16 + j * 4 + 1] * inv, acc[i * 16 + j * 4 + 2] * inv,
                                              acc[i * 16 + j * 4 + 3] * inv);
                        dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    if (part == 0) p.out_scale[(size_t)tile.nt * p.rows + row] = s;
                }
            } else {
                // 32 bytes of every row at a time go through the warp's staging, so that a store writes whole sectors
                const int to = live ? (p.out_rows ? p.out_rows[row] : row) : -1;
                const int c0 = tile.nt * C::BUF + part * C::COLS;
                if (p.row_scale) {
#pragma unroll
                    for (int i = 0; i < C::COLS; ++i) acc[i] *= rs;
                }
                if (p.bias) {
#pragma unroll
                    for (int i = 0; i < C::COLS; ++i) acc[i] += c0 + i < p.N ? p.bias[c0 + i] : 0.0f;
                }
                const int flip = (lane >> 2) & 1;
                auto put = [&](int piece, uint4 v) { *reinterpret_cast<uint4*>(mine + lane * 32 + ((piece ^ flip) * 16)) = v; };
                auto get = [&](int i) {                               // 16 bytes of row i * 16 + lane / 2
                    const int r = i * 16 + (lane >> 1);
                    return *reinterpret_cast<const uint4*>(mine + r * 32 + (((lane & 1) ^ ((r >> 2) & 1)) * 16));
                };
                if (p.out_bf16) {
                    bf16* out = static_cast<bf16*>(p.out);
#pragma unroll
                    for (int c = 0; c < C::COLS; c += 16) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t w[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const __nv_bfloat162 two = __floats2bfloat162_rn(acc[c + h * 8 + j * 2], acc[c + h * 8 + j * 2 + 1]);
                                w[j] = *reinterpret_cast<const uint32_t*>(&two);
                            }
                            put(h, make_uint4(w[0], w[1], w[2], w[3]));
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int r = __shfl_sync(0xffffffffu, to, i * 16 + (lane >> 1));
                            const uint4 v = get(i);
                            const int n = c0 + c + (lane & 1) * 8;
                            if (r < 0 || n >= p.N) continue;
                            bf16* dst = out + (size_t)r * p.N + n;
                            if (p.vec && n + 8 <= p.N) {
                                *reinterpret_cast<uint4*>(dst) = v;
                            } else {
                                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    if (n + j < p.N) reinterpret_cast<unsigned short*>(dst)[j] = (unsigned short)(w[j / 2] >> (16 * (j & 1)));
                            }
                        }
                        __syncwarp();
                    }
                } else {
                    float* out = static_cast<float*>(p.out);
#pragma unroll
                    for (int c = 0; c < C::COLS; c += 8) {
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            put(h, make_uint4(__float_as_uint(acc[c + h * 4]), __float_as_uint(acc[c + h * 4 + 1]),
                                              __float_as_uint(acc[c + h * 4 + 2]), __float_as_uint(acc[c + h * 4 + 3])));
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int r = __shfl_sync(0xffffffffu, to, i * 16 + (lane >> 1));
                            const uint4 v = get(i);
                            const int n = c0 + c + (lane & 1) * 4;
                            if (r < 0 || n >= p.N) continue;
                            float* dst = out + (size_t)r * p.N + n;
                            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                            if (p.accumulate) {                       // one addend an element from this launch
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    if (n + j < p.N) atomicAdd(dst + j, __uint_as_float(w[j]));
                            } else if (p.vec && n + 4 <= p.N) {
                                *reinterpret_cast<uint4*>(dst) = v;
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    if (n + j < p.N) dst[j] = __uint_as_float(w[j]);
                            }
                        }
                        __syncwarp();
                    }
                }
            }
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == READERS + 1) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, 2 * C::BUF);
    }
}

template <int MODE, int TILES>
int launch(const CUtensorMap& ma, const CUtensorMap& mw, const Params& p, int ctas, cudaStream_t stream) {
    const auto kernel = fp8_gemm_kernel<MODE, TILES>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<TILES>::SMEM) != cudaSuccess) return SHARPI_LAUNCH_FAILED;
    SHARPI_LAUNCH_PDL(kernel, ctas, THREADS, Cfg<TILES>::SMEM, stream, ma, mw, p);
    return SHARPI_OK;
}

}  // namespace

// a [rows, K] with rows `lda` bytes apart, w [E, N, K] with rows `ldw` and groups `ldw * N` bytes apart (multiples of 16).
// swiglu: out e4m3 with rows `ldq` bytes apart and out_scale [N / 256, rows]; else out float32 / bfloat16 [*, N].
SHARPI_API int sharpi_fp8_gemm(const void* a, long long lda, const float* a_scale, const void* w, long long ldw, const float* w_scale,
                               const int* group_offsets, const int* out_rows, const float* row_scale, const int* scale_rows,
                               const float* bias, void* out, long long ldq, float* out_scale, int* status, int rows, int N, int K,
                               int E, int swiglu, int out_bf16, int accumulate, int sms, cudaStream_t stream) {
    if (rows <= 0 || N <= 0) return SHARPI_OK;
    if (K <= 0 || E <= 0 || (E > 1 && !group_offsets) || sms <= 0 || (swiglu && (N % 256 || ldq % 16 || !out_scale)) ||
        (accumulate && (out_bf16 || swiglu)))
        return SHARPI_BAD_ARGUMENT;
    if (lda % 16 || ldw % 16 || lda < K || ldw < K || ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(w)) & 15) ||
        (swiglu && (reinterpret_cast<uintptr_t>(out) & 15)))
        return SHARPI_UNALIGNED;
    const long long m_tiles = (rows + BM - 1) / BM + (E > 1 ? (rows < E ? rows : E) : 0);    // at most
    CUtensorMap ma, mw;
    if (!tmap::make_u8_map(&ma, a, K, rows, 0, lda, A_BOX) || !tmap::make_u8_map(&mw, w, K, N, E, ldw, WN)) return SHARPI_BAD_ARGUMENT;
    Params p = {};
    p.a_scale = a_scale;
    p.w_scale = w_scale;
    p.group_offsets = group_offsets;
    p.out_rows = out_rows;
    p.row_scale = row_scale;
    p.scale_rows = scale_rows;
    p.bias = bias;
    p.out = out;
    p.out_scale = out_scale;
    p.status = status;
    p.ldq = ldq;
    p.rows = rows;
    p.N = N;
    p.E = E;
    p.NB = (N + WN - 1) / WN;
    p.KB = (K + BK - 1) / BK;
    p.out_bf16 = out_bf16;
    p.accumulate = accumulate;
    p.vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && N % (out_bf16 ? 8 : 4) == 0;
    const int cols = swiglu ? 128 : 256;
    const long long tiles = m_tiles * (((swiglu ? N / 2 : N) + cols - 1) / cols);
    if (tiles > 0x3fffffff) return SHARPI_BAD_ARGUMENT;
    const int ctas = (int)(tiles < sms ? tiles : sms);
    return swiglu ? launch<MODE_SWIGLU, 2>(ma, mw, p, ctas, stream) : launch<MODE_STORE, 2>(ma, mw, p, ctas, stream);
}
