// Products of block-scaled 8-bit operands on the 5th-generation tensor cores, dense or per expert:
//
//   C[m, n] = sum over blocks b of K of  sa[b, m] * sw[n / 128, b] * sum over k in b of  a[m, k] * w[n, k]
//
// a: e4m3 [rows, K], one float32 scale for 128 neighbours of a row; w: e4m3 [E, N, K], one for 128 x 128.  The tensor core
// adds the 128 products of a block in float32 (tcgen05.mma kind::f8f6f4, four instructions of K = 32); because the scale
// changes with every block the sum leaves tensor memory then and is multiplied and added in float32 registers (fma, one
// rounding a block).
//
// Layout.  A tile is 128 activation rows (the M side of the instruction, the lanes of tensor memory) by two weight tiles of
// 128 rows.  A stage holds 128 bytes of K (one swizzle row) of both operands.  Blocks go to two tensor-memory buffers in
// turn, so the tensor core works on one block while the block before it is read out.  Eight warps read: two groups of four
// (128 lanes), each with half of the columns, a row and 128 sums a thread; one warp issues the copies, one the MMAs, two
// multiply the scales of rows and weights into a ring in shared memory (a factor a row and weight tile), so the readers' loop
// is loads from tensor memory and paired multiply-adds with one factor.  The registers go where the sums are (setmaxnreg: 2 x
// 224 + 56).  4096 x 16384 x 5120: 330 us; sixteen readers with 64 sums each (104 registers, which spill) 356; with the operands
// swapped (weight rows on the lanes, a factor a column) 650 to 920.  The walks spill 0 (store) and 4 bytes a thread (SwiGLU), the
// clusters 104 and 12.
//
// Two grids.  Many tiles: one CTA an SM that walks tiles of all experts, those of one weight tile one after the other; copies
// and MMAs of its next tile run while the last one's sums are written.  Few tiles: a cluster of S CTAs a tile, each with its
// part of K; the parts meet in the CTAs' shared memory and are added in the order of K, row r by CTA r mod S.
//
// Two epilogues:
//   MODE_STORE   C[out_row, n] = (or +=) s D + bias   float32 or bfloat16; out_row = out_rows[sorted row] or the sorted row,
//                s = row_scale[scale_rows[sorted row] or sorted row] or 1.  Where rows of C start on 32 bytes a thread stores its
//                row, a sector a store; elsewhere sixteen columns at a time change hands in shared memory.  4096 x 16384 x 512:
//                float32 94 us, bfloat16 65 (all rows through shared memory, two columns of sectors at a time: 107 and 73);
//                16380 columns 98, 16383 columns 153
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
constexpr int BN = 2 * WN;           // weight rows of a tile (the N of the instruction)
constexpr int BK = fp8::BLOCK;       // K bytes of a stage
constexpr int READERS = 8;           // warps that read tensor memory
constexpr int THREADS = 32 * (READERS + 4);
constexpr int A_BYTES = BM * BK, W_BYTES = WN * BK, STAGE = A_BYTES + 2 * W_BYTES, STAGES = 4;
constexpr int RING = 8;              // blocks of scale factors, [2][BM] floats each
constexpr int STAGING = READERS * 32 * 16 * 4;
constexpr int BARRIERS = 2 * STAGES + 4 + 2 * RING + 1;
constexpr int SMEM = STAGES * STAGE + RING * 2 * BM * 4 + STAGING + BARRIERS * 8 + 16 + 1024;
constexpr int MAX_SPLIT = 8;

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
    int a_box;                       // rows of an activation copy
    int split;                       // CTAs of a cluster, each with its part of K
    int out_bf16, accumulate, vec;   // vec: the boundary on which rows of out start: 32, 16 or 0 (less)
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

// The barriers of sm100.cuh by shared-memory address
__device__ __forceinline__ bool wait_at(uint32_t bar, uint32_t parity, uint32_t limit) {
    for (uint32_t i = 0; i < limit; ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t"
            "}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ void commit_at(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool elect_one() {
    uint32_t mine;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "}"
        : "=r"(mine));
    return mine != 0;
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

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// 16 bytes of the shared memory of the cluster's CTA `rank`, at the address that `here` has in this CTA's
__device__ __forceinline__ float4 peer_float4(uint32_t here, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(here), "r"(rank));
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

// silu(g) * u.  The exponential and the reciprocal are single instructions; what rounding the exponent -g log2(e) leaves (2^x
// is off by x 2^-24 ln 2 of its value otherwise) is a factor behind it, and a Newton step sharpens the reciprocal: an error
// here sends a value to the next e4m3 number.  A large negative g gives -0 * u.
__device__ __forceinline__ float silu_mul(float g, float u) {
    const float x = -1.4426950408889634f * g, left = fmaf(-1.4426950408889634f, g, -x) - 1.925963033e-8f * g;
    const bool plain = fabsf(x) < 120.0f;
    const float e = ex2_approx(x), d = 1.0f + (plain ? fmaf(e, 0.6931471806f * left, e) : e), r = rcp_approx(d);
    return g * (plain ? fmaf(r, fmaf(-d, r, 1.0f), r) : r) * u;
}

struct Tile {
    int group;                       // -1: no more tiles
    int row0, rows, nt;              // its rows, index of its pair of weight tiles
};

// Tile t of a launch: group after group, in a group weight tile after weight tile, in those the row tiles.  A warp looks it up
// together: lane l counts the tiles of group base + l.  Nothing is kept from one tile to the next: the readers' registers
// are full.
__device__ __forceinline__ Tile find_tile(int t, const Params& p, int n_tiles) {
    const int lane = threadIdx.x & 31;
    Tile r;
    r.group = -1;
    r.row0 = r.rows = r.nt = 0;
    int before = 0;
    for (int base = 0; base < p.E; base += 32) {
        int start = 0, end = 0;
        if (base + lane < p.E) {
            start = p.group_offsets ? min(max(p.group_offsets[base + lane], 0), p.rows) : 0;
            end = p.group_offsets ? min(p.group_offsets[base + lane + 1], p.rows) : p.rows;
        }
        const int count = end > start ? (end - start + BM - 1) / BM * n_tiles : 0;
        int incl = count;
        if (p.E > 1) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
        }
        const int first = before + incl - count;
        const unsigned hit = __ballot_sync(0xffffffffu, t >= first && t < first + count);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int s = __shfl_sync(0xffffffffu, start, src), f = __shfl_sync(0xffffffffu, first, src);
            const int rows = __shfl_sync(0xffffffffu, end, src) - s;
            const int row_tiles = (rows + BM - 1) / BM;
            r.group = base + src;
            r.nt = (t - f) / row_tiles;
            const int at = (t - f - r.nt * row_tiles) * BM;
            r.row0 = s + at;
            r.rows = min(BM, rows - at);
            break;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    return r;
}

// One output element's value and place (MODE_STORE)
__device__ __forceinline__ void put(const Params& p, size_t at, float v) {
    if (p.out_bf16) static_cast<bf16*>(p.out)[at] = __float2bfloat16_rn(v);
    else if (p.accumulate) atomicAdd(static_cast<float*>(p.out) + at, v);     // one addend an element from this launch
    else static_cast<float*>(p.out)[at] = v;
}

__device__ __forceinline__ float row_factor(const Params& p, int row) {
    return p.row_scale ? p.row_scale[p.scale_rows ? p.scale_rows[row] : row] : 1.0f;
}

// 32 bytes to a 32-byte boundary
__device__ __forceinline__ void store_32(void* to, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// WAIT_TEST: nothing is loaded behind the first block of K and every wait gives up after a few thousand polls
template <int MODE, bool SPLIT, bool WAIT_TEST>
__global__ void __launch_bounds__(THREADS, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const Params p) {
    constexpr uint32_t POLLS = WAIT_TEST ? 1u << 12 : WAIT_LIMIT;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* ring = reinterpret_cast<float*>(smem + STAGES * STAGE);                        // [RING][2][BM]
    float* staging = ring + RING * 2 * BM;                                                // [READERS][32][16]
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + READERS * 32 * 16);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* sc_full = acc_empty + 2;
    uint64_t* sc_empty = sc_full + RING;
    uint64_t* drained = sc_empty + RING;
    uint32_t* slot = reinterpret_cast<uint32_t*>(drained + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int I = p.N / 2;
    const int n_tiles = MODE == MODE_SWIGLU ? I / WN : (p.N + BN - 1) / BN;
    // this CTA's tiles and its part of K
    const int rank = SPLIT ? blockIdx.x % p.split : 0;
    const int t_first = SPLIT ? blockIdx.x / p.split : blockIdx.x, t_step = SPLIT ? 0x40000000 : gridDim.x;
    const int kb0 = SPLIT ? p.KB * rank / p.split : 0, kb1 = SPLIT ? p.KB * (rank + 1) / p.split : p.KB;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
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
    if (warp == READERS) {
        prefetch_tensormap(&map_w);
        prefetch_tensormap(&map_a);
    }
    if (warp == READERS + 1) {
        tmem_alloc(slot, 2 * BN);
        tmem_relinquish();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *slot;
    pdl_wait();

    Tile only = {-1, 0, 0, 0};                                        // SPLIT: the cluster's tile
    if (warp >= READERS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        int it = 0;                                                   // blocks of K so far, over all tiles
        bool ok = true;
        if (warp == READERS) {
            // ---- copies ----------------------------------------------------------------------
            for (int t = t_first; ok; t += t_step) {
                const Tile tile = find_tile(t, p, n_tiles);
                if (tile.group < 0) break;
                const int n0 = tile.nt * (MODE == MODE_SWIGLU ? WN : BN), n1 = MODE == MODE_SWIGLU ? I + n0 : n0 + WN;
                const int boxes = (tile.rows + p.a_box - 1) / p.a_box;
                if (lane == 0) {
                    for (int kb = kb0; kb < kb1; ++kb, ++it) {
                        const int s = it % STAGES;
                        if (it >= STAGES) ok = mbar_wait(&empty[s], (it / STAGES - 1) & 1, POLLS);
                        if (!ok) { atomicExch(p.status, 1); break; }
                        if (WAIT_TEST && kb > 0) continue;
                        uint8_t* stage = smem + s * STAGE;
                        mbar_arrive_expect_tx(&full[s], boxes * p.a_box * BK + 2 * W_BYTES);
                        tma_load_3d(stage + A_BYTES, &map_w, &full[s], kb * BK, n0, tile.group);
                        tma_load_3d(stage + A_BYTES + W_BYTES, &map_w, &full[s], kb * BK, n1, tile.group);
                        // rows of the tile only (its other lanes hold what was there; nobody reads them)
                        for (int b = 0; b < boxes; ++b) tma_load_2d(stage + b * p.a_box * BK, &map_a, &full[s], kb * BK, tile.row0 + b * p.a_box);
                    }
                }
                ok = __shfl_sync(0xffffffffu, (int)ok, 0);
            }
            if (!ok && lane == 0)                                     // let the copies that were started land
                for (int i = max(0, it - STAGES); i < it; ++i) mbar_wait(&full[i % STAGES], (i / STAGES) & 1, min(POLLS, 1u << 16));
        } else if (warp == READERS + 1) {
            // ---- MMAs: the whole warp walks (its counters and addresses are uniform), one thread issues ----------------
            const uint32_t idesc = instr_desc_e4m3(BM, BN);
            const uint64_t desc0 = smem_desc_k_sw128(smem);
            const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty), got0 = smem_u32(acc_full), free0 = smem_u32(acc_empty);
            for (int t = t_first; ok; t += t_step) {
                const Tile tile = find_tile(t, p, n_tiles);
                if (tile.group < 0) break;
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const uint32_t s = it % STAGES, b = it & 1;
                    ok = wait_at(free0 + 8 * b, ((it >> 1) & 1) ^ 1, POLLS);      // (the phase before the first counts as complete)
                    if (!ok) { if (lane == 0) atomicExch(p.status, 7); break; }
                    ok = wait_at(full0 + 8 * s, (it / STAGES) & 1, POLLS);
                    if (!ok) { if (lane == 0) atomicExch(p.status, 2); break; }
                    tcgen05_fence_after();
                    const uint64_t da = desc0 + s * (STAGE >> 4), dw = da + (A_BYTES >> 4);
                    const uint32_t d = tmem + b * BN;
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < BK / 32; ++k) mma_e4m3_ss(d, da + 2 * k, dw + 2 * k, idesc, k != 0);
                        commit_at(empty0 + 8 * s);
                        commit_at(got0 + 8 * b);
                    }
                    __syncwarp();
                }
            }
            if (!ok && lane == 0) {                                   // tensor memory is given back when all MMAs are done
                mma_commit(drained);
                mbar_wait(drained, 0, 1u << 16);
            }
        } else {
            // ---- scales: this warp the blocks of one parity --------------------------------------
            for (int t = t_first; ok; t += t_step) {
                const Tile tile = find_tile(t, p, n_tiles);
                if (tile.group < 0) break;
                const int nb = tile.nt * (MODE == MODE_SWIGLU ? 1 : 2);
                const float* w0 = p.w_scale + ((size_t)tile.group * p.NB + nb) * p.KB;
                // a weight tile behind the last row of weights has no scales (its sums are not stored)
                const float* w1 = p.w_scale + ((size_t)tile.group * p.NB + (MODE == MODE_SWIGLU ? nb + I / WN : min(nb + 1, p.NB - 1))) * p.KB;
                const int last = tile.row0 + tile.rows - 1;
                const int skip = (it ^ (warp - READERS - 2)) & 1;
                for (int kb = kb0 + skip; kb < kb1; kb += 2) {
                    const int i = it + kb - kb0, r = i % RING;
                    const float* a = p.a_scale + (size_t)kb * p.rows;
                    float sa[BM / 32];
#pragma unroll
                    for (int j = 0; j < BM / 32; ++j) sa[j] = a[min(tile.row0 + j * 32 + lane, last)];
                    const float s0 = w0[kb], s1 = w1[kb];
                    if (i >= RING) ok = mbar_wait(&sc_empty[r], (i / RING - 1) & 1, POLLS);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) { if (lane == 0) atomicExch(p.status, 8); break; }
#pragma unroll
                    for (int j = 0; j < BM / 32; ++j) {
                        float* dst = ring + r * 2 * BM + j * 32 + lane;
                        dst[0] = sa[j] * s0;
                        dst[BM] = sa[j] * s1;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[r]);
                }
                it += kb1 - kb0;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ---- readers: warp w has lanes 32 (w % 4) .. + 31 (a row a thread) and half w / 4 of the columns: a weight tile
        // (store), or the same 64 columns of the gate's and the up tile (SwiGLU) ----------------------------------------
        const int part = warp >> 2, at = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + part * (MODE == MODE_SWIGLU ? WN / 2 : WN);
        constexpr int SECOND = MODE == MODE_SWIGLU ? WN : WN / 2;     // from this thread's first 64 columns to its others
        int it = 0, turn = 0;
        bool ok = true;
        for (int t = t_first; ok; t += t_step, turn ^= 1) {
            const Tile tile = find_tile(t, p, n_tiles);
            if (tile.group < 0) break;
            const int row = tile.row0 + at;
            const bool live = at < tile.rows;
            // asked for here, in front of the tile's blocks, not when their sums wait for them
            const float rs = live && !SPLIT ? row_factor(p, row) : 0.0f;
            const int to = live && !SPLIT ? (MODE == MODE_STORE && p.out_rows ? p.out_rows[row] : row) : -1;
            float acc[2][64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[0][i] = acc[1][i] = 0.0f;
            const bool any = (warp & 3) * 32 < tile.rows;             // a warp without rows keeps the count alone
            for (int kb = kb0; kb < kb1 && !any; ++kb, ++it) {
                ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[it & 1], (it / 2) & 1, POLLS));
                if (!ok) { if (lane == 0) atomicExch(p.status, 3); break; }
                if (lane == 0) {
                    mbar_arrive(&acc_empty[it & 1]);
                    mbar_arrive(&sc_empty[it % RING]);
                }
            }
            for (int kb = kb0; kb < kb1 && any; ++kb, ++it) {
                const int b = it & 1, r = it % RING;
                ok = mbar_wait(&sc_full[r], (it / RING) & 1, POLLS);
                const float* f = ring + r * 2 * BM + at;
                const float s0 = f[MODE == MODE_STORE ? part * BM : 0], s1 = MODE == MODE_SWIGLU ? f[BM] : s0;
                ok = ok && mbar_wait(&acc_full[b], (it / 2) & 1, POLLS);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) { if (lane == 0) atomicExch(p.status, 3); break; }
                tcgen05_fence_after();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t v[2][32];
                    tmem_ld_32_nowait(lanes + b * BN + h * SECOND, v[0]);
                    tmem_ld_32_nowait(lanes + b * BN + h * SECOND + 32, v[1]);
                    tmem_ld_wait();
                    if (h == 1) {                                     // all read: the buffer is free
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(&acc_empty[b]);
                            mbar_arrive(&sc_empty[r]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 64; i += 2) fma2(acc[h][i], acc[h][i + 1], v[i / 32][i % 32], v[i / 32][i % 32 + 1], h == 0 ? s0 : s1);
                }
            }
            if constexpr (SPLIT) {
                // this CTA's sums, [row][256 columns] with the 16-byte pieces of a row swapped by the row's last three bits,
                // where its stages were: every copy has landed and every MMA has read it, or the call has failed
                only = tile;
                if (!ok) break;
                if (live) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 64; i += 4) {
                            const int piece = (part * (MODE == MODE_SWIGLU ? WN / 2 : WN) + h * SECOND + i) / 4;
                            *reinterpret_cast<float4*>(smem + at * (BN * 4) + (piece ^ (at & 7)) * 16) =
                                make_float4(acc[h][i], acc[h][i + 1], acc[h][i + 2], acc[h][i + 3]);
                        }
                }
                break;
            }
            if (MODE == MODE_STORE && !ok) break;
            float* mine = staging + warp * 32 * 16;
            if constexpr (MODE == MODE_SWIGLU) {
                // 64 columns of h a thread; the block's maximum over the two parts
                uint32_t* peak = reinterpret_cast<uint32_t*>(staging) + turn * BM * 2 + at * 2;
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    acc[0][i] = silu_mul(acc[0][i] * rs, acc[1][i] * rs);
                    m = max(m, fp8::abs_bits(acc[0][i]));
                }
                peak[part] = m;
                ok = named_barrier_all(1 + (warp & 3), 64, ok);       // a part that gave up takes the other along
                if (!ok) break;
                m = max(m, peak[part ^ 1]);
                const float s = fp8::scale_of(m), inv = 1.0f / s;
                if (live) {
                    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + (size_t)row * p.ldq + tile.nt * WN + part * 64);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float* x = &acc[0][i * 16 + j * 4];
                            w[j] = fp8::pack4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
                        }
                        dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    if (part == 0) p.out_scale[(size_t)tile.nt * p.rows + row] = s;
                }
            } else {
                const int c0 = tile.nt * BN + part * WN;
                if (p.row_scale) {
#pragma unroll
                    for (int i = 0; i < WN; ++i) acc[i / 64][i % 64] *= rs;
                }
                if (p.bias) {
#pragma unroll
                    for (int i = 0; i < WN; ++i) acc[i / 64][i % 64] += c0 + i < p.N ? p.bias[c0 + i] : 0.0f;
                }
                if (p.vec == 32 && !p.accumulate) {
                    // a row a thread, 32 bytes (a whole sector) at a time
                    if (p.out_bf16) {
                        bf16* dst = static_cast<bf16*>(p.out) + (size_t)to * p.N + c0;
#pragma unroll
                        for (int i = 0; i < WN; i += 16) {
                            uint32_t w[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const __nv_bfloat162 two = __floats2bfloat162_rn(acc[i / 64][i % 64 + 2 * j], acc[i / 64][i % 64 + 2 * j + 1]);
                                w[j] = *reinterpret_cast<const uint32_t*>(&two);
                            }
                            if (live && c0 + i < p.N) store_32(dst + i, w);
                        }
                    } else {
                        float* dst = static_cast<float*>(p.out) + (size_t)to * p.N + c0;
#pragma unroll
                        for (int i = 0; i < WN; i += 8) {
                            uint32_t w[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(acc[i / 64][i % 64 + j]);
                            if (live && c0 + i < p.N) store_32(dst + i, w);
                        }
                    }
                } else {
                    // rows that start elsewhere, or sums that are added: sixteen columns of every row at a time through the warp's
                    // staging (the pieces of a row swapped by two bits of it), so that neighbouring columns are neighbouring lanes'
                    const int have = min(32, tile.rows - (warp & 3) * 32);
#pragma unroll
                    for (int c = 0; c < WN; c += 16) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float* x = &acc[c / 64][c % 64 + q * 4];
                            *reinterpret_cast<float4*>(mine + lane * 16 + (q ^ ((lane >> 1) & 3)) * 4) = make_float4(x[0], x[1], x[2], x[3]);
                        }
                        __syncwarp();
                        if (p.vec && !p.accumulate) {
#pragma unroll
                            for (int r0 = 0; r0 < 32; r0 += 8) {
                                const int r = r0 + (lane >> 2), n = c0 + c + (lane & 3) * 4, from = __shfl_sync(0xffffffffu, to, r);
                                if (r >= have || n >= p.N) continue;
                                const float4 v = *reinterpret_cast<const float4*>(mine + r * 16 + ((lane ^ (r >> 1)) & 3) * 4);
                                const float x[4] = {v.x, v.y, v.z, v.w};
                                if (p.out_bf16) store_four(static_cast<bf16*>(p.out) + (size_t)from * p.N + n, x);
                                else store_four(static_cast<float*>(p.out) + (size_t)from * p.N + n, x);
                            }
                        } else {
#pragma unroll 4
                            for (int r0 = 0; r0 < have; r0 += 2) {
                                const int r = r0 + (lane >> 4), n = c0 + c + (lane & 15), from = __shfl_sync(0xffffffffu, to, r);
                                if (r < have && n < p.N)
                                    put(p, (size_t)from * p.N + n, mine[r * 16 + ((((lane & 15) / 4) ^ (r >> 1)) & 3) * 4 + lane % 4]);
                            }
                        }
                        __syncwarp();
                    }
                }
            }
        }
    }
    if constexpr (SPLIT) {
        cluster_sync();
        if (warp < READERS && only.group >= 0) {
            // a warp a row: 4 neighbouring columns a lane (of both weight tiles), the CTAs' parts in the order of K
            const int n0 = only.nt * (MODE == MODE_SWIGLU ? WN : BN);
            for (int c = rank + p.split * warp; c < only.rows; c += p.split * READERS) {
                const uint32_t here = smem_u32(smem) + c * (BN * 4) + ((lane ^ (c & 7)) * 16);
                float4 v[2] = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
#pragma unroll 4
                for (int r = 0; r < p.split; ++r) {
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const float4 x = peer_float4(here + w * WN * 4, r);
                        v[w].x += x.x;
                        v[w].y += x.y;
                        v[w].z += x.z;
                        v[w].w += x.w;
                    }
                }
                const int row = only.row0 + c;
                const float rs = row_factor(p, row);
                if constexpr (MODE == MODE_SWIGLU) {
                    const float h[4] = {silu_mul(v[0].x * rs, v[1].x * rs), silu_mul(v[0].y * rs, v[1].y * rs),
                                        silu_mul(v[0].z * rs, v[1].z * rs), silu_mul(v[0].w * rs, v[1].w * rs)};
                    uint32_t m = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) m = max(m, fp8::abs_bits(h[i]));
                    const float scale = fp8::scale_of(__reduce_max_sync(0xffffffffu, m)), inv = 1.0f / scale;
                    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.out) + (size_t)row * p.ldq + n0 + lane * 4) =
                        fp8::pack4(h[0] * inv, h[1] * inv, h[2] * inv, h[3] * inv);
                    if (lane == 0) p.out_scale[(size_t)only.nt * p.rows + row] = scale;
                } else {
                    const size_t to = p.out_rows ? p.out_rows[row] : row;
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const int n = n0 + w * WN + lane * 4;
                        if (n >= p.N) continue;
                        float x[4] = {v[w].x, v[w].y, v[w].z, v[w].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (p.row_scale) x[i] *= rs;
                            if (p.bias) x[i] += p.bias[min(n + i, p.N - 1)];
                        }
                        if (p.vec && !p.accumulate) {
                            if (p.out_bf16) store_four(static_cast<bf16*>(p.out) + to * p.N + n, x);
                            else store_four(static_cast<float*>(p.out) + to * p.N + n, x);
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (n + i < p.N) put(p, to * p.N + n + i, x[i]);
                        }
                    }
                }
            }
        }
        cluster_sync();                                               // nobody leaves while its sums are read
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == READERS + 1) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, 2 * BN);
    }
}

// The shared memory that a kernel may take, set once a device
template <typename K>
bool allow_shared(K kernel, bool (&done)[64]) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= 64) return false;
    if (!done[device]) done[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) == cudaSuccess;
    return done[device];
}

template <int MODE, bool SPLIT, bool WAIT_TEST>
int launch(const CUtensorMap& ma, const CUtensorMap& mw, const Params& p, int ctas, cudaStream_t stream) {
    const auto kernel = fp8_gemm_kernel<MODE, SPLIT, WAIT_TEST>;
    static bool done[64];
    if (!allow_shared(kernel, done)) return SHARPI_LAUNCH_FAILED;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = ctas;
    cfg.blockDim = THREADS;
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (SPLIT) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = p.split;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (sharpi_pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, ma, mw, p) == cudaSuccess ? SHARPI_OK : SHARPI_LAUNCH_FAILED;
}

// How many clusters of `split` CTAs the device holds at once (asked once a device)
int clusters_at_once(int split) {
    constexpr int DEVICES = 64;
    static int known[DEVICES][MAX_SPLIT + 1];
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= DEVICES) return 0;
    if (known[device][split] == 0) {
        const auto kernel = fp8_gemm_kernel<MODE_STORE, true, false>;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = 8 * split;
        cfg.blockDim = THREADS;
        cfg.dynamicSmemBytes = SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = split;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0)
            n = -1;
        known[device][split] = n;
    }
    return known[device][split];
}

// Into how many CTAs a tile's K is cut: the fewest blocks of K one after the other, a wave of clusters counted as its blocks
// and what starting it and joining the parts takes.  1 x 7168 x 5120: 11.9 us in four, 21.8 uncut, 19.4 in five (more clusters than
// the GPU holds); 45 x 5003 x 4100: 11.3 in six, 25.3 uncut; 8 rows of 32 experts of 2048 x 1408: 8.9 in two, 9.6 uncut.
int choose_split(long long tiles, int KB, int sms) {
    int best = 1;
    long long least = (tiles + sms - 1) / sms * KB + 3;
    for (int s = 2; s <= MAX_SPLIT && s <= KB; ++s) {
        const int at_once = clusters_at_once(s);
        if (at_once <= 0) continue;
        const long long cost = (tiles + at_once - 1) / at_once * ((KB + s - 1) / s + 5);
        if (cost < least) {
            least = cost;
            best = s;
        }
    }
    return best;
}

template <int MODE, bool WAIT_TEST>
int launch_mode(const CUtensorMap& ma, const CUtensorMap& mw, const Params& p, long long tiles, int sms, cudaStream_t stream) {
    return p.split > 1 ? launch<MODE, true, WAIT_TEST>(ma, mw, p, (int)tiles * p.split, stream)
                       : launch<MODE, false, WAIT_TEST>(ma, mw, p, (int)(tiles < sms ? tiles : sms), stream);
}

bool wait_test = false;

}  // namespace

// Test hook: the NEXT launch runs the kernel whose waits run out: it writes the code of one of them and returns with its tensor
// memory freed.  (A kernel of its own: a limit that is an argument took the others 1 % of their time.)
SHARPI_API void sharpi_fp8_set_wait_test() { wait_test = true; }

// a [rows, K] with rows `lda` bytes apart, w [E, N, K] with rows `ldw` and groups `ldw * N` bytes apart (multiples of 16).
// swiglu: out e4m3 with rows `ldq` bytes apart and out_scale [N / 256, rows]; else out float32 / bfloat16 [*, N].
// split: 0 = chosen here, else into how many CTAs a tile's K is cut.
SHARPI_API int sharpi_fp8_gemm(const void* a, long long lda, const float* a_scale, const void* w, long long ldw, const float* w_scale,
                               const int* group_offsets, const int* out_rows, const float* row_scale, const int* scale_rows,
                               const float* bias, void* out, long long ldq, float* out_scale, int* status, int rows, int N, int K,
                               int E, int swiglu, int out_bf16, int accumulate, int split, int sms, cudaStream_t stream) {
    if (rows <= 0 || N <= 0) return SHARPI_OK;
    if (K <= 0 || E <= 0 || (E > 1 && !group_offsets) || sms <= 0 || (swiglu && (N % 256 || ldq % 16 || !out_scale)) ||
        (accumulate && (out_bf16 || swiglu)) || split < 0 || split > MAX_SPLIT || split > (K + BK - 1) / BK)
        return SHARPI_BAD_ARGUMENT;
    if (lda % 16 || ldw % 16 || lda < K || ldw < K || ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(w)) & 15) ||
        (swiglu && (reinterpret_cast<uintptr_t>(out) & 15)))
        return SHARPI_UNALIGNED;
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
    const uintptr_t starts = reinterpret_cast<uintptr_t>(out) | (uintptr_t)N * (out_bf16 ? 2 : 4);
    p.vec = starts % 32 == 0 ? 32 : starts % 16 == 0 ? 16 : 0;
    const long long row_tiles = rows < E ? rows : (rows + BM - 1) / BM + (E > 1 ? E : 0);        // at most
    const long long tiles = row_tiles * (swiglu ? N / BN : (N + BN - 1) / BN);
    if (tiles > 0x3fffffff / MAX_SPLIT) return SHARPI_BAD_ARGUMENT;
    p.split = split ? split : choose_split(tiles, p.KB, sms);
    // copies as small as a few rows, as few as many rows of one matrix allow
    p.a_box = rows <= 16 ? 16 : E == 1 && rows > 96 ? 128 : 32;
    CUtensorMap ma, mw;
    if (!tmap::make_u8_map(&ma, a, K, rows, 0, lda, p.a_box) || !tmap::make_u8_map(&mw, w, K, N, E, ldw, WN)) return SHARPI_BAD_ARGUMENT;
    const bool test = wait_test;
    wait_test = false;
    if (test) return swiglu ? launch_mode<MODE_SWIGLU, true>(ma, mw, p, tiles, sms, stream) : launch_mode<MODE_STORE, true>(ma, mw, p, tiles, sms, stream);
    return swiglu ? launch_mode<MODE_SWIGLU, false>(ma, mw, p, tiles, sms, stream) : launch_mode<MODE_STORE, false>(ma, mw, p, tiles, sms, stream);
}
