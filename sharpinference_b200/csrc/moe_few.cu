// A whole mixture-of-experts layer for up to 16 tokens in two kernels:
//
//   router    z = h Wr^T (float32), a warp a (token, expert)
//   experts   every token's k experts and their weights from z; act = silu(g) * u over the gate|up rows of the experts that
//             any token chose; a barrier over the grid; y[t] = add[t] + sum over the token's experts of w Wd act
//
// With few tokens the layer is a stream of the chosen experts' weights, so the second kernel is laid out for that alone: one
// CTA an SM, weight rows dealt out evenly over the warps whatever expert they belong to, each weight read once, in 16-byte
// pieces straight into registers.  Teams of 1 to 16 warps share K in turn (the more K has, the more); a warp asks for its next
// step of 4 KB when it has multiplied the last (up to 64 KB an SM in flight; reading at 6.4 TB/s with a microsecond of latency
// takes 44 KB; asking whole rows into L2 ahead of that took 3 to 8 % longer).  8 tokens, 1 of 16 experts of 5120 x 8192 in 8 bits:
// 178 us, 4.6 TB/s.  The activations come through L1: a copy of them in shared memory left too little of it for the loads on
// their way (2 of 16 experts, bfloat16: 16 tokens of 5120 118 us and 194 with the copy, 8 of 8192 103 and 116, 8 of 2048 the
// same).  Weights are the 16-row operand of the MMA (eight gate rows and their up rows, or sixteen rows of the down
// matrix), tokens the eight columns; a column of a token that did not choose the expert is computed and dropped (gate|up), or is
// zeros and its sums stay as they were (down: selected, not added, since 0 times an infinity or a NaN among the expert's weights
// is a NaN; 9 to 16 tokens with bfloat16 weights take 1 to 4 % longer for it, the others nothing).  Because the down product is
// linear, a token's experts are one long sum over (expert, inner element): act is multiplied by the router's weight before (weights
// on the output).  The warps' parts are added in warp order: a call's result is the same every time, but the order (float32
// rounding) of a token's sum goes by which experts the whole call reaches.
//
// bfloat16 weights: mma.sync m16n8k16.  act is two bfloat16, its rounding and what that left (together within 2^-16 of its
// value), multiplied one after the other into the same sums.  With the first alone (2^-8) a layer in bfloat16 is off by 1.4 times
// its own rounding; the second costs 27.8 us for 27.0 (one token, 8 of 128 experts, 2048 x 768) and 163 for 145 (16 tokens; the
// selection of sums brings 2 more).
//
// e4m3 weights with a scale for 128 x 128 (fp8.cuh): an e4m3 value is a float16 one (cvt, two an instruction), and the MMA is
// m16n8k16 on float16.  (mma.sync on e4m3 is no instruction of this GPU's: it converts both operands for every tile, 1000
// instructions a step of 4 KB where this takes 250.)  The activations are float16 times a power of two s for 128 neighbours such
// that the largest |x / s| is 2^14 to 2^15: of h's eight bits none is lost down to 2^-31 of its block's largest value; act is off by
// 2^-11 of its value, or, below 2^-28 of its block's largest, by 2^-39 of that.  A block's 128 products are added in float32, then
// scaled and added.  Infinities and NaN make a block's scale NaN.  9 to 16 tokens spill (202 bytes a thread; bfloat16 18, else none).
//
// The barrier needs all CTAs on the GPU at once: the launch is cooperative.  Its counters lie in the call's own workspace and
// are set to zero by the router kernel.  The wait is bounded; on a timeout the kernel sets *status and returns.
#include "fp8.cuh"
#include "mma_sync.cuh"

#include <cuda_fp16.h>

namespace {

constexpr int MAX_T = 16, MAX_K = 32, MAX_E = 1024;
constexpr int IN_REGISTERS = 128;              // experts whose scores a warp holds in registers while it chooses
constexpr int WARPS = 16, THREADS = 32 * WARPS;
constexpr int NT = 2;                          // tiles of sixteen weight rows that a warp has at a time
constexpr uint32_t BARRIER_LIMIT = 1u << 22;

struct Params {
    const float* z;               // [T, E]
    const float* bias;            // [E] or null
    const float* correction;      // [E] or null
    const uint8_t* x;             // [T] rows ldx bytes apart: h, or (e4m3 weights) h / x_scale in float16
    const float* x_scale;         // e4m3: [T, blocks of H]
    const void* gate_up;          // [E, 2 I, ldg] bytes apart
    const void* down;             // [E, H, ldd] bytes apart
    const float* gate_up_scale;   // e4m3: [E, blocks of 2 I, blocks of H]
    const float* down_scale;      // e4m3: [E, blocks of H, blocks of I]
    const float* add;             // [T, H] or null
    void* act;                    // bf16 weights: bf16 [active, T, Ip]; e4m3: float [active, T, Ip]
    bf16* act_low;                // bf16 weights: what act's rounding left, [active, T, Ip]
    __half* act16;                // e4m3: act / act_scale [active, T, Ip]
    float* act_scale;             // e4m3: [active, T, blocks of I]
    void* out;                    // [T, H]
    int* barrier;                 // two counters
    int* status;
    long long ldg, ldd;           // bytes
    int ldx, T, E, k, H, I, Ip;   // Ip: I rounded up to 128
    int softmax, renormalize, on_input, out_bf16;
    int team;                     // warps that share the K of gate and up rows
    float scale;
    uint32_t polls;               // of a barrier's counter before a wait gives up
};

// The scale of a block whose largest magnitude has the bits `amax`: a power of two such that amax / s < 2^15
__device__ __forceinline__ float half_scale(uint32_t amax) {
    if (amax >= 0x7f800000u) return __int_as_float(0x7fc00000);           // infinity or NaN
    const int e = max((int)(amax >> 23), 15);                             // amax < 2^(e - 126)
    return __uint_as_float((uint32_t)(e - 14) << 23);                     // 2^(e - 141)
}
// Four neighbours of a block with scale s in float16
__device__ __forceinline__ uint2 halves(const float (&v)[4], float s) {
    const float inv = s == s ? 1.0f / s : 0.0f;                           // (a power of two; what has no scale counts for nothing)
    const __half2 a = __floats2half2_rn(v[0] * inv, v[1] * inv), b = __floats2half2_rn(v[2] * inv, v[3] * inv);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// One warp a (token, expert), the additions in the order of the router kernels for more tokens: lane l adds the elements
// 128 i + 4 l + u in ascending i into chain u, the chains and then the lanes are added in a fixed order.
template <typename T>
__global__ void __launch_bounds__(128)
moe_few_router_kernel(const T* h, int ldh, const float* wr, int tokens, int H, int E, int vec, float* z, int* barrier,
                      const bf16* rows, int ld_rows, __half* rows16, int ld16, float* x_scale) {
    const int item = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int e = item / tokens, t = item - e * tokens;
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x < 2) barrier[threadIdx.x] = 0;
    if (e >= E) {                                        // e4m3 weights: the warps behind the experts' make h float16
        const int kb = e - E, k = kb * fp8::BLOCK + lane * 4;
        if (kb * fp8::BLOCK >= ld16) return;
        float v[4];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = k + i < H ? __bfloat162float(rows[(size_t)t * ld_rows + k + i]) : 0.0f;
            m = max(m, fp8::abs_bits(v[i]));
        }
        const float s = half_scale(__reduce_max_sync(0xffffffffu, m));
        *reinterpret_cast<uint2*>(rows16 + (size_t)t * ld16 + k) = halves(v, s);
        if (lane == 0) x_scale[(size_t)t * (ld16 / fp8::BLOCK) + kb] = s;
        return;
    }
    const T* x = h + (size_t)t * ldh;
    const float* w = wr + (size_t)e * H;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (vec) {
        constexpr int BATCH = 8;                         // loads in flight, whatever is left of the row
#pragma unroll 1
        for (int i0 = 4 * lane; i0 < H; i0 += 128 * BATCH) {
            float4 wv[BATCH];
            float xv[BATCH][4];
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                const int i = i0 + 128 * b;
                if (i >= H) continue;
                wv[b] = *reinterpret_cast<const float4*>(w + i);
                if constexpr (sizeof(T) == 4) {
                    const float4 q = *reinterpret_cast<const float4*>(x + i);
                    xv[b][0] = q.x; xv[b][1] = q.y; xv[b][2] = q.z; xv[b][3] = q.w;
                } else {
                    const uint2 q = *reinterpret_cast<const uint2*>(x + i);
                    xv[b][0] = __uint_as_float(q.x << 16); xv[b][1] = __uint_as_float(q.x & 0xffff0000u);
                    xv[b][2] = __uint_as_float(q.y << 16); xv[b][3] = __uint_as_float(q.y & 0xffff0000u);
                }
            }
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                if (i0 + 128 * b >= H) continue;
                acc[0] = fmaf(xv[b][0], wv[b].x, acc[0]);
                acc[1] = fmaf(xv[b][1], wv[b].y, acc[1]);
                acc[2] = fmaf(xv[b][2], wv[b].z, acc[2]);
                acc[3] = fmaf(xv[b][3], wv[b].w, acc[3]);
            }
        }
    } else {
        for (int i = 4 * lane; i < H; i += 128) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u < H) acc[u] = fmaf(to_float(x[i + u]), w[i + u], acc[u]);
        }
    }
    const float s = warp_sum((acc[0] + acc[1]) + (acc[2] + acc[3]));
    if (lane == 0) z[(size_t)t * E + e] = s;
}

__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four e4m3 values as float16
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t"
        ".reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t"
        "}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}

// How a step of a warp reads K: a lane has 16 bytes of two weight rows (eight apart in the tile) in each of two pieces; lanes
// 4 g + t of a row lie side by side.  Which elements of K share an MMA is free as long as both operands agree: lane t's
// elements are its k values.
constexpr int STEP = 128;         // bytes of a row: one block of e4m3, 64 bfloat16 values

// The first `left` of 16 bytes, zeros behind them
__device__ __forceinline__ uint4 cut(uint4 v, int left) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = left - 4 * i;
        w[i] = n >= 4 ? w[i] : n <= 0 ? 0u : w[i] & (0xffffffffu >> (32 - 8 * n));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A tile's weights of a step: [row g or g + 8][piece].  `len`: bytes of a row; behind them zeros, whatever lies between rows.
__device__ __forceinline__ void fetch(uint4 (&w)[2][2], const uint8_t* low, const uint8_t* high, int at, int len) {
    const int k = at + (threadIdx.x & 3) * 16;
    if (at + STEP <= len) {
        w[0][0] = load_stream(low + k);
        w[1][0] = load_stream(high + k);
        w[0][1] = load_stream(low + k + 64);
        w[1][1] = load_stream(high + k + 64);
    } else {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int left = len - (k + 64 * p);
            w[0][p] = left > 0 ? cut(load_stream(low + k + 64 * p), left) : make_uint4(0u, 0u, 0u, 0u);
            w[1][p] = left > 0 ? cut(load_stream(high + k + 64 * p), left) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
}

// Eight tokens' elements of a step: [piece][16-byte parts of a lane's elements of its token's row].  `left`: bytes of the row
// from here on.
template <bool W8>
struct Tokens {
    static constexpr int PARTS = W8 ? 2 : 1;
    uint4 v[2][PARTS];
    __device__ __forceinline__ void load(const uint8_t* row, int left) {
        const int k = (threadIdx.x & 3) * (16 * PARTS);
        if (left >= 2 * 64 * PARTS) {
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int q = 0; q < PARTS; ++q) v[p][q] = *reinterpret_cast<const uint4*>(row + k + 64 * PARTS * p + 16 * q);
        } else {
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
                    const int at = k + 64 * PARTS * p + 16 * q;
                    v[p][q] = at < left ? *reinterpret_cast<const uint4*>(row + at) : make_uint4(0u, 0u, 0u, 0u);
                }
        }
    }
};

// sums[n][4] += a tile's products with the tokens 8 n .. + 7: rows g (elements 0, 1) and g + 8 (2, 3) by tokens 2 t and 2 t + 1
template <bool W8, int COLS>
__device__ __forceinline__ void multiply(float (&sums)[COLS][4], const uint4 (&w)[2][2], const Tokens<W8> (&x)[COLS]) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const uint32_t low[4] = {w[0][p].x, w[0][p].y, w[0][p].z, w[0][p].w}, high[4] = {w[1][p].x, w[1][p].y, w[1][p].z, w[1][p].w};
#pragma unroll
        for (int j = 0; j < (W8 ? 4 : 2); ++j) {
            uint32_t a[4];
            if constexpr (W8) {
                widen(low[j], a[0], a[2]);
                widen(high[j], a[1], a[3]);
            } else {
                a[0] = low[2 * j];
                a[1] = high[2 * j];
                a[2] = low[2 * j + 1];
                a[3] = high[2 * j + 1];
            }
#pragma unroll
            for (int n = 0; n < COLS; ++n) {
                const uint4 v = x[n].v[p][W8 ? j / 2 : 0];
                const uint32_t b0 = j % 2 ? v.z : v.x, b1 = j % 2 ? v.w : v.y;
                if constexpr (W8) mma_f16(sums[n], a, b0, b1);
                else mma16::mma_bf16(sums[n], a, b0, b1);
            }
        }
    }
}

// What a block's products are multiplied by (e4m3): the scales of rows g and g + 8 and of tokens 2 t and 2 t + 1 (0: a token that
// did not choose the expert; a block's scale is 2^-126 at least)
template <int COLS>
struct Factors {
    float row[2], token[COLS][2];
};

// The same with a block's sums scaled before they are added (e4m3)
template <bool W8, int COLS>
__device__ __forceinline__ void accumulate(float (&acc)[COLS][4], const uint4 (&w)[2][2], const Tokens<W8> (&x)[COLS], const Factors<COLS>& f) {
    if constexpr (W8) {
        float part[COLS][4];
#pragma unroll
        for (int n = 0; n < COLS; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) part[n][j] = 0.0f;
        multiply<W8, COLS>(part, w, x);
#pragma unroll
        for (int n = 0; n < COLS; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[n][j] = f.token[n][j % 2] != 0.0f ? fmaf(part[n][j], f.row[j / 2] * f.token[n][j % 2], acc[n][j]) : acc[n][j];
    } else {
        multiply<W8, COLS>(acc, w, x);
    }
}

struct alignas(16) Shared {
    float4 part[WARPS][NT][MAX_T / 8][32];   // a warp's sums of a tile as the lanes have them
    uint4 zeros[16];                         // what a token that did not choose an expert has there
    float weight[MAX_T * MAX_K];             // by (token, choice)
    int chosen[MAX_T * MAX_K];
    unsigned users[MAX_E];                   // tokens that chose an expert
    int slot[MAX_E];
    int expert[MAX_T * MAX_K];               // the chosen experts in ascending order
    unsigned mask[MAX_T * MAX_K];            // their tokens
    int first[MAX_T * MAX_K];                // where their tokens' weights begin in
    float factor[MAX_T * MAX_K];             // [slot][its tokens in order]
    int2 count[MAX_E / 32];                  // of 32 experts: chosen ones, and their tokens together
    int2 unit[WARPS][NT];                    // [team][tile]: (slot, unit) of a team's units
    int active;
    int go;
};
static_assert(sizeof(Shared) % 16 == 0, "rows of 16-byte pieces lie behind it");

// A float as a number in its order, the two zeros equal; NaN lowest
__device__ __forceinline__ uint32_t order(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);          // (-0 + 0 = 0)
    return v == v ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}

// Token t's choices by a warp, as the router kernels choose (the lowest index among equals).  A NaN among a token's logits makes
// its weights NaN.  (Code that runs once waits for its instructions: it is short, and its loops are loops.)
__device__ __forceinline__ void choose(const Params& p, Shared& sm, uint32_t* rest, int t) {
    const int lane = threadIdx.x & 31;
    const float* z = p.z + (size_t)t * p.E;
    auto score = [&](int e) {
        const float v = z[e] + (p.bias ? p.bias[e] : 0.0f);
        return p.softmax ? v : 1.0f / (1.0f + expf(-v));
    };
    bool broken = false;
    int mine = 0;                                          // lane j keeps the j-th choice
    // The largest of all lanes' `best`, and the lowest of the experts that have it; nothing but NaN left: any, but a valid one
    auto pick = [&](int j, uint32_t best, int at) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        at = (int)__reduce_min_sync(0xffffffffu, best == top && best ? (unsigned)at : (unsigned)p.E);
        if (at >= p.E) at = j;
        if (lane == j) mine = at;
        return at;
    };
    if (p.E <= IN_REGISTERS) {                             // four a lane
        uint32_t key[4];
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = lane + 32 * i < p.E ? score(lane + 32 * i) : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            broken |= s[i] != s[i];
            key[i] = lane + 32 * i < p.E ? order(p.correction ? s[i] + p.correction[lane + 32 * i] : s[i]) : 0u;
        }
#pragma unroll 1
        for (int j = 0; j < p.k; ++j) {
            uint32_t best = key[0];
            int at = lane;
#pragma unroll
            for (int i = 1; i < 4; ++i)
                if (key[i] > best) { best = key[i]; at = lane + 32 * i; }      // the first of equals
            at = pick(j, best, at);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (at == lane + 32 * i) key[i] = 0u;
        }
    } else {
#pragma unroll 4
        for (int e = lane; e < p.E; e += 32) {
            const float s = score(e);
            broken |= s != s;
            rest[e] = order(p.correction ? s + p.correction[e] : s);
        }
#pragma unroll 1
        for (int j = 0; j < p.k; ++j) {
            uint32_t best = 0;
            int at = p.E;
#pragma unroll 4
            for (int e = lane; e < p.E; e += 32)
                if (rest[e] > best) { best = rest[e]; at = e; }
            at = pick(j, best, at);
            if (at % 32 == lane) rest[at] = 0u;
        }
    }
    broken = __any_sync(0xffffffffu, broken);
    float s = 0.0f;
    if (lane < p.k) {
        s = score(mine);
        atomicOr(&sm.users[mine], 1u << t);
        sm.chosen[t * p.k + lane] = mine;
    }
    if (p.softmax) {                                       // (with a correction any of the chosen may have the largest logit)
        const float top = warp_max(lane < p.k ? s : -INFINITY);
        s = lane < p.k ? expf(s - top) : 0.0f;
    }
    const float total = warp_sum(s);
    if (lane < p.k) sm.weight[t * p.k + lane] = broken ? __int_as_float(0x7fc00000) : s * (p.softmax || p.renormalize ? p.scale / total : p.scale);
}

// Bytes of shared memory for the scores of the choice (up to 128 experts: registers hold them)
constexpr int scores_bytes(int T, int E) { return E <= IN_REGISTERS ? 0 : (T * E * 4 + 15) / 16 * 16; }

// A barrier of `threads` threads of the CTA, a multiple of 32
__device__ __forceinline__ void named_barrier(int id, int threads) {
    if (threads == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Every thread of the grid behind every other's stores.  False: gave up.
__device__ __forceinline__ bool grid_barrier(int* counter, int* go, uint32_t polls) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        atomicAdd(counter, 1);
        int seen = 0;
        for (uint32_t i = 0; i < polls && !seen; ++i) {
            int v;
            asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
            seen = v >= (int)gridDim.x;
        }
        *go = seen;
    }
    __syncthreads();
    return *go != 0;
}

template <bool W8, int COLS>
__global__ void __launch_bounds__(THREADS, 1)
moe_few_kernel(const Params p) {
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& sm = *reinterpret_cast<Shared*>(smem);
    uint32_t* const rest = reinterpret_cast<uint32_t*>(smem + sizeof(Shared));      // [T, E], or nothing
    constexpr int SIZE = W8 ? 1 : 2;                                      // bytes of a weight
    constexpr int X_STEP = W8 ? 2 * STEP : STEP;                          // bytes of a step of a token's row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    for (int e = threadIdx.x; e < p.E; e += THREADS) sm.users[e] = 0;
    if (threadIdx.x < 16) sm.zeros[threadIdx.x] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    pdl_wait();
    // ---- who goes where (every CTA for itself) ------------------------------------------------
    if (warp < p.T) choose(p, sm, rest + warp * p.E, warp);
    __syncthreads();
    // the chosen experts in ascending order: a warp counts 32 experts, and those in front of them
    const int chunks = (p.E + 31) / 32;
#pragma unroll 1
    for (int i = warp; i < chunks; i += WARPS) {
        const int e = i * 32 + lane;
        const unsigned users = e < p.E ? sm.users[e] : 0u;
        const unsigned any = __ballot_sync(0xffffffffu, users != 0), pairs = __reduce_add_sync(0xffffffffu, __popc(users));
        if (lane == 0) sm.count[i] = make_int2(__popc(any), (int)pairs);
    }
    __syncthreads();
#pragma unroll 1
    for (int i = warp; i < chunks; i += WARPS) {
        const int e = i * 32 + lane;
        const unsigned users = e < p.E ? sm.users[e] : 0u, any = __ballot_sync(0xffffffffu, users != 0);
        const int2 here = lane < i ? sm.count[lane] : make_int2(0, 0);
        const int n = (int)__reduce_add_sync(0xffffffffu, (unsigned)here.x), before = (int)__reduce_add_sync(0xffffffffu, (unsigned)here.y);
        int incl = __popc(users);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (users) {
            const int s = n + __popc(any & ((1u << lane) - 1));
            sm.slot[e] = s;
            sm.expert[s] = e;
            sm.mask[s] = users;
            sm.first[s] = before + incl - __popc(users);
        }
        if (lane == 0 && i + 1 == chunks) sm.active = n + __popc(any);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.T * p.k; i += THREADS) {
        const int a = sm.slot[sm.chosen[i]], t = i / p.k;
        sm.factor[sm.first[a] + __popc(sm.mask[a] & ((1u << t) - 1))] = sm.weight[i];
    }
    __syncthreads();
    const int active = sm.active;

    uint4 w[NT][2][2];                                                    // the step that is on its way
    float acc[NT][COLS][4];
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int n = 0; n < COLS; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][n][j] = 0.0f;
    };
    auto leave = [&]() {                                                  // this warp's sums for the others to add
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int n = 0; n < COLS; ++n) sm.part[warp][i][n][lane] = make_float4(acc[i][n][0], acc[i][n][1], acc[i][n][2], acc[i][n][3]);
    };
    auto joined = [&](int from, int warps, int i, int n, int l) {         // the warps' sums together
        float4 v = sm.part[from][i][n][l];
        for (int q = 1; q < warps; ++q) {
            const float4 o = sm.part[from + q][i][n][l];
            v.x += o.x;
            v.y += o.y;
            v.z += o.z;
            v.w += o.w;
        }
        return v;
    };

    // ---- act: units of eight gate rows and their up rows, dealt out over the teams, up to NT units at a time ------------
    {
        const int per = (p.I + 7) / 8, NB = (2 * p.I + fp8::BLOCK - 1) / fp8::BLOCK, KB = (p.H + fp8::BLOCK - 1) / fp8::BLOCK;
        const int len = p.H * SIZE, steps = (len + STEP - 1) / STEP;
        const long long units = (long long)active * per;
        const int team = p.team;
        const int me = warp % team, my_team = warp / team, teams = gridDim.x * (WARPS / team), index = blockIdx.x * (WARPS / team) + my_team;
        const int u_begin = (int)(units * index / teams), u_end = (int)(units * (index + 1) / teams);
        const uint8_t* x_row[COLS];                                       // (a token there is not has another's row: it is dropped)
        const float* x_scale[COLS];
#pragma unroll
        for (int n = 0; n < COLS; ++n) {
            x_row[n] = p.x + min(8 * n + g, p.T - 1) * p.ldx;
            x_scale[n] = p.x_scale + min(8 * n + 2 * t4, p.T - 1) * KB;
        }
        const int odd[2] = {2 * t4 + 1 < p.T ? KB : 0, 8 + 2 * t4 + 1 < p.T ? KB : 0};
        const size_t to_up = (size_t)p.I * p.ldg;
        // the units of a group: slot, column, this lane's gate row (the up row lies to_up bytes on) and both rows' scales
        struct Unit {
            const uint8_t* gate;
            int slot, unit;
            unsigned scale[2];
        } next[NT];
        int a = u_begin / per, c = u_begin - a * per, next_tiles = 0;     // of the first unit behind the groups looked up
        auto look_up = [&](int u) {
            next_tiles = min(NT, u_end - u);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int e = sm.expert[a], r = min(c * 8 + g, p.I - 1);
                next[j].slot = a;
                next[j].unit = c;
                next[j].gate = static_cast<const uint8_t*>(p.gate_up) + (unsigned long long)(unsigned)(e * 2 * p.I + r) * (unsigned)p.ldg;
                if constexpr (W8) {
                    next[j].scale[0] = (unsigned)(e * NB + r / fp8::BLOCK) * (unsigned)KB;
                    next[j].scale[1] = (unsigned)(e * NB + (p.I + r) / fp8::BLOCK) * (unsigned)KB;
                }
                if (u + j + 1 < u_end && j < next_tiles && ++c == per) {
                    c = 0;
                    ++a;
                }
            }
        };
        auto fetch_at = [&](int at) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
                if (j < next_tiles) fetch(w[j], next[j].gate, next[j].gate + to_up, at, len);
        };
        if (u_begin < u_end) {
            look_up(u_begin);
            fetch_at(me * STEP);                                          // (a team has at most a quarter as many warps as steps)
        }
        for (int u = u_begin; u < u_end; u += NT) {
            clear();
            const int tiles = next_tiles;
            Unit now[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) now[j] = next[j];
            for (int s = me; s < steps; s += team) {
                Tokens<W8> xs[COLS];
                Factors<COLS> f[NT];
#pragma unroll
                for (int n = 0; n < COLS; ++n) xs[n].load(x_row[n] + s * X_STEP, p.ldx - s * X_STEP);
                if constexpr (W8) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        f[j].row[0] = p.gate_up_scale[now[j].scale[0] + s];
                        f[j].row[1] = p.gate_up_scale[now[j].scale[1] + s];
#pragma unroll
                        for (int n = 0; n < COLS; ++n) {
                            f[j].token[n][0] = x_scale[n][s];
                            f[j].token[n][1] = x_scale[n][s + odd[n]];
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    if (j < tiles) accumulate<W8, COLS>(acc[j], w[j], xs, f[j]);
                if (s + team < steps) {
                    fetch_at((s + team) * STEP);
                } else if (u + NT < u_end) {
                    look_up(u + NT);
                    fetch_at(me * STEP);
                }
            }
            named_barrier(1 + my_team, team * 32);                        // the sums before these are added by now
            if (me == 0 && lane == 0) {
#pragma unroll
                for (int j = 0; j < NT; ++j) sm.unit[my_team][j] = j < tiles ? make_int2(now[j].slot, now[j].unit) : make_int2(-1, 0);
            }
            leave();
            named_barrier(1 + my_team, team * 32);
            for (int o = me * 32 + lane; o < NT * COLS * 32; o += team * 32) {
                const int j = o / (COLS * 32), n = o / 32 % COLS, l = o % 32;
                const int2 unit = sm.unit[my_team][j];
                const int col = unit.y * 8 + l / 4;
                if (unit.x < 0 || col >= p.I) continue;
                const float4 v = joined(my_team * team, team, j, n, l);
                const unsigned m = sm.mask[unit.x];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int t = 8 * n + 2 * (l % 4) + i;
                    if (!(m >> t & 1)) continue;
                    float gv = i ? v.y : v.x, uv = i ? v.w : v.z;
                    const float weight = sm.factor[sm.first[unit.x] + __popc(m & ((1u << t) - 1))];
                    if (p.on_input) { gv *= weight; uv *= weight; }
                    float h = gv / (1.0f + expf(-gv)) * uv;
                    if (!p.on_input) h *= weight;
                    const size_t at = ((size_t)unit.x * p.T + t) * p.Ip + col;
                    if constexpr (W8) static_cast<float*>(p.act)[at] = h;
                    else {
                        const bf16 high = __float2bfloat16_rn(h);
                        const float v = __bfloat162float(high);
                        static_cast<bf16*>(p.act)[at] = high;
                        p.act_low[at] = __float2bfloat16_rn(fabsf(v) < INFINITY ? h - v : 0.0f);
                    }
                }
            }
        }
    }

    // ---- y: rows of the down matrices, dealt out over the grid, sixteen or thirty-two at a time; the sum runs over the blocks
    // of K of all chosen experts.  The first weights are asked for ahead of the barrier. -----------------------------------
    const int NB = (p.H + fp8::BLOCK - 1) / fp8::BLOCK, KB = (p.I + fp8::BLOCK - 1) / fp8::BLOCK;
    const int r_begin = (int)((long long)p.H * blockIdx.x / gridDim.x), r_end = (int)((long long)p.H * (blockIdx.x + 1) / gridDim.x);
    const int len = p.I * SIZE, per = (len + STEP - 1) / STEP, items = active * per;
    // A step of a warp is two tiles of one block, or one tile of two blocks where that is all there is: a block in a row of
    // K is an item (slot, block), and the items go round the warps
    struct Item {
        int slot, block;
    };
    int r0 = r_begin;                                                     // first row of the group on its way
    bool two = false;                                                     // whether it has two tiles
    Item item[2];                                                         // what is on its way (two tiles: one)
    int at = 0;                                                           // items of this warp before it
    auto item_of = [&](int i) {
        Item r;
        r.slot = i / per;
        r.block = i - r.slot * per;
        return r;
    };
    auto down_row = [&](int slot, int r) {
        return static_cast<const uint8_t*>(p.down) + ((size_t)sm.expert[slot] * p.H + min(r, r_end - 1)) * p.ldd;
    };
    auto fetch_items = [&]() {                                            // from `at` on
        if (two) {
            const int i = at * WARPS + warp;
            if (i >= items) return;
            item[0] = item_of(i);
            fetch(w[0], down_row(item[0].slot, r0 + g), down_row(item[0].slot, r0 + 8 + g), item[0].block * STEP, len);
            fetch(w[1], down_row(item[0].slot, r0 + 16 + g), down_row(item[0].slot, r0 + 24 + g), item[0].block * STEP, len);
        } else {
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                const int i = (at + f) * WARPS + warp;
                item[f].slot = -1;
                if (i >= items) continue;
                item[f] = item_of(i);
                fetch(w[f], down_row(item[f].slot, r0 + g), down_row(item[f].slot, r0 + 8 + g), item[f].block * STEP, len);
            }
        }
    };
    if (r_begin < r_end) {
        two = r_end - r0 > 16;
        fetch_items();
    }
    bool met = grid_barrier(p.barrier, &sm.go, p.polls);
    if constexpr (W8) {
        // act in float16, a warp a (slot, token, block)
        if (met) {
            for (int i = blockIdx.x * WARPS + warp; i < active * p.T * KB; i += gridDim.x * WARPS) {
                const int r = i / KB, b = i - r * KB, slot = r / p.T, t = r - slot * p.T;
                if (!(sm.mask[slot] >> t & 1)) continue;
                const int col = b * fp8::BLOCK + lane * 4;
                const float* src = static_cast<const float*>(p.act) + (size_t)r * p.Ip + col;
                float v[4];
                uint32_t m = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] = col + j < p.I ? src[j] : 0.0f;
                    m = max(m, fp8::abs_bits(v[j]));
                }
                const float s = half_scale(__reduce_max_sync(0xffffffffu, m));
                *reinterpret_cast<uint2*>(p.act16 + (size_t)r * p.Ip + col) = halves(v, s);
                if (lane == 0) p.act_scale[(size_t)r * KB + b] = s;
            }
            met = grid_barrier(p.barrier + 1, &sm.go, p.polls);
        }
    }
    if (!met) {
        if (threadIdx.x == 0) atomicExch(p.status, 19);
        return;
    }
    const uint8_t* const act = W8 ? reinterpret_cast<const uint8_t*>(p.act16) : static_cast<const uint8_t*>(p.act);
    // the tokens' elements of an item, and what its products are multiplied by in the rows from r on
    auto tokens_of = [&](Tokens<W8> (&xs)[COLS], const uint8_t* act, const Item& i) {
        const unsigned m = sm.mask[i.slot];
#pragma unroll
        for (int n = 0; n < COLS; ++n) {
            const int t = 8 * n + g;
            const bool in = m >> t & 1;
            xs[n].load(in ? act + ((size_t)i.slot * p.T + t) * 2 * p.Ip + i.block * X_STEP : reinterpret_cast<const uint8_t*>(sm.zeros),
                       W8 ? X_STEP : in ? len - i.block * X_STEP : X_STEP);
        }
    };
    auto factors_of = [&](Factors<COLS>& f, const Item& i, int r) {
        if constexpr (W8) {
            const unsigned m = sm.mask[i.slot], e = sm.expert[i.slot] * NB;
            f.row[0] = p.down_scale[(e + (unsigned)min(r + g, p.H - 1) / fp8::BLOCK) * (unsigned)KB + i.block];
            f.row[1] = p.down_scale[(e + (unsigned)min(r + 8 + g, p.H - 1) / fp8::BLOCK) * (unsigned)KB + i.block];
#pragma unroll
            for (int n = 0; n < COLS; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int t = 8 * n + 2 * t4 + j;
                    f.token[n][j] = m >> t & 1 ? p.act_scale[(unsigned)(i.slot * p.T + t) * (unsigned)KB + i.block] : 0.0f;
                }
        }
    };
    const uint8_t* const low = reinterpret_cast<const uint8_t*>(p.act_low);
    auto add = [&](float (&sums)[COLS][4], const uint4 (&tile)[2][2], const Tokens<W8> (&xs)[COLS], const Tokens<W8> (&rest)[COLS], const Factors<COLS>& f,
                   const Item& item) {
        if constexpr (W8) {
            accumulate<W8, COLS>(sums, tile, xs, f);
        } else {
            float next[COLS][4];
#pragma unroll
            for (int n = 0; n < COLS; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) next[n][j] = sums[n][j];
            multiply<W8, COLS>(next, tile, xs);
            multiply<W8, COLS>(next, tile, rest);
            const unsigned m = sm.mask[item.slot] >> (2 * t4);
#pragma unroll
            for (int n = 0; n < COLS; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) sums[n][j] = m >> (8 * n + j % 2) & 1 ? next[n][j] : sums[n][j];
        }
    };
    for (int r = r_begin, rows; r < r_end; r += rows) {
        const bool pair = two;
        rows = pair ? 32 : 16;
        clear();
        for (at = 0; at * WARPS + warp < items;) {
            Tokens<W8> xs[COLS], rest[COLS];                              // (rest: bf16 weights)
            Factors<COLS> f;
            const Item first = item[0], second = item[1];
            tokens_of(xs, act, first);
            if constexpr (!W8) tokens_of(rest, low, first);
            factors_of(f, first, r);
            if (pair) {
                add(acc[0], w[0], xs, rest, f, first);
                if constexpr (W8) {
                    f.row[0] = p.down_scale[((unsigned)sm.expert[first.slot] * NB + (unsigned)min(r + 16 + g, p.H - 1) / fp8::BLOCK) * (unsigned)KB + first.block];
                    f.row[1] = p.down_scale[((unsigned)sm.expert[first.slot] * NB + (unsigned)min(r + 24 + g, p.H - 1) / fp8::BLOCK) * (unsigned)KB + first.block];
                }
                add(acc[1], w[1], xs, rest, f, first);
                ++at;
            } else {
                add(acc[0], w[0], xs, rest, f, first);
                if (second.slot >= 0) {
                    tokens_of(xs, act, second);
                    if constexpr (!W8) tokens_of(rest, low, second);
                    factors_of(f, second, r);
                    add(acc[0], w[1], xs, rest, f, second);
                }
                at += 2;
            }
            if (at * WARPS + warp < items) fetch_items();
        }
        // the next group's first weights are on their way while these sums are joined
        if (r + rows < r_end) {
            r0 = r + rows;
            two = r_end - r0 > 16;
            at = 0;
            fetch_items();
        }
        if (r > r_begin) __syncthreads();                                 // the sums before these are added by now
        leave();
        __syncthreads();
        if (threadIdx.x < NT * COLS * 32) {
            const int j = threadIdx.x / (COLS * 32), n = threadIdx.x / 32 % COLS, l = threadIdx.x % 32;
            if (j == 0 || pair) {
                const float4 v = joined(0, WARPS, j, n, l);
                const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = r + 16 * j + l / 4 + 8 * (i / 2), t = 8 * n + 2 * (l % 4) + i % 2;
                    if (row >= r_end || t >= p.T) continue;
                    const size_t to = (size_t)t * p.H + row;
                    const float y = p.add ? x[i] + p.add[to] : x[i];
                    if (p.out_bf16) static_cast<bf16*>(p.out)[to] = __float2bfloat16_rn(y);
                    else static_cast<float*>(p.out)[to] = y;
                }
            }
        }
    }
}

// The shared memory that a kernel may take, set once a device to what its largest call takes: the limit belongs to the
// function, and calls of several sizes may be on their way from several threads
template <typename K>
bool allow_shared(K kernel, bool (&done)[64]) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= 64) return false;
    if (!done[device])
        done[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            (int)sizeof(Shared) + scores_bytes(MAX_T, MAX_E)) == cudaSuccess;
    return done[device];
}

template <bool W8, int COLS>
int launch(Params& p, int sms, cudaStream_t stream) {
    const auto kernel = moe_few_kernel<W8, COLS>;
    static bool done[64];
    if (!allow_shared(kernel, done)) return SHARPI_LAUNCH_FAILED;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = sms;
    cfg.blockDim = THREADS;
    cfg.dynamicSmemBytes = sizeof(Shared) + scores_bytes(p.T, p.E);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = sharpi_pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? SHARPI_OK : SHARPI_LAUNCH_FAILED;
}

uint32_t test_polls = BARRIER_LIMIT;

}  // namespace

// Test hook: the waits of the NEXT launch poll `polls` times at most (0: every block gives up at once, writes the code and
// returns).
SHARPI_API void sharpi_moe_few_set_wait_test(unsigned polls) { test_polls = polls; }

// h bf16 [T, H] rows ldh elements apart (bf16 weights: ldh a multiple of 8, 16-byte alignment), x: what the router reads,
// float32 or bfloat16 [T, ldx]; weights bf16, or e4m3 with scales; rows ldg / ldd bytes apart; work: 16-byte aligned.
SHARPI_API int sharpi_moe_few(const void* x, int x_dtype, int ldx, const void* h, int ldh, const float* router, const float* bias,
                              const float* correction, const void* gate_up, long long ldg, const float* gate_up_scale,
                              const void* down, long long ldd, const float* down_scale, const float* add, void* work, int* status,
                              void* out, int out_bf16, int T, int E, int k, int H, int I, int softmax, int renormalize, float scale,
                              int on_input, int sms, cudaStream_t stream) {
    if (T <= 0) return SHARPI_OK;
    if (T > MAX_T || E <= 0 || E > MAX_E || k <= 0 || k > MAX_K || k > E || H <= 0 || I <= 0 || sms <= 0 || 2LL * E * I > 0x7fffffff ||
        (gate_up_scale == nullptr) != (down_scale == nullptr) || ldh < H || (x_dtype != SHARPI_F32 && x_dtype != SHARPI_BF16))
        return SHARPI_BAD_ARGUMENT;
    const bool w8 = gate_up_scale != nullptr;
    if (((reinterpret_cast<uintptr_t>(gate_up) | reinterpret_cast<uintptr_t>(down) | reinterpret_cast<uintptr_t>(work)) & 15) ||
        ldg % 16 || ldd % 16 || (!w8 && (ldh % 8 || H % 8 || I % 8 || (reinterpret_cast<uintptr_t>(h) & 15))) || (w8 && I % 2))
        return SHARPI_UNALIGNED;
    const long long slots = (long long)T * k < E ? (long long)T * k : E;
    const int Ip = (I + 127) / 128 * 128, KB = (H + 127) / 128;
    uint8_t* at = static_cast<uint8_t*>(work);
    auto take = [&](long long bytes) {
        uint8_t* r = at;
        at += (bytes + 15) / 16 * 16;
        return r;
    };
    Params p = {};
    p.barrier = reinterpret_cast<int*>(take(8));
    float* z = reinterpret_cast<float*>(take(4LL * T * E));
    p.act = take(slots * T * Ip * (w8 ? 4 : 2));
    __half* rows16 = nullptr;
    float* x_scale = nullptr;
    if (!w8) p.act_low = reinterpret_cast<bf16*>(take(slots * T * Ip * 2));
    if (w8) {
        p.act16 = reinterpret_cast<__half*>(take(slots * T * Ip * 2));
        p.act_scale = reinterpret_cast<float*>(take(slots * T * (Ip / 128) * 4));
        rows16 = reinterpret_cast<__half*>(take(2LL * T * KB * 128));
        x_scale = reinterpret_cast<float*>(take(4LL * T * KB));
    }
    p.z = z; p.bias = bias; p.correction = correction;
    p.x = w8 ? reinterpret_cast<const uint8_t*>(rows16) : static_cast<const uint8_t*>(h);
    p.ldx = w8 ? KB * 256 : ldh * 2;
    p.x_scale = x_scale;
    const int vec = H % 4 == 0 && ldx % 4 == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(router)) & 15) == 0;
    const int blocks = (int)(((long long)T * (E + (w8 ? KB : 0)) + 3) / 4);
    const bf16* rows = static_cast<const bf16*>(h);
    if (x_dtype == SHARPI_F32)
        SHARPI_LAUNCH_PDL(moe_few_router_kernel<float>, blocks, 128, 0, stream, static_cast<const float*>(x), ldx, router, T, H, E, vec, z,
                          p.barrier, rows, ldh, rows16, w8 ? KB * 128 : 0, x_scale);
    else
        SHARPI_LAUNCH_PDL(moe_few_router_kernel<bf16>, blocks, 128, 0, stream, static_cast<const bf16*>(x), ldx, router, T, H, E, vec, z,
                          p.barrier, rows, ldh, rows16, w8 ? KB * 128 : 0, x_scale);
    p.gate_up = gate_up; p.down = down; p.gate_up_scale = gate_up_scale; p.down_scale = down_scale;
    p.add = add; p.out = out; p.status = status;
    p.ldg = ldg; p.ldd = ldd;
    p.T = T; p.E = E; p.k = k; p.H = H; p.I = I; p.Ip = Ip;
    p.polls = test_polls;
    test_polls = BARRIER_LIMIT;
    p.softmax = softmax; p.renormalize = renormalize; p.on_input = on_input; p.out_bf16 = out_bf16; p.scale = scale;
    // As many warps a team as leave each of them four steps of a row's K, so that joining their sums stays a small part; where the
    // teams then have 20 units and more, whose count no longer has to come out even, half as many.  Four steps against eight: 1 to
    // 4 tokens, 2 of 8 experts of 2048 x 768, e4m3 15.6 to 19.4 us against 18.8 to 22.2; 12 tokens, 6 of 64 experts of 4096 x 1024,
    // e4m3 186 against 176.
    const int steps = (H * (w8 ? 1 : 2) + STEP - 1) / STEP;
    p.team = 1;
    while (p.team < WARPS && p.team * 8 <= steps) p.team *= 2;
    if (p.team > 1 && slots * ((I + 7) / 8) >= 20LL * sms * (WARPS / p.team)) p.team /= 2;
    const bool wide = T > 8;
    return w8 ? (wide ? launch<true, 2>(p, sms, stream) : launch<true, 1>(p, sms, stream))
              : (wide ? launch<false, 2>(p, sms, stream) : launch<false, 1>(p, sms, stream));
}
