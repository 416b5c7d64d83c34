// A whole mixture-of-experts layer for up to 16 tokens in two kernels:
//
//   router    z = h Wr^T (float32), a warp a (token, expert)
//   experts   every token's k experts and their weights from z; act = silu(g) * u over the gate|up rows of the experts that
//             any token chose; a barrier over the grid; y[t] = add[t] + sum over the token's experts of w Wd act
//
// With few tokens the layer is a stream of the chosen experts' weights, so the second kernel is laid out for that alone: one
// CTA an SM, weight rows dealt out evenly over the warps whatever expert they belong to, each weight read once, in 16-byte
// pieces straight into registers.  Teams of 1 to 16 warps share K in turn (the more K has, the more); a warp asks for its next
// step of up to 4 KB when it has multiplied the last (up to 64 KB an SM in flight; reading at 6.4 TB/s with a microsecond of
// latency takes 44 KB).  All tokens are the 16-row operand of the MMA against tiles of eight weight rows; a row of a token that did not choose the expert is computed and dropped (gate|up) or
// zero (down).  Because the down product is linear, a token's experts are one long sum over (expert, inner element): act is
// multiplied by the router's weight before (weights on the output).  The warps' parts are added in warp order: a call's result
// is the same every time, but the order (float32 rounding) of a token's sum goes by which experts the whole call reaches.
//
// bfloat16 weights: mma.sync m16n8k16, act rounded to bfloat16 (2^-9 of its value) as in the other bfloat16 mixtures.
//
// e4m3 weights with a scale for 128 x 128 (fp8.cuh): an e4m3 value is a float16 one (cvt, two an instruction), and the MMA is
// m16n8k16 on float16.  (mma.sync on e4m3 is no instruction of this GPU's: it converts both operands for every tile, 1000
// instructions a step of 4 KB where this takes 250.)  The activations are float16 times a power of two s for 128 neighbours such
// that |x / s| < 2^15: of h's eight bits none is lost down to 2^-32 of its block's largest value, act is off by 2^-12 of its
// value.  A block's 128 products are added in float32, then scaled and added.  Infinities and NaN make a block's scale NaN.
//
// The barrier needs all CTAs on the GPU at once: the launch is cooperative.  Its counters lie in the call's own workspace and
// are set to zero by the router kernel.  The wait is bounded; on a timeout the kernel sets *status and returns.
#include "fp8.cuh"
#include "mma_sync.cuh"

namespace {

constexpr int MAX_T = 16, MAX_K = 32, MAX_E = 1024;
constexpr int WARPS = 16, THREADS = 32 * WARPS;
constexpr int NT = 4;                          // tiles of eight weight rows that a warp has at a time
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
    __half* act16;                // e4m3: act / act_scale [active, T, Ip]
    float* act_scale;             // e4m3: [active, T, blocks of I]
    void* out;                    // [T, H]
    int* barrier;                 // two counters
    int* status;
    long long ldg, ldd;           // bytes
    int ldx, T, E, k, H, I, Ip;   // Ip: I rounded up to 128
    int softmax, renormalize, on_input, out_bf16, staged;      // staged: the rows x fit into shared memory
    int team;                     // warps that share the K of gate and up rows
    float scale;
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
#pragma unroll 8
        for (int i = 4 * lane; i < H; i += 128) {
            const float4 wv = *reinterpret_cast<const float4*>(w + i);
            float xv[4];
            if constexpr (sizeof(T) == 4) {
                const float4 q = *reinterpret_cast<const float4*>(x + i);
                xv[0] = q.x; xv[1] = q.y; xv[2] = q.z; xv[3] = q.w;
            } else {
                const uint2 q = *reinterpret_cast<const uint2*>(x + i);
                xv[0] = __uint_as_float(q.x << 16); xv[1] = __uint_as_float(q.x & 0xffff0000u);
                xv[2] = __uint_as_float(q.y << 16); xv[3] = __uint_as_float(q.y & 0xffff0000u);
            }
            acc[0] = fmaf(xv[0], wv.x, acc[0]);
            acc[1] = fmaf(xv[1], wv.y, acc[1]);
            acc[2] = fmaf(xv[2], wv.z, acc[2]);
            acc[3] = fmaf(xv[3], wv.w, acc[3]);
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

// How a step of a warp reads K: a lane has 16 bytes of a weight row in each of two pieces; lanes 4 g + t of a row lie side
// by side.  Which elements of K share an MMA is free as long as both operands agree: lane t's elements are its k values.
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

// The weights of a step of a warp; `row`: this lane's row of every tile (where a tile has none, any row: its sums are
// dropped), `tiles` of which are read; `len`: bytes of a row.
__device__ __forceinline__ void fetch(uint4 (&w)[NT][2], const uint8_t* const (&row)[NT], int tiles, int at, int len) {
    const int k = at + (threadIdx.x & 3) * 16;
    if (at + STEP <= len) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
            if (i < tiles) {
                w[i][0] = load_stream(row[i] + k);
                w[i][1] = load_stream(row[i] + k + 64);
            }
    } else {                                                              // behind the end: zeros, whatever lies between rows
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int left = len - (k + 64 * p);
                w[i][p] = i < tiles && left > 0 ? cut(load_stream(row[i] + k + 64 * p), left) : make_uint4(0u, 0u, 0u, 0u);
            }
    }
}

// acc += the step's products.  lo / hi: this lane's token row (and the row eight below) at the step's first element, null:
// zeros; e4m3: `f_lo`, `f_hi`: scales of the token rows' block, scale[i]: of the block of this lane's two sums of tile i.
// left: bytes from the step's first to the end of the (zero-padded) token rows.
template <bool W8, bool WIDE>
__device__ __forceinline__ void multiply(float (&acc)[NT][4], const uint4 (&w)[NT][2], int tiles, const uint8_t* lo, const uint8_t* hi, int left,
                                         float f_lo, float f_hi, const float (&scale)[NT]) {
    constexpr int PARTS = W8 ? 2 : 1;                                     // 16-byte parts of a lane's elements of a token row
    const int k = (threadIdx.x & 3) * (16 * PARTS);
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    float part[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][j] = W8 ? 0.0f : acc[i][j];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int at = k + p * 64 * PARTS;
        const bool in = at < left;
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
            const uint4 l = lo && in ? *reinterpret_cast<const uint4*>(lo + at + 16 * q) : zero;
            const uint4 h = WIDE && hi && in ? *reinterpret_cast<const uint4*>(hi + at + 16 * q) : zero;
            const uint32_t a0[4] = {l.x, h.x, l.y, h.y}, a1[4] = {l.z, h.z, l.w, h.w};
            // the tiles in turn: a product that adds to what the one before it left waits for that
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t (&a)[4] = j ? a1 : a0;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    if (i >= tiles) continue;
                    if constexpr (W8) {
                        const uint32_t word = q ? (j ? w[i][p].w : w[i][p].z) : (j ? w[i][p].y : w[i][p].x);
                        uint32_t b0, b1;
                        widen(word, b0, b1);
                        mma_f16(part[i], a, b0, b1);
                    } else {
                        mma16::mma_bf16(part[i], a, j ? w[i][p].z : w[i][p].x, j ? w[i][p].w : w[i][p].y);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const float s_lo = scale[i] * f_lo, s_hi = scale[i] * f_hi;
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = W8 ? fmaf(part[i][j], j < 2 ? s_lo : s_hi, acc[i][j]) : part[i][j];
    }
}

struct alignas(16) Shared {
    float part[WARPS][NT][2][MAX_T][4];      // [warp][tile][half of its eight rows][token][row]
    float weight[MAX_T * MAX_K];             // by (token, choice)
    int chosen[MAX_T * MAX_K];
    unsigned users[MAX_E];                   // tokens that chose an expert
    int slot[MAX_E];
    int expert[MAX_T * MAX_K];               // the chosen experts in ascending order
    unsigned mask[MAX_T * MAX_K];            // their tokens
    int first[MAX_T * MAX_K];                // where their tokens' weights begin in
    float factor[MAX_T * MAX_K];             // [slot][its tokens in order]
    int2 unit[WARPS][NT];                    // [team][tile]: (slot, first column) of a team's units
    int active;
    int go;
};
static_assert(sizeof(Shared) % 16 == 0, "rows of 16-byte pieces lie behind it");

// Warp t: token t's choices, as the router kernels choose (the lowest index among equals).  A NaN among a token's logits makes its weights NaN.
__device__ __forceinline__ void choose(const Params& p, Shared& sm, float* score, int t) {
    const int lane = threadIdx.x & 31;
    float* c_s = score + (size_t)t * 2 * p.E;             // what the choice goes by, then what the weights go by
    float* s_s = c_s + p.E;
    const float* z = p.z + (size_t)t * p.E;
    bool broken = false;
    for (int e = lane; e < p.E; e += 32) {
        const float v = z[e] + (p.bias ? p.bias[e] : 0.0f);
        const float s = p.softmax ? v : 1.0f / (1.0f + expf(-v));
        broken |= s != s;
        s_s[e] = s;
        c_s[e] = p.correction ? s + p.correction[e] : s;
    }
    broken = __any_sync(0xffffffffu, broken);
    __syncwarp();
    float total = 0.0f, top = 0.0f, mine = 0.0f;
    for (int j = 0; j < p.k; ++j) {
        float best = -INFINITY;
        int at = 0x7fffffff;
        for (int e = lane; e < p.E; e += 32) {
            const float c = c_s[e];
            if (c > best) { best = c; at = e; }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ob = __shfl_xor_sync(0xffffffffu, best, o);
            const int oa = __shfl_xor_sync(0xffffffffu, at, o);
            if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
        }
        if (at >= p.E) at = j < p.E ? j : 0;               // no score is above minus infinity: any expert, but a valid one
        float s = s_s[at];
        if (p.softmax) {
            if (j == 0) top = s;
            s = expf(s - top);
        }
        total += s;
        if (lane == j) mine = s;
        if (lane == 0) {
            sm.chosen[t * p.k + j] = at;
            c_s[at] = -INFINITY;
        }
        __syncwarp();
    }
    if (lane < p.k) {
        float w = p.softmax ? mine * (p.scale / total) : mine * (p.renormalize ? p.scale / total : p.scale);
        sm.weight[t * p.k + lane] = broken ? __int_as_float(0x7fc00000) : w;
    }
}

// A barrier of `threads` threads of the CTA, a multiple of 32
__device__ __forceinline__ void named_barrier(int id, int threads) {
    if (threads == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Every thread of the grid behind every other's stores.  False: gave up.
__device__ __forceinline__ bool grid_barrier(int* counter, int* go) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        atomicAdd(counter, 1);
        int seen = 0;
        for (uint32_t i = 0; i < BARRIER_LIMIT && !seen; ++i) {
            int v;
            asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
            seen = v >= (int)gridDim.x;
        }
        *go = seen;
    }
    __syncthreads();
    return *go != 0;
}

template <bool W8, bool WIDE>
__global__ void __launch_bounds__(THREADS, 1)
moe_few_kernel(const Params p) {
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& sm = *reinterpret_cast<Shared*>(smem);
    float* score = reinterpret_cast<float*>(smem + sizeof(Shared));      // [T, 2, E]
    constexpr int SIZE = W8 ? 1 : 2;                                      // bytes of a weight
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    // rows x in shared memory: a pitch of 64 bytes over a multiple of 128 puts two rows' 64 bytes into different banks
    const int pitch = (p.ldx + 127) / 128 * 128 + 64;
    uint8_t* const staged = smem + sizeof(Shared) + ((size_t)p.T * 2 * p.E * 4 + 15) / 16 * 16;
    pdl_wait();
    if (p.staged) {
        const int each = p.ldx / 16;
        for (int i = threadIdx.x; i < p.T * each; i += THREADS) {
            const int r = i / each, c = (i - r * each) * 16;
            mma16::cp_async_16(staged + (size_t)r * pitch + c, p.x + (size_t)r * p.ldx + c, 16);
        }
    }
    mma16::cp_async_commit();

    // ---- who goes where (every CTA for itself) ------------------------------------------------
    for (int e = threadIdx.x; e < p.E; e += THREADS) sm.users[e] = 0;
    for (int t = warp; t < p.T; t += WARPS) choose(p, sm, score, t);
    __syncthreads();
    for (int i = threadIdx.x; i < p.T * p.k; i += THREADS) atomicOr(&sm.users[sm.chosen[i]], 1u << (i / p.k));
    __syncthreads();
    if (warp == 0) {
        int n = 0, before = 0;
        for (int e0 = 0; e0 < p.E; e0 += 32) {
            const int e = e0 + lane;
            const unsigned m = e < p.E ? sm.users[e] : 0u;
            const unsigned any = __ballot_sync(0xffffffffu, m != 0);
            int incl = __popc(m);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            if (m) {
                const int s = n + __popc(any & ((1u << lane) - 1));
                sm.slot[e] = s;
                sm.expert[s] = e;
                sm.mask[s] = m;
                sm.first[s] = before + incl - __popc(m);
            }
            n += __popc(any);
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) sm.active = n;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.T * p.k; i += THREADS) {
        const int a = sm.slot[sm.chosen[i]], t = i / p.k;
        sm.factor[sm.first[a] + __popc(sm.mask[a] & ((1u << t) - 1))] = sm.weight[i];
    }
    mma16::cp_async_wait_all();
    __syncthreads();
    const int active = sm.active;

    uint4 w[NT][2];                                                       // the step that is on its way
    float acc[NT][4];
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
    };
    auto leave = [&]() {                                                  // this warp's sums for the others to add
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            float (&d)[2][MAX_T][4] = sm.part[warp][i];
            *reinterpret_cast<float2*>(&d[t4 >> 1][g][2 * (t4 & 1)]) = make_float2(acc[i][0], acc[i][1]);
            if (WIDE) *reinterpret_cast<float2*>(&d[t4 >> 1][g + 8][2 * (t4 & 1)]) = make_float2(acc[i][2], acc[i][3]);
        }
    };

    // ---- act: units of four gate rows and their up rows, dealt out over the teams, up to NT units at a time -------------
    {
        const int team = p.team, me = warp % team, my_team = warp / team, teams = gridDim.x * (WARPS / team);
        const int per = (p.I + 3) / 4, NB = (2 * p.I + fp8::BLOCK - 1) / fp8::BLOCK, KB = (p.H + fp8::BLOCK - 1) / fp8::BLOCK;
        const long long units = (long long)active * per;
        const int index = blockIdx.x * (WARPS / team) + my_team;
        const int u_begin = (int)(units * index / teams), u_count = (int)(units * (index + 1) / teams) - u_begin;
        const int groups = (u_count + NT - 1) / NT, size = groups ? u_count / groups : 0, larger = groups ? u_count - size * groups : 0;
        const int len = p.H * SIZE, steps = (len + STEP - 1) / STEP;
        const uint8_t* const x = p.staged ? staged : p.x;
        const unsigned ld = p.staged ? pitch : p.ldx;
        const uint8_t* const x_lo = g < p.T ? x + g * ld : nullptr;
        const uint8_t* const x_hi = WIDE && g + 8 < p.T ? x + (g + 8) * ld : nullptr;
        int a = u_begin / per, c = u_begin - a * per;                     // slot and unit within of the next group's first
        const uint8_t* row[NT];
        unsigned scale_at[NT];
        int next_tiles = 0;
        unsigned next_scale_at[NT];
        int2 next_unit = make_int2(0, 0);                                 // lane i < NT: of unit i
        // the rows and scales of group i, whose first unit is (a, c); on to the group behind it
        auto look_up = [&](int i) {
            next_tiles = size + (i < larger);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int e = sm.expert[a], r = min(c * 4 + (g & 3), p.I - 1);
                row[j] = static_cast<const uint8_t*>(p.gate_up) + (unsigned long long)(unsigned)(e * 2 * p.I + (g < 4 ? r : p.I + r)) * (unsigned)p.ldg;
                if constexpr (W8) {
                    // sums 2 t4 and 2 t4 + 1 of the tile: gate rows for t4 < 2, up rows above; as I is even two neighbours lie
                    // in one block of 128 rows
                    const int n = min(c * 4 + 2 * (t4 & 1), p.I - 2) + (t4 < 2 ? 0 : p.I);
                    next_scale_at[j] = (unsigned)(e * NB + n / fp8::BLOCK) * (unsigned)KB;
                }
                if (lane == j) next_unit = make_int2(a, c * 4);
                if (j + 1 <= next_tiles && !(j + 1 == next_tiles && i + 1 == groups) && ++c == per) {
                    c = 0;
                    ++a;
                }
            }
        };
        if (groups) {
            look_up(0);
            fetch(w, row, next_tiles, me * STEP, len);                    // (a team has at most a quarter as many warps as steps)
        }
        for (int i = 0; i < groups; ++i) {
            clear();
            const int tiles = next_tiles;
            const int2 unit = next_unit;
#pragma unroll
            for (int j = 0; j < NT; ++j) scale_at[j] = next_scale_at[j];
            for (int s = me; s < steps; s += team) {
                const int at = s * STEP, x_at = s * (W8 ? 2 * STEP : STEP);
                float scale[NT], f_lo = 0.0f, f_hi = 0.0f;
                if constexpr (W8) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) scale[j] = p.gate_up_scale[scale_at[j] + s];
                    if (g < p.T) f_lo = p.x_scale[g * KB + s];
                    if (WIDE && g + 8 < p.T) f_hi = p.x_scale[(g + 8) * KB + s];
                }
                multiply<W8, WIDE>(acc, w, tiles, x_lo ? x_lo + x_at : nullptr, WIDE && x_hi ? x_hi + x_at : nullptr, p.ldx - x_at, f_lo, f_hi, scale);
                if (s + team < steps) {
                    fetch(w, row, tiles, at + team * STEP, len);
                } else if (i + 1 < groups) {
                    look_up(i + 1);
                    fetch(w, row, next_tiles, me * STEP, len);
                }
            }
            named_barrier(1 + my_team, team * 32);                        // the sums before these are added by now
            if (me == 0 && lane < NT) sm.unit[my_team][lane] = lane < tiles ? unit : make_int2(-1, 0);
            leave();
            named_barrier(1 + my_team, team * 32);
            for (int o = me * 32 + lane; o < NT * MAX_T * 4; o += team * 32) {
                const int j = o / (MAX_T * 4), t = o / 4 % MAX_T;
                const int2 unit = sm.unit[my_team][j];
                const int col = unit.y + o % 4;
                if (unit.x < 0 || t >= p.T || col >= p.I) continue;
                const unsigned m = sm.mask[unit.x];
                if (!(m >> t & 1)) continue;
                float gv = 0.0f, uv = 0.0f;
                for (int q = 0; q < team; ++q) {
                    gv += sm.part[my_team * team + q][j][0][t][o % 4];
                    uv += sm.part[my_team * team + q][j][1][t][o % 4];
                }
                const float f = sm.factor[sm.first[unit.x] + __popc(m & ((1u << t) - 1))];
                if (p.on_input) { gv *= f; uv *= f; }
                float v = gv / (1.0f + expf(-gv)) * uv;
                if (!p.on_input) v *= f;
                const size_t at = ((size_t)unit.x * p.T + t) * p.Ip + col;
                if constexpr (W8) static_cast<float*>(p.act)[at] = v;
                else static_cast<bf16*>(p.act)[at] = __float2bfloat16_rn(v);
            }
        }
    }

    // ---- y: rows of the down matrices, dealt out over the grid; the sum runs over all chosen experts.  The first weights
    // are asked for ahead of the barrier. ---------------------------------------------------------------------------------
    const int pairs = (p.H + 1) / 2, NB = (p.H + fp8::BLOCK - 1) / fp8::BLOCK, KB = (p.I + fp8::BLOCK - 1) / fp8::BLOCK;
    const int r_begin = 2 * (int)((long long)pairs * blockIdx.x / gridDim.x);
    const int r_end = min(p.H, 2 * (int)((long long)pairs * (blockIdx.x + 1) / gridDim.x));
    const int all_tiles = (r_end - r_begin + 7) / 8, groups = (all_tiles + NT - 1) / NT;
    const int len = p.I * SIZE, per = (len + STEP - 1) / STEP, steps = active * per;
    // steps go round the warps: (slot, step within) and on by WARPS
    const int round_a = WARPS / per, round_s = WARPS - round_a * per, warp_a = warp / per, warp_s = warp - warp_a * per;
    int a = warp_a, k = warp_s;                                           // of the step on its way
    unsigned row_at[NT];
    auto rows_of = [&](int first) {
#pragma unroll
        for (int i = 0; i < NT; ++i) row_at[i] = (unsigned)min(r_begin + (first + i) * 8 + g, r_end - 1);
    };
    auto fetch_down = [&](int tiles) {
        const uint8_t* const base = static_cast<const uint8_t*>(p.down) + (size_t)sm.expert[a] * p.H * p.ldd;
        const uint8_t* row[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) row[i] = base + (unsigned long long)row_at[i] * (unsigned)p.ldd;
        fetch(w, row, tiles, k * STEP, len);
    };
    auto tile_of = [&](int i) { return all_tiles * i / groups; };         // group i: tiles from ... on
    if (groups && warp < steps) {
        rows_of(0);
        fetch_down(tile_of(1));
    }
    bool met = grid_barrier(p.barrier, &sm.go);
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
            met = grid_barrier(p.barrier + 1, &sm.go);
        }
    }
    if (!met) {
        if (threadIdx.x == 0) atomicExch(p.status, 19);
        return;
    }
    for (int i = 0; i < groups; ++i) {
        const int first = tile_of(i), tiles = tile_of(i + 1) - first, r0 = r_begin + first * 8, r1 = min(r_end, r0 + tiles * 8);
        unsigned block[NT];                                               // (rows from an even one on: both sums' lie in one block)
#pragma unroll
        for (int j = 0; j < NT; ++j) block[j] = (unsigned)min(r0 + j * 8 + 2 * t4, p.H - 1) / fp8::BLOCK;
        clear();
        for (int s = warp; s < steps; s += WARPS) {
            const int e = sm.expert[a], from = k;
            const unsigned m = sm.mask[a], r = (unsigned)(a * p.T + g);
            const bool in_lo = m >> g & 1, in_hi = WIDE && (m >> (g + 8) & 1);
            const uint8_t* lo = nullptr;
            const uint8_t* hi = nullptr;
            float scale[NT], f_lo = 0.0f, f_hi = 0.0f;
            const uint8_t* const act = W8 ? reinterpret_cast<const uint8_t*>(p.act16) : static_cast<const uint8_t*>(p.act);
            const unsigned x_at = from * (W8 ? 2 * STEP : STEP);
            if (in_lo) lo = act + (size_t)r * 2 * p.Ip + x_at;
            if (in_hi) hi = act + (size_t)(r + 8) * 2 * p.Ip + x_at;
            if constexpr (W8) {
                if (in_lo) f_lo = p.act_scale[r * KB + from];
                if (in_hi) f_hi = p.act_scale[(r + 8) * KB + from];
#pragma unroll
                for (int j = 0; j < NT; ++j) scale[j] = p.down_scale[(unsigned)(e * NB + block[j]) * (unsigned)KB + from];
            }
            multiply<W8, WIDE>(acc, w, tiles, lo, hi, W8 ? 2 * STEP : len - from * STEP, f_lo, f_hi, scale);
            a += round_a;
            k += round_s;
            if (k >= per) {
                k -= per;
                ++a;
            }
            if (s + WARPS < steps) {
                fetch_down(tiles);
            } else if (i + 1 < groups) {
                a = warp_a;
                k = warp_s;
                rows_of(first + tiles);
                fetch_down(tile_of(i + 2) - first - tiles);
            }
        }
        if (i > 0) __syncthreads();                                       // the sums before these are added by now
        leave();
        __syncthreads();
        for (int o = threadIdx.x; o < NT * 2 * MAX_T * 4; o += THREADS) {
            const int j = o >> 7, half = o >> 6 & 1, t = o / 4 % MAX_T, c = o % 4, r = r0 + j * 8 + half * 4 + c;
            if (r >= r1 || t >= p.T) continue;
            float v = 0.0f;
#pragma unroll
            for (int q = 0; q < WARPS; ++q) v += sm.part[q][j][half][t][c];
            const size_t to = (size_t)t * p.H + r;
            if (p.add) v += p.add[to];
            if (p.out_bf16) static_cast<bf16*>(p.out)[to] = __float2bfloat16_rn(v);
            else static_cast<float*>(p.out)[to] = v;
        }
    }
}

template <bool W8, bool WIDE>
int launch(Params& p, int sms, cudaStream_t stream) {
    const auto kernel = moe_few_kernel<W8, WIDE>;
    const size_t scores = ((size_t)p.T * 2 * p.E * sizeof(float) + 15) / 16 * 16;
    const size_t rows = (size_t)p.T * ((p.ldx + 127) / 128 * 128 + 64);
    constexpr size_t MOST = 226 * 1024;
    p.staged = sizeof(Shared) + scores + rows <= MOST;
    const size_t smem = sizeof(Shared) + scores + (p.staged ? rows : 0);
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return SHARPI_LAUNCH_FAILED;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = sms;
    cfg.blockDim = THREADS;
    cfg.dynamicSmemBytes = smem;
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

}  // namespace

// h bf16 [T, H] rows ldh elements apart (bf16 weights: ldh a multiple of 8, 16-byte alignment), x: what the router reads,
// float32 or bfloat16 [T, ldx]; weights bf16, or e4m3 with scales; rows ldg / ldd bytes apart; work: 16-byte aligned.
SHARPI_API int sharpi_moe_few(const void* x, int x_dtype, int ldx, const void* h, int ldh, const float* router, const float* bias,
                              const float* correction, const void* gate_up, long long ldg, const float* gate_up_scale,
                              const void* down, long long ldd, const float* down_scale, const float* add, void* work, int* status,
                              void* out, int out_bf16, int T, int E, int k, int H, int I, int softmax, int renormalize, float scale,
                              int on_input, int sms, cudaStream_t stream) {
    if (T <= 0) return SHARPI_OK;
    if (T > MAX_T || E <= 0 || E > MAX_E || k <= 0 || k > MAX_K || k > E || H <= 0 || I <= 0 || sms <= 0 ||
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
    p.softmax = softmax; p.renormalize = renormalize; p.on_input = on_input; p.out_bf16 = out_bf16; p.scale = scale;
    // as many warps a team as leave each of them four steps of a row's K, so that joining their sums stays a small part
    const int steps = (H * (w8 ? 1 : 2) + STEP - 1) / STEP;
    p.team = 1;
    while (p.team < WARPS && p.team * 8 <= steps) p.team *= 2;
    const bool wide = T > 8;
    return w8 ? (wide ? launch<true, true>(p, sms, stream) : launch<true, false>(p, sms, stream))
              : (wide ? launch<false, true>(p, sms, stream) : launch<false, false>(p, sms, stream));
}
