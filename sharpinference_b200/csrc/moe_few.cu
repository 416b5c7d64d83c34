// A whole mixture-of-experts layer for up to 16 tokens in two kernels:
//
//   router    z = h Wr^T (float32), a warp a (token, expert)
//   experts   every token's k experts and their weights from z; act = silu(g) * u over the gate|up rows of the experts that
//             any token chose; a barrier over the grid; y[t] = add[t] + sum over the token's experts of w Wd act
//
// With few tokens the layer is a stream of the chosen experts' weights, so the second kernel is laid out for that alone: one
// CTA an SM, weight rows dealt out evenly over the CTAs whatever expert they belong to, each weight read once, in 16-byte
// pieces straight into registers, several pieces of a lane in flight.  All tokens are the 16-row operand of mma.sync
// m16n8k16 (bfloat16, float32 sums) against eight weight rows; a row of a token that did not choose the expert is computed
// and dropped (gate|up) or zero (down).  Because the down product is linear, a token's experts are one long sum over
// (expert, inner element): act is multiplied by the router's weight before (weights on the output), and all of a CTA's warps
// share the sum.  The warps' parts are added in warp order: a call's result is the same every time, but the order (float32
// rounding) of a token's sum goes by which experts the whole call reaches.
//
// Weights are bfloat16, or e4m3 with a scale for 128 x 128 (fp8.cuh).  An e4m3 value becomes bfloat16 exactly by moving its
// bits and a multiplication with 2^120; a block's products are added in float32 first, then scaled and added.  (The code of
// e4m3's NaN reads as 480 here; fp8_weight writes it only into blocks whose scale is NaN or infinite, and those stay NaN.)
//
// act is rounded to bfloat16 (2^-9 of its value at most) as in the other bfloat16 mixtures: it enters a tensor-core product.
//
// The barrier needs all CTAs on the GPU at once: the launch is cooperative.  Its counter lies in the call's own workspace and
// is set to zero by the router kernel.  The wait is bounded; on a timeout the kernel sets *status and returns.
#include "fp8.cuh"

namespace {

constexpr int MAX_T = 16, MAX_K = 32, MAX_E = 1024;
constexpr int WARPS = 16, THREADS = 32 * WARPS;
constexpr uint32_t BARRIER_LIMIT = 1u << 22;

struct Params {
    const float* z;               // [T, E]
    const float* bias;            // [E] or null
    const float* correction;      // [E] or null
    const bf16* h;                // [T, ldh]
    const void* gate_up;          // [E, 2 I, ldg] bytes apart
    const void* down;             // [E, H, ldd] bytes apart
    const float* gate_up_scale;   // e4m3: [E, blocks of 2 I, blocks of H]
    const float* down_scale;      // e4m3: [E, blocks of H, blocks of I]
    const float* add;             // [T, H] or null
    bf16* act;                    // [active, T, Ip]
    void* out;                    // [T, H]
    int* barrier;
    int* status;
    long long ldg, ldd;           // bytes
    int ldh, T, E, k, H, I, Ip;   // Ip: I rounded up to 16
    int softmax, renormalize, on_input, out_bf16;
    float scale;
};

// One warp a (token, expert), the additions in the order of the router kernels for more tokens: lane l adds the elements
// 128 i + 4 l + u in ascending i into chain u, the chains and then the lanes are added in a fixed order.
template <typename T>
__global__ void __launch_bounds__(128)
moe_few_router_kernel(const T* h, int ldh, const float* wr, int tokens, int H, int E, int vec, float* z, int* barrier) {
    const int item = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int e = item / tokens, t = item - e * tokens;
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0) *barrier = 0;
    if (e >= E) return;
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

__device__ __forceinline__ uint4 load_weights(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four e4m3 values as bfloat16, exactly: the bits s eeee mmm move to s 0000eeee mmm0000, which is the value times 2^-120
// (e4m3's subnormals become bfloat16's)
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t top = (w & 0x80808080u) | ((w >> 4) & 0x07070707u), low = (w << 4) & 0xf0f0f0f0u;
    const uint32_t a = __byte_perm(low, top, 0x5140), b = __byte_perm(low, top, 0x7362);
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x7b807b80u));
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x7b807b80u));
}

// How a step of a warp reads K: a lane has 16 bytes of a weight row in each of PIECES pieces; lanes 4 g + t of a row lie side
// by side.  Which elements of K share an MMA is free as long as both operands agree: lane t's bytes are its k values.
template <bool W8>
struct Step {
    static constexpr int VALUES = W8 ? 16 : 8;            // of a lane's 16 bytes
    static constexpr int PIECE = 4 * VALUES;              // elements of K
    static constexpr int PIECES = 2;
    static constexpr int K = PIECE * PIECES;              // 128 (one block) or 64
};

// Where the weights of a step lie, and what multiplies them
struct Source {
    const uint8_t* row[4];        // this lane's weight row of every tile (null: none), at the step's first element
    const float* scale[4];        // e4m3: the scale of this lane's two sums of every tile
};

template <bool W8, bool WIDE, int NT>
__device__ __forceinline__ void fetch(uint4 (&w)[NT][2], const Source& s, int k0, int K) {
    using S = Step<W8>;
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int k = k0 + p * S::PIECE + t * S::VALUES;
#pragma unroll
        for (int i = 0; i < NT; ++i)
            w[i][p] = s.row[i] && k < K ? load_weights(s.row[i] + (size_t)k * (W8 ? 1 : 2)) : make_uint4(0u, 0u, 0u, 0u);
    }
}

// acc += the step's products.  x: this lane's token row (and the row eight below) at element 0 of K, null: zeros; Kp: the
// row's width with zeros behind K.
template <bool W8, bool WIDE, int NT>
__device__ __forceinline__ void multiply(float (&acc)[NT][4], const uint4 (&w)[NT][2], const Source& s, const bf16* x_lo, const bf16* x_hi, int k0, int Kp) {
    using S = Step<W8>;
    const int t = threadIdx.x & 3;
    float part[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][j] = W8 ? 0.0f : acc[i][j];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int k = k0 + p * S::PIECE + t * S::VALUES;
        uint32_t lo[S::VALUES / 2], hi[S::VALUES / 2];
#pragma unroll
        for (int q = 0; q < S::VALUES / 8; ++q) {
            uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
            if (x_lo && k < Kp) a = *reinterpret_cast<const uint4*>(x_lo + k + 8 * q);
            if (WIDE && x_hi && k < Kp) b = *reinterpret_cast<const uint4*>(x_hi + k + 8 * q);
            lo[4 * q] = a.x; lo[4 * q + 1] = a.y; lo[4 * q + 2] = a.z; lo[4 * q + 3] = a.w;
            hi[4 * q] = b.x; hi[4 * q + 1] = b.y; hi[4 * q + 2] = b.z; hi[4 * q + 3] = b.w;
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const uint32_t word[4] = {w[i][p].x, w[i][p].y, w[i][p].z, w[i][p].w};
#pragma unroll
            for (int j = 0; j < S::VALUES / 4; ++j) {
                const uint32_t a[4] = {lo[2 * j], hi[2 * j], lo[2 * j + 1], hi[2 * j + 1]};
                if constexpr (W8) {
                    uint32_t b0, b1;
                    widen(word[j], b0, b1);
                    mma(part[i], a, b0, b1);
                } else {
                    mma(part[i], a, word[2 * j], word[2 * j + 1]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const float f = W8 && s.scale[i] ? s.scale[i][k0 / fp8::BLOCK] : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = W8 ? fmaf(part[i][j], f, acc[i][j]) : part[i][j];
    }
}

struct Shared {
    float part[WARPS][4][2][MAX_T][4];       // [warp][tile][half of its eight rows][token][row]
    float weight[MAX_T * MAX_K];             // by (token, choice)
    int chosen[MAX_T * MAX_K];
    unsigned users[MAX_E];                   // tokens that chose an expert
    int slot[MAX_E];
    int expert[MAX_T * MAX_K];               // the chosen experts in ascending order
    unsigned mask[MAX_T * MAX_K];
    float factor[MAX_T * MAX_K][MAX_T];      // [slot][token]
    int active;
    int go;
};

// Warp t: token t's choices, as the router kernels choose (the lowest index among equals).  A NaN among a token's logits makes its weights NaN.
__device__ __forceinline__ void choose(const Params& p, Shared& sm, float* score, int t) {
    const int lane = threadIdx.x & 31;
    float* c_s = score + (size_t)t * p.E;
    const float* z = p.z + (size_t)t * p.E;
    bool broken = false;
    for (int e = lane; e < p.E; e += 32) {
        const float v = z[e] + (p.bias ? p.bias[e] : 0.0f);
        const float s = p.softmax ? v : 1.0f / (1.0f + expf(-v));
        broken |= s != s;
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
        const float v = z[at] + (p.bias ? p.bias[at] : 0.0f);
        float s = p.softmax ? v : 1.0f / (1.0f + expf(-v));
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
    float* score = reinterpret_cast<float*>(smem + sizeof(Shared));      // [T, E]
    using S = Step<W8>;
    constexpr int NT = 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    pdl_wait();

    // ---- who goes where (every CTA for itself) ------------------------------------------------
    for (int e = threadIdx.x; e < p.E; e += THREADS) sm.users[e] = 0;
    if (warp < p.T) choose(p, sm, score, warp);
    __syncthreads();
    for (int i = threadIdx.x; i < p.T * p.k; i += THREADS) atomicOr(&sm.users[sm.chosen[i]], 1u << (i / p.k));
    __syncthreads();
    if (warp == 0) {
        int n = 0;
        for (int e0 = 0; e0 < p.E; e0 += 32) {
            const int e = e0 + lane;
            const unsigned m = e < p.E ? sm.users[e] : 0u;
            const unsigned any = __ballot_sync(0xffffffffu, m != 0);
            if (m) {
                const int s = n + __popc(any & ((1u << lane) - 1));
                sm.slot[e] = s;
                sm.expert[s] = e;
                sm.mask[s] = m;
            }
            n += __popc(any);
        }
        if (lane == 0) sm.active = n;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.T * p.k; i += THREADS) sm.factor[sm.slot[sm.chosen[i]]][i / p.k] = sm.weight[i];
    __syncthreads();
    const int active = sm.active;

    // ---- act: units of four gate rows and their up rows, dealt out over the grid ------------------
    {
        const int per = p.Ip / 4, NB = (2 * p.I + fp8::BLOCK - 1) / fp8::BLOCK, KB = (p.H + fp8::BLOCK - 1) / fp8::BLOCK;
        const long long units = (long long)active * per;
        const int u_begin = (int)(units * blockIdx.x / gridDim.x), u_end = (int)(units * (blockIdx.x + 1) / gridDim.x);
        const int steps = (p.H + S::K - 1) / S::K;
        const bf16* x_lo = g < p.T ? p.h + (size_t)g * p.ldh : nullptr;
        const bf16* x_hi = WIDE && g + 8 < p.T ? p.h + (size_t)(g + 8) * p.ldh : nullptr;
        auto where = [&](int u0, Source& s) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int u = u0 + i;
                s.row[i] = nullptr;
                s.scale[i] = nullptr;
                if (u >= u_end) continue;
                const int a = u / per, c = (u - a * per) * 4, e = sm.expert[a];
                const int r = c + (g & 3);
                if (r < p.I) s.row[i] = static_cast<const uint8_t*>(p.gate_up) + ((size_t)e * 2 * p.I + (g < 4 ? r : p.I + r)) * p.ldg;
                // sums 2 t4 and 2 t4 + 1 of the tile: gate rows for t4 < 2, up rows above; as I is even two neighbours lie in one
                // block of 128 rows
                if (W8 && c + 2 * (t4 & 1) < p.I)
                    s.scale[i] = p.gate_up_scale + ((size_t)e * NB + (t4 < 2 ? c + 2 * t4 : p.I + c + 2 * (t4 - 2)) / fp8::BLOCK) * KB;
            }
        };
        for (int u0 = u_begin; u0 < u_end; u0 += NT) {
            Source src;
            where(u0, src);
            float acc[NT][4];
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
            for (int s = warp; s < steps; s += WARPS) {
                uint4 w[NT][2];
                fetch<W8, WIDE, NT>(w, src, s * S::K, p.H);
                multiply<W8, WIDE, NT>(acc, w, src, x_lo, x_hi, s * S::K, p.ldh);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                float (&d)[2][MAX_T][4] = sm.part[warp][i];
                *reinterpret_cast<float2*>(&d[t4 >> 1][g][2 * (t4 & 1)]) = make_float2(acc[i][0], acc[i][1]);
                if (WIDE) *reinterpret_cast<float2*>(&d[t4 >> 1][g + 8][2 * (t4 & 1)]) = make_float2(acc[i][2], acc[i][3]);
            }
            __syncthreads();
            if (threadIdx.x < NT * MAX_T * 4) {
                const int i = threadIdx.x / (MAX_T * 4), t = threadIdx.x / 4 % MAX_T, c = threadIdx.x % 4, u = u0 + i;
                if (u < u_end && t < p.T) {
                    const int a = u / per, col = (u - a * per) * 4 + c;
                    if (sm.mask[a] >> t & 1) {
                        float gv = 0.0f, uv = 0.0f;
#pragma unroll
                        for (int w = 0; w < WARPS; ++w) {
                            gv += sm.part[w][i][0][t][c];
                            uv += sm.part[w][i][1][t][c];
                        }
                        const float f = sm.factor[a][t];
                        if (p.on_input) { gv *= f; uv *= f; }
                        float v = gv / (1.0f + expf(-gv)) * uv;
                        if (!p.on_input) v *= f;
                        p.act[((size_t)a * p.T + t) * p.Ip + col] = __float2bfloat16_rn(col < p.I ? v : 0.0f);
                    }
                }
            }
            __syncthreads();
        }
    }
    if (!grid_barrier(p.barrier, &sm.go)) {
        if (threadIdx.x == 0) atomicExch(p.status, 19);
        return;
    }

    // ---- y: rows of the down matrices, dealt out over the grid; the sum runs over all chosen experts ----------------
    {
        const int pairs = (p.H + 1) / 2, NB = (p.H + fp8::BLOCK - 1) / fp8::BLOCK, KB = (p.I + fp8::BLOCK - 1) / fp8::BLOCK;
        const int r_begin = 2 * (int)((long long)pairs * blockIdx.x / gridDim.x);
        const int r_end = min(p.H, 2 * (int)((long long)pairs * (blockIdx.x + 1) / gridDim.x));
        const int per = (p.I + S::K - 1) / S::K, steps = active * per;
        for (int r0 = r_begin; r0 < r_end; r0 += 8 * NT) {
            float acc[NT][4];
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
            for (int s = warp; s < steps; s += WARPS) {
                const int a = s / per, k0 = (s - a * per) * S::K, e = sm.expert[a];
                const unsigned m = sm.mask[a];
                Source src;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const int r = r0 + i * 8 + g, c = r0 + i * 8 + 2 * t4;
                    src.row[i] = r < r_end ? static_cast<const uint8_t*>(p.down) + ((size_t)e * p.H + r) * p.ldd : nullptr;
                    src.scale[i] = W8 && c < r_end ? p.down_scale + ((size_t)e * NB + c / fp8::BLOCK) * KB : nullptr;
                }
                const bf16* x = p.act + ((size_t)a * p.T + g) * p.Ip;
                uint4 w[NT][2];
                fetch<W8, WIDE, NT>(w, src, k0, p.I);
                multiply<W8, WIDE, NT>(acc, w, src, m >> g & 1 ? x : nullptr, WIDE && (m >> (g + 8) & 1) ? x + (size_t)8 * p.Ip : nullptr, k0, p.Ip);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                float (&d)[2][MAX_T][4] = sm.part[warp][i];
                *reinterpret_cast<float2*>(&d[t4 >> 1][g][2 * (t4 & 1)]) = make_float2(acc[i][0], acc[i][1]);
                if (WIDE) *reinterpret_cast<float2*>(&d[t4 >> 1][g + 8][2 * (t4 & 1)]) = make_float2(acc[i][2], acc[i][3]);
            }
            __syncthreads();
            {
                const int i = threadIdx.x >> 7, half = threadIdx.x >> 6 & 1, t = threadIdx.x / 4 % MAX_T, c = threadIdx.x % 4;
                const int r = r0 + i * 8 + half * 4 + c;
                if (r < r_end && t < p.T) {
                    float v = 0.0f;
#pragma unroll
                    for (int w = 0; w < WARPS; ++w) v += sm.part[w][i][half][t][c];
                    const size_t at = (size_t)t * p.H + r;
                    if (p.add) v += p.add[at];
                    if (p.out_bf16) static_cast<bf16*>(p.out)[at] = __float2bfloat16_rn(v);
                    else static_cast<float*>(p.out)[at] = v;
                }
            }
            __syncthreads();
        }
    }
}

template <bool W8, bool WIDE>
int launch(const Params& p, int sms, cudaStream_t stream) {
    const auto kernel = moe_few_kernel<W8, WIDE>;
    const size_t smem = sizeof(Shared) + (size_t)p.T * p.E * sizeof(float);
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return SHARPI_LAUNCH_FAILED;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = sms;
    cfg.blockDim = THREADS;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? SHARPI_OK : SHARPI_LAUNCH_FAILED;
}

}  // namespace

// h bf16 [T, ldh] (zeros behind H up to ldh), x: what the router reads, float32 or bfloat16 [T, ldx]; weights bf16, or e4m3
// with scales; rows ldg / ldd bytes apart.  z [T, E] and act [min(E, T k), T, I rounded up to 16] are the caller's workspace.
SHARPI_API int sharpi_moe_few(const void* x, int x_dtype, int ldx, const void* h, int ldh, const float* router, const float* bias,
                              const float* correction, const void* gate_up, long long ldg, const float* gate_up_scale,
                              const void* down, long long ldd, const float* down_scale, const float* add, float* z, void* act,
                              int* barrier, int* status, void* out, int out_bf16, int T, int E, int k, int H, int I, int softmax,
                              int renormalize, float scale, int on_input, int sms, cudaStream_t stream) {
    if (T <= 0) return SHARPI_OK;
    if (T > MAX_T || E <= 0 || E > MAX_E || k <= 0 || k > MAX_K || k > E || H <= 0 || I <= 0 || sms <= 0 ||
        (gate_up_scale == nullptr) != (down_scale == nullptr) || ldh < H || (x_dtype != SHARPI_F32 && x_dtype != SHARPI_BF16))
        return SHARPI_BAD_ARGUMENT;
    const bool w8 = gate_up_scale != nullptr;
    if (((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(gate_up) | reinterpret_cast<uintptr_t>(down) |
          reinterpret_cast<uintptr_t>(act)) & 15) || ldg % 16 || ldd % 16 || ldh % (w8 ? 16 : 8) || (!w8 && (H % 8 || I % 8)) ||
        (w8 && I % 2))
        return SHARPI_UNALIGNED;
    const int vec = H % 4 == 0 && ldx % 4 == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(router)) & 15) == 0;
    const int blocks = (int)(((long long)T * E + 3) / 4);
    if (x_dtype == SHARPI_F32)
        SHARPI_LAUNCH_PDL(moe_few_router_kernel<float>, blocks, 128, 0, stream, static_cast<const float*>(x), ldx, router, T, H, E, vec, z, barrier);
    else
        SHARPI_LAUNCH_PDL(moe_few_router_kernel<bf16>, blocks, 128, 0, stream, static_cast<const bf16*>(x), ldx, router, T, H, E, vec, z, barrier);
    Params p = {};
    p.z = z; p.bias = bias; p.correction = correction;
    p.h = static_cast<const bf16*>(h);
    p.gate_up = gate_up; p.down = down; p.gate_up_scale = gate_up_scale; p.down_scale = down_scale;
    p.add = add; p.act = static_cast<bf16*>(act); p.out = out; p.barrier = barrier; p.status = status;
    p.ldg = ldg; p.ldd = ldd; p.ldh = ldh;
    p.T = T; p.E = E; p.k = k; p.H = H; p.I = I; p.Ip = (I + 15) / 16 * 16;
    p.softmax = softmax; p.renormalize = renormalize; p.on_input = on_input; p.out_bf16 = out_bf16; p.scale = scale;
    const bool wide = T > 8;
    return w8 ? (wide ? launch<true, true>(p, sms, stream) : launch<true, false>(p, sms, stream))
              : (wide ? launch<false, true>(p, sms, stream) : launch<false, false>(p, sms, stream));
}
