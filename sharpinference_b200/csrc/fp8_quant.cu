// Quantisation to block-scaled 8-bit values (the definition is in fp8.cuh).
//
//   rows     x [M, K] float32 or bfloat16 (rows may lie apart, `rows` may gather them) -> q [M, K] e4m3, scale [blocks, M]:
//            a scale for 128 neighbours of one row.  A block's scales of all rows lie together, which is how the products
//            read them (a thread a row).
//   weight   w [E, N, K] -> q [E, N, K], scale [E, ceil(N / 128), ceil(K / 128)]: a scale for 128 rows by 128 columns.
//
// Rows of q are `ldq` bytes apart, a multiple of 16 (what a TMA copy of them needs); the bytes behind K are zeros.
//
// Both are bound by the bytes they move: a piece of 16 bytes stays in registers between the maximum and the rounding (a weight's
// blocks at its edges are read again).  8192 x 5120 float32 35.8 us, 5.9 TB/s; bfloat16 23.5 us, 5.4; a weight of 7001 x 5112 18.7.  The
// maximum of bfloat16 is taken two elements an instruction, on their bits.
#include "fp8.cuh"

namespace {

template <typename T> struct Piece;                      // 16 bytes of input
template <> struct Piece<float> {
    static constexpr int N = 4;
    // the largest magnitude's bits, as a float's
    static __device__ __forceinline__ uint32_t amax(const uint4& x) {
        return max(max(x.x & 0x7fffffffu, x.y & 0x7fffffffu), max(x.z & 0x7fffffffu, x.w & 0x7fffffffu));
    }
    static __device__ __forceinline__ void open(const uint4& x, float (&v)[4]) {
        v[0] = __uint_as_float(x.x); v[1] = __uint_as_float(x.y); v[2] = __uint_as_float(x.z); v[3] = __uint_as_float(x.w);
    }
};
template <> struct Piece<bf16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ uint32_t amax(const uint4& x) {
        const uint32_t m = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
        return max(m << 16, m & 0xffff0000u);
    }
    static __device__ __forceinline__ void open(const uint4& x, float (&v)[8]) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};

// The elements k .. k + N - 1 of a row of K as they lie in memory; zeros behind its end.  They are opened when all of a thread's
// pieces have been asked for: opening one waits for it.  VEC: rows start on 16 bytes.  Else the two aligned pieces that hold
// the elements are read (the second only if the row reaches into it; what shares an aligned piece with an element can be
// read) and shifted together:
template <typename T, bool VEC>
struct Raw {
    uint4 lo, hi;
    __device__ __forceinline__ void ask(const T* row, int k, int K) {
        lo = hi = make_uint4(0u, 0u, 0u, 0u);
        if (k >= K) return;
        if (VEC) {
            lo = *reinterpret_cast<const uint4*>(row + k);
        } else {
            const uintptr_t at = reinterpret_cast<uintptr_t>(row + k), first = at & ~uintptr_t(15);
            lo = *reinterpret_cast<const uint4*>(first);
            if (first + 16 < min(reinterpret_cast<uintptr_t>(row + K), at + 16)) hi = *reinterpret_cast<const uint4*>(first + 16);
        }
    }
    __device__ __forceinline__ uint4 piece(const T* row, int k, int K) const {
        constexpr int N = Piece<T>::N;
        uint4 x = lo;
        if (!VEC) {
            const int off = (int)(reinterpret_cast<uintptr_t>(row + k) & 15);
            uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
            if (off & 8) {
#pragma unroll
                for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
            }
            if (off & 4) {
#pragma unroll
                for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
            }
            const int bits = (off & 3) * 8;
            x = make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                           __funnelshift_r(w[3], w[4], bits));
        }
        if (k + N > K) {                                 // (the bits from `left` on in its four words)
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int left = (K - k) * (int)sizeof(T) * 8 - 32 * i;
                w[i] = left >= 32 ? w[i] : left <= 0 ? 0u : w[i] & (0xffffffffu >> (32 - left));
            }
            x = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return x;
    }
};

// The piece in 8 bits at dst (4 or 8 bytes, aligned so); `room`: bytes of the row from there on.
template <typename T>
__device__ __forceinline__ void store_piece(uint8_t* dst, int room, const uint4& x, float inv) {
    constexpr int N = Piece<T>::N;
    float v[N];
    Piece<T>::open(x, v);
    if (room <= 0) return;                               // ldq is a multiple of 16: a piece fits whole or not at all
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) w[i] = fp8::pack4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv, v[4 * i + 3] * inv);
    if constexpr (N == 4) *reinterpret_cast<uint32_t*>(dst) = w[0];
    else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
}

constexpr int ROWS_WARPS = 8, FEW_BYTES = 9 << 20;
// A warp takes 512 bytes of each of EACH neighbouring rows: one block (float32) or two (bfloat16) of each.  Up to 9 MB of x: one,
// which is the shortest way from a load to a store; more: four, 64 bytes in flight a thread.  Rows of 5120, one against four, us:
// 6 MB 3.0 and 3.5 (float32), 3.2 and 4.0 (bfloat16); 12 MB 4.5 and 4.2, 5.2 and 5.0; 48 MB 15.5 and 12.5, 17.4 and 15.0.  (Eight rows
// of bfloat16 2 to 11 % longer, 40 % where rows start anywhere.)
template <typename T, bool VEC, int EACH>
__global__ void __launch_bounds__(ROWS_WARPS * 32)
fp8_rows_kernel(const T* x, long long ldx, const int* rows, int M, int K, uint8_t* q, long long ldq, float* scale) {
    constexpr int N = Piece<T>::N, LANES = fp8::BLOCK / N, SIDE = 32 / LANES;
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int kb = (blockIdx.y * (blockDim.x / 32) + (threadIdx.x >> 5)) * SIDE + lane / LANES, k = kb * fp8::BLOCK + (lane % LANES) * N;
    const long long row0 = (long long)blockIdx.x * EACH;
    Raw<T, VEC> raw[EACH];
    const T* row[EACH];
#pragma unroll
    for (int r = 0; r < EACH; ++r) {
        const long long m = min(row0 + r, (long long)M - 1);
        row[r] = x + (rows ? rows[m] : m) * ldx;
    }
#pragma unroll
    for (int r = 0; r < EACH; ++r) raw[r].ask(row[r], k, K);
    float s[EACH];
#pragma unroll
    for (int r = 0; r < EACH; ++r) {
        const uint4 piece = raw[r].piece(row[r], k, K);
        uint32_t m = Piece<T>::amax(piece);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        s[r] = fp8::scale_of(m);
        if (row0 + r < M) store_piece<T>(q + (row0 + r) * ldq + k, (int)(ldq - k), piece, 1.0f / s[r]);
    }
    if (lane % LANES == 0 && kb * fp8::BLOCK < K) {
        float* dst = scale + (long long)kb * M + row0;
        if (EACH % 4 == 0 && M % 4 == 0) {               // (a multiple of four rows from here on)
#pragma unroll
            for (int r = 0; r + 3 < EACH; r += 4)
                if (row0 + r < M) *reinterpret_cast<float4*>(dst + r) = make_float4(s[r], s[r + 1], s[r + 2], s[r + 3]);
        } else {
#pragma unroll
            for (int r = 0; r < EACH; ++r)
                if (row0 + r < M) dst[r] = s[r];
        }
    }
}

constexpr int WEIGHT_THREADS = 256;

// A CTA takes a block of 128 x 128.
template <typename T, bool VEC>
__global__ void __launch_bounds__(WEIGHT_THREADS)
fp8_weight_kernel(const T* w, int N_, int K, long long ldw, long long group, uint8_t* q, long long ldq, float* scale) {
    constexpr int N = Piece<T>::N, LANES = fp8::BLOCK / N, SIDE = WEIGHT_THREADS / LANES, EACH = fp8::BLOCK / SIDE;
    __shared__ uint32_t part[WEIGHT_THREADS / 32];
    pdl_wait();
    const int k = blockIdx.x * fp8::BLOCK + (threadIdx.x % LANES) * N;
    const int n0 = blockIdx.y * fp8::BLOCK + threadIdx.x / LANES;
    const T* src = w + blockIdx.z * group;
    uint8_t* const dst = q + ((long long)blockIdx.z * N_) * ldq;
    // A whole block of aligned rows stays in registers; blocks at the edges and rows that start anywhere are read again (from
    // L1 and L2), which leaves room for more of them on an SM
    const bool whole = VEC && (blockIdx.x + 1) * fp8::BLOCK <= K && (blockIdx.y + 1) * fp8::BLOCK <= N_;
    uint4 kept[EACH];
    uint32_t m = 0;
    if (whole) {
#pragma unroll
        for (int r = 0; r < EACH; ++r) kept[r] = *reinterpret_cast<const uint4*>(src + (n0 + r * SIDE) * ldw + k);
#pragma unroll
        for (int r = 0; r < EACH; ++r) m = max(m, Piece<T>::amax(kept[r]));
    } else {
#pragma unroll 1
        for (int r0 = 0; r0 < EACH; r0 += 4) {
            Raw<T, VEC> raw[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) raw[r].ask(src + (n0 + (r0 + r) * SIDE) * ldw, k, n0 + (r0 + r) * SIDE < N_ ? K : 0);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                m = max(m, Piece<T>::amax(raw[r].piece(src + (n0 + (r0 + r) * SIDE) * ldw, k, n0 + (r0 + r) * SIDE < N_ ? K : 0)));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WEIGHT_THREADS / 32; ++i) m = max(m, part[i]);
    const float s = fp8::scale_of(m), inv = 1.0f / s;
    if (whole) {
#pragma unroll
        for (int r = 0; r < EACH; ++r) store_piece<T>(dst + (n0 + r * SIDE) * ldq + k, N, kept[r], inv);
    } else {
#pragma unroll 1
        for (int r0 = 0; r0 < EACH; r0 += 4) {
            Raw<T, VEC> raw[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) raw[r].ask(src + (n0 + (r0 + r) * SIDE) * ldw, k, n0 + (r0 + r) * SIDE < N_ ? K : 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int n = n0 + (r0 + r) * SIDE;
                if (n < N_) store_piece<T>(dst + n * ldq + k, (int)(ldq - k), raw[r].piece(src + n * ldw, k, K), inv);
            }
        }
    }
    if (threadIdx.x == 0) scale[((long long)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = s;
}

template <typename T>
bool vectors(const void* x, long long ld, long long group) {
    return (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ld * (long long)sizeof(T) % 16 == 0 && group * (long long)sizeof(T) % 16 == 0;
}

template <typename T, int EACH>
int rows_launch(const T* x, long long ldx, const int* rows, int M, int K, uint8_t* q, long long ldq, float* scale, cudaStream_t stream) {
    constexpr int SIDE = 32 / (fp8::BLOCK / Piece<T>::N);
    // a CTA's warps lie along K, as evenly as up to eight come
    const int groups = (K + SIDE * fp8::BLOCK - 1) / (SIDE * fp8::BLOCK), along = (groups + ROWS_WARPS - 1) / ROWS_WARPS;
    const int threads = 32 * ((groups + along - 1) / along);
    const dim3 grid((M + EACH - 1) / EACH, along);
    if (along > 65535) return SHARPI_BAD_ARGUMENT;
    if (vectors<T>(x, ldx, 0)) SHARPI_LAUNCH_PDL((fp8_rows_kernel<T, true, EACH>), grid, threads, 0, stream, x, ldx, rows, M, K, q, ldq, scale);
    else SHARPI_LAUNCH_PDL((fp8_rows_kernel<T, false, EACH>), grid, threads, 0, stream, x, ldx, rows, M, K, q, ldq, scale);
    return SHARPI_OK;
}

template <typename T>
int rows_impl(const void* x, long long ldx, const int* rows, int M, int K, void* q, long long ldq, float* scale, cudaStream_t stream) {
    const T* src = static_cast<const T*>(x);
    uint8_t* dst = static_cast<uint8_t*>(q);
    return (long long)M * K * (long long)sizeof(T) <= FEW_BYTES ? rows_launch<T, 1>(src, ldx, rows, M, K, dst, ldq, scale, stream)
                   : rows_launch<T, 4>(src, ldx, rows, M, K, dst, ldq, scale, stream);
}

template <typename T>
int weight_impl(const void* w, int E, int N, int K, long long ldw, long long group, void* q, long long ldq, float* scale, cudaStream_t stream) {
    const dim3 grid((K + fp8::BLOCK - 1) / fp8::BLOCK, (N + fp8::BLOCK - 1) / fp8::BLOCK, E);
    if (grid.y > 65535 || grid.z > 65535) return SHARPI_BAD_ARGUMENT;
    const T* src = static_cast<const T*>(w);
    uint8_t* dst = static_cast<uint8_t*>(q);
    if (vectors<T>(w, ldw, group)) SHARPI_LAUNCH_PDL((fp8_weight_kernel<T, true>), grid, WEIGHT_THREADS, 0, stream, src, N, K, ldw, group, dst, ldq, scale);
    else SHARPI_LAUNCH_PDL((fp8_weight_kernel<T, false>), grid, WEIGHT_THREADS, 0, stream, src, N, K, ldw, group, dst, ldq, scale);
    return SHARPI_OK;
}

}  // namespace

SHARPI_API int sharpi_fp8_rows(const void* x, int dtype, long long ldx, const int* rows, int M, int K, void* q, long long ldq,
                               float* scale, cudaStream_t stream) {
    if (M <= 0 || K <= 0) return SHARPI_OK;
    if (ldq < K || ldq % 16 != 0 || (reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(scale) & 15)) return SHARPI_UNALIGNED;
    return dtype == SHARPI_BF16 ? rows_impl<bf16>(x, ldx, rows, M, K, q, ldq, scale, stream)
         : dtype == SHARPI_F32 ? rows_impl<float>(x, ldx, rows, M, K, q, ldq, scale, stream) : (int)SHARPI_BAD_ARGUMENT;
}

SHARPI_API int sharpi_fp8_weight(const void* w, int dtype, int E, int N, int K, long long ldw, long long group, void* q,
                                 long long ldq, float* scale, cudaStream_t stream) {
    if (E <= 0 || N <= 0 || K <= 0) return SHARPI_OK;
    if (ldq < K || ldq % 16 != 0 || (reinterpret_cast<uintptr_t>(q) & 15)) return SHARPI_UNALIGNED;
    return dtype == SHARPI_BF16 ? weight_impl<bf16>(w, E, N, K, ldw, group, q, ldq, scale, stream)
         : dtype == SHARPI_F32 ? weight_impl<float>(w, E, N, K, ldw, group, q, ldq, scale, stream) : (int)SHARPI_BAD_ARGUMENT;
}
