// int8.hip -- rows quantised to 8 bits and the int8 matrix product with a scale per row and per channel (gfx950).
//
// C_mn = a_m b_n sum_k A_mk B_nk + ...: the sums run on the int8 matrix unit (exact in int32), the scales and biases in
// the epilogue.  Two kernels: for few rows of A one pass over B straight from HBM to registers (bound by B's bytes);
// for many rows LDS tiles (bound by the product, or for short rows by writing C).
#include <hip/hip_runtime.h>

#include "dense.hpp"

namespace rs {
namespace {

// ---- quantising rows: a wave per row -------------------------------------------------------------------------------
// x / s to the nearest integer, ties to even, as if the quotient were exact.  The fp32 quotient decides all but the
// neighbourhood of a tie (its error is below 2^-15 at |x / s| <= 127); there |x| is compared with (r + 1/2) s, which
// is exact in fp64.
__device__ __forceinline__ int quantize(float x, float s, float inv, bool safe) {
    const float ax = fabsf(x);
    float t = ax * inv;
    if (!safe) t = static_cast<float>(static_cast<double>(ax) / static_cast<double>(s));
    float r = floorf(t);
    const float d = t - r;
    int q;
    if (d > 0.499f && d < 0.501f) {
        const double tie = (static_cast<double>(r) + 0.5) * static_cast<double>(s), a = static_cast<double>(ax);
        const int ri = static_cast<int>(r);
        q = a > tie ? ri + 1 : a < tie ? ri : ri + (ri & 1);
    } else {
        q = static_cast<int>(rintf(t));
    }
    q = min(q, 127);
    return x < 0.f ? -q : q;
}

template <typename E>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const E* __restrict__ X, int64_t ldx, int64_t rows, int64_t cols,
                                                           int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale) {
    const int lane = threadIdx.x & 63;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    const E* x = X + r * ldx;
    uint32_t m = 0;
    for (int64_t c = lane; c < cols; c += 64) {
        const uint32_t b = __float_as_uint(static_cast<float>(x[c])) & 0x7FFFFFFFu;
        m = b > m ? b : m;
    }
    m = wave_max_u32(m);
    const bool finite = m < 0x7F800000u;
    const float s = finite ? __uint_as_float(m) * (1.f / 127.f) : __uint_as_float(0x7FC00000u);
    if (lane == 0) scale[r] = s;
    const bool some = finite && s > 0.f, safe = s > 7.9e-31f;
    const float inv = 1.f / s;
    int8_t* o = q + r * ldq;
    for (int64_t c = lane; c < cols; c += 64)
        o[c] = static_cast<int8_t>(some ? quantize(static_cast<float>(x[c]), s, inv, safe) : 0);
}

// ---- the product ---------------------------------------------------------------------------------------------------
struct I8Args {
    const int8_t *A, *B;
    int64_t m, n, k, lda, ldb, ldc;
    const float *a_scale, *b_scale, *row_bias, *col_bias;
    void* C;
};

// 16 bytes of a row from column c on, zeros past column k (nothing past it is read).  VEC: the row starts at a
// 16-byte address.
template <bool VEC>
__device__ __forceinline__ i32x4 load16(const int8_t* row, int64_t c, int64_t k) {
    i32x4 v = {0, 0, 0, 0};
    if (VEC && c + 16 <= k) return *reinterpret_cast<const i32x4*>(row + c);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (VEC && c + 4 * w + 4 <= k) {
            v[w] = *reinterpret_cast<const int*>(row + c + 4 * w);
        } else {
            uint32_t u = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (c + 4 * w + b < k) u |= static_cast<uint32_t>(static_cast<uint8_t>(row[c + 4 * w + b])) << (8 * b);
            v[w] = static_cast<int>(u);
        }
    }
    return v;
}

template <typename E>
__device__ __forceinline__ void store_scores(const I8Args& a, int64_t m, int64_t n0, const int (&acc)[4], float sa, float rb) {
#pragma clang fp contract(fast)
    E* C = static_cast<E*>(a.C) + m * a.ldc;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n0 + e < a.n) {
            float v = static_cast<float>(acc[e]) * (sa * a.b_scale[n0 + e]) + rb;
            if (a.col_bias) v += a.col_bias[n0 + e];
            C[n0 + e] = static_cast<E>(v);
        }
}

// Few rows of A (m <= 16): they sit in LDS; each wave takes 16 rows of B at a time straight from HBM into
// 16x16x64 MFMAs (first operand B's rows, second A's).
constexpr int kFewRows = 16;
constexpr int kFewMaxK = 4096;
template <typename E, bool VEC>
__global__ __launch_bounds__(256) void i8_few_kernel(I8Args a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lk = lane >> 4;
    const int kc = static_cast<int>(ceil_div(a.k, 64));  // steps of 64
    i32x4* xs = reinterpret_cast<i32x4*>(smem);          // [kc][64 lanes]
    for (int i = threadIdx.x; i < kc * 64; i += 256) {
        const int64_t row = i & 15;
        xs[i] = row < a.m ? load16<VEC>(a.A + row * a.lda, static_cast<int64_t>(i >> 6) * 64 + ((i & 63) >> 4) * 16, a.k) : i32x4{0, 0, 0, 0};
    }
    __syncthreads();
    const float sa = lr < a.m ? a.a_scale[lr] : 0.f, rb = lr < a.m && a.row_bias ? a.row_bias[lr] : 0.f;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + wave; t * 16 < a.n; t += static_cast<int64_t>(gridDim.x) * 4) {
        const int64_t n = t * 16 + lr;
        const int8_t* row = a.B + (n < a.n ? n : a.n - 1) * a.ldb;
        i32x4 acc = {0, 0, 0, 0};
        for (int s = 0; s < kc; ++s)
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(load16<VEC>(row, static_cast<int64_t>(s) * 64 + lk * 16, a.k), xs[s * 64 + lane], acc, 0, 0, 0);
        // lane: row m = lr of A, registers: rows 4 lk + e of B
        if (lr < a.m) {
            const int o[4] = {acc[0], acc[1], acc[2], acc[3]};
            store_scores<E>(a, lr, t * 16 + 4 * lk, o, sa, rb);
        }
    }
}

// Many rows: 128 x 128 tiles of C, four waves of 64 x 64, steps of 64 along k through a double-buffered LDS tile.
constexpr int kT = 128, kStep = 64;
template <typename E, bool VEC>
__global__ __launch_bounds__(256) void i8_tile_kernel(I8Args a) {
    __shared__ __attribute__((aligned(16))) char smem[2][2 * kT * kStep];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 31, half = lane >> 5;
    const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    const int64_t m0 = static_cast<int64_t>(blockIdx.x) * kT, n0 = static_cast<int64_t>(blockIdx.y) * kT;
    const int steps = static_cast<int>(ceil_div(a.k, kStep));
    // 16-byte chunk c of row r sits at chunk c ^ ((r / 2) mod 4)
    auto at = [](int r, int c) { return (r * 4 + (c ^ ((r >> 1) & 3))) * 16; };
    i32x4 st[4];
    auto fetch = [&](int s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int ch = i * 256 + threadIdx.x, r = (ch >> 2) & (kT - 1), c = ch & 3;
            const bool b = i >= 2;
            const int64_t row = (b ? n0 : m0) + r, rows = b ? a.n : a.m;
            st[i] = row < rows ? load16<VEC>((b ? a.B + row * a.ldb : a.A + row * a.lda), static_cast<int64_t>(s) * kStep + c * 16, a.k) : i32x4{0, 0, 0, 0};
        }
    };
    auto put = [&](int buf) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int ch = i * 256 + threadIdx.x, r = (ch >> 2) & (kT - 1), c = ch & 3;
            *reinterpret_cast<i32x4*>(smem[buf] + (i >= 2 ? kT * kStep : 0) + at(r, c)) = st[i];
        }
    };
    i32x16 acc[2][2];  // [n][m]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = i32x16{0};
    fetch(0);
    put(0);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        if (s + 1 < steps) fetch(s + 1);
        const char *tA = smem[s & 1], *tB = tA + kT * kStep;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i32x4 fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = *reinterpret_cast<const i32x4*>(tA + at(wm + 32 * i + lr, 2 * h + half));
                fb[i] = *reinterpret_cast<const i32x4*>(tB + at(wn + 32 * i + lr, 2 * h + half));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[i], fa[j], acc[i][j], 0, 0, 0);
        }
        if (s + 1 < steps) put((s + 1) & 1);
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t m = m0 + wm + 32 * j + lr;
        if (m >= a.m) continue;
        const float sa = a.a_scale[m], rb = a.row_bias ? a.row_bias[m] : 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int o[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                store_scores<E>(a, m, n0 + wn + 32 * i + 8 * g + 4 * half, o, sa, rb);
            }
    }
}

template <typename E, bool VEC>
void launch_i8(const I8Args& a, hipStream_t st) {
    if (a.m <= kFewRows && a.k <= kFewMaxK) {
        const int lds = static_cast<int>(ceil_div(a.k, 64)) * 1024;
        const int64_t blocks = ceil_div(a.n, 64);
        i8_few_kernel<E, VEC><<<static_cast<uint32_t>(std::min<int64_t>(blocks, 2048)), 256, lds, st>>>(a);
    } else {
        // rows of A vary fastest: the blocks that run together share B's tile
        i8_tile_kernel<E, VEC><<<dim3(static_cast<uint32_t>(ceil_div(a.m, kT)), static_cast<uint32_t>(ceil_div(a.n, kT))), 256, 0, st>>>(a);
    }
    RS_HIP(hipGetLastError());
}

}  // namespace
}  // namespace rs

extern "C" int rs_quantize_rows(rs_ctx* ctx, int32_t type, int64_t n_rows, int64_t n_cols, const void* X, int64_t ldx, int8_t* q,
                                int64_t ldq, float* scale, void* stream) {
    using namespace rs;
    if (!type_ok(type)) return set_error(ctx, RS_ERR_INVALID, "type must be RS_TYPE_F32, RS_TYPE_BF16 or RS_TYPE_F16");
    if (n_rows < 0 || n_rows > INT32_MAX) return set_error(ctx, RS_ERR_INVALID, "n_rows out of range");
    if (n_cols < 1) return set_error(ctx, RS_ERR_INVALID, "n_cols must be at least 1");
    if (n_rows == 0) return RS_OK;
    for (const std::string& b : {check_matrix("X", X, n_cols, ldx, type_size(type)), check_matrix("q", q, n_cols, ldq, 1),
                                 check_matrix("scale", scale, 1, 1, 4)})
        if (!b.empty()) return set_error(ctx, RS_ERR_INVALID, b);
    return dense_guard(ctx, [&]() -> int {
        const hipStream_t st = pick_stream(ctx, stream);
        with_type(type, [&](auto e) {
            using E = typename decltype(e)::type;
            quantize_rows_kernel<E><<<static_cast<uint32_t>(ceil_div(n_rows, 4)), 256, 0, st>>>(static_cast<const E*>(X), ldx, n_rows,
                                                                                              n_cols, q, ldq, scale);
        });
        RS_HIP(hipGetLastError());
        return RS_OK;
    });
}

extern "C" int rs_i8_matmul(rs_ctx* ctx, int64_t m, int64_t n, int64_t k, const int8_t* A, int64_t lda, const float* a_scale,
                            const int8_t* B, int64_t ldb, const float* b_scale, const float* row_bias, const float* col_bias,
                            int32_t out_type, void* C, int64_t ldc, void* stream) {
    using namespace rs;
    if (!type_ok(out_type)) return set_error(ctx, RS_ERR_INVALID, "out_type must be RS_TYPE_F32, RS_TYPE_BF16 or RS_TYPE_F16");
    if (m < 0 || m > INT32_MAX) return set_error(ctx, RS_ERR_INVALID, "m out of range");
    if (n < 0 || n > 65535LL * kT) return set_error(ctx, RS_ERR_INVALID, "n out of range");
    if (k < 1) return set_error(ctx, RS_ERR_INVALID, "k must be at least 1");
    if (k > RS_I8_MAX_K) return set_error(ctx, RS_ERR_UNSUPPORTED, "k must be at most 65536 (exact int32 sums)");
    if (m == 0 || n == 0) return RS_OK;
    for (const std::string& b : {check_matrix("A", A, k, lda, 1), check_matrix("B", B, k, ldb, 1), check_matrix("a_scale", a_scale, 1, 1, 4),
                                 check_matrix("b_scale", b_scale, 1, 1, 4), check_matrix("C", C, n, ldc, type_size(out_type)),
                                 row_bias ? check_matrix("row_bias", row_bias, 1, 1, 4) : std::string(),
                                 col_bias ? check_matrix("col_bias", col_bias, 1, 1, 4) : std::string()})
        if (!b.empty()) return set_error(ctx, RS_ERR_INVALID, b);
    I8Args a{A, B, m, n, k, lda, ldb, ldc, a_scale, b_scale, row_bias, col_bias, C};
    const bool vec = (reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B) | static_cast<uintptr_t>(lda) | static_cast<uintptr_t>(ldb)) % 16 == 0;
    return dense_guard(ctx, [&]() -> int {
        const hipStream_t st = pick_stream(ctx, stream);
        with_type(out_type, [&](auto e) {
            using E = typename decltype(e)::type;
            if (vec)
                launch_i8<E, true>(a, st);
            else
                launch_i8<E, false>(a, st);
        });
        return RS_OK;
    });
}
