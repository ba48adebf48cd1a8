// ortho.hip -- the orthogonalised form of a factor table's update by Newton-Schulz products (gfx950).
//
// With G tall (long side R, short side S; a wide G is the same with its sides exchanged), X_{j+1} = X_j M_j,
// M_j = a I + b A_j + c A_j^2, A_j = X_j^T X_j: all of them are polynomials of the one S x S matrix A_0 = G^T G / |G|^2, so
//   X_steps = G T / |G|,  T = M_0 M_1 ...,  A_{j+1} = M_j A_j M_j,
// and the table is read once for A_0 (whose trace is |G|^2) and once for G T, instead of three products of the
// table per step.  The S x S chain runs in fp64: A_j's error grows by up to a^2 per step in the directions of small
// singular values, which fp32 sums would not stand.
#include <hip/hip_runtime.h>

#include <cmath>

#include "dense.hpp"

namespace rs {
namespace {

constexpr int kGT = 64;   // tile of the Gram matrix
constexpr int kGR = 32;   // long-side rows of a step
constexpr int kAR = 128;  // long-side rows of an apply tile

struct OrthoPlan {
    int64_t r;         // long side
    int32_t s, sp;     // short side, and padded to kGT
    int32_t nb, pairs; // Gram tiles per side, tiles of the lower triangle
    int32_t splits;
    int64_t per;       // long-side rows of a split
    int64_t o_part, o_mat[6], bytes;  // A0, A, M, U, Ta, Tb
};

OrthoPlan make_plan(int64_t rows, int64_t cols) {
    OrthoPlan p{};
    p.r = std::max(rows, cols);
    p.s = static_cast<int32_t>(std::min(rows, cols));
    p.sp = static_cast<int32_t>(round_up(p.s, kGT));
    p.nb = p.sp / kGT;
    p.pairs = p.nb * (p.nb + 1) / 2;
    const int64_t want = std::max<int64_t>(1, 1024 / p.pairs);
    p.per = round_up(std::max<int64_t>(ceil_div(p.r, want), 64), kGR);
    p.splits = static_cast<int32_t>(ceil_div(p.r, p.per));
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at += round_up(bytes, 256);
        return o;
    };
    p.o_part = take(static_cast<int64_t>(p.splits) * p.pairs * kGT * kGT * 8);
    for (int64_t& o : p.o_mat) o = take(static_cast<int64_t>(p.sp) * p.sp * 8);
    p.bytes = at;
    return p;
}

// element (long index r, short index i) of the table
template <typename E, bool WIDE>
__device__ __forceinline__ float elem(const E* G, int64_t ld, int64_t r, int i) {
    return static_cast<float>(WIDE ? G[i * ld + r] : G[r * ld + i]);
}

// ---- Gram tiles of a piece of the long side (fp64 sums of exact products) ------------------------------------------
template <typename E, bool WIDE>
__global__ __launch_bounds__(256) void ortho_gram_kernel(const E* __restrict__ G, int64_t ld, OrthoPlan p, double* __restrict__ part) {
    __shared__ float gi[kGR][kGT + 1], gj[kGR][kGT + 1];
    int ib = 0, t = blockIdx.x;
    while (t > ib) t -= ++ib;  // tile t of the lower triangle: row ib, column t
    const int jb = t;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lc = lane & 15, lk = lane >> 4;
    const int wi = (wave & 1) * 32, wj = (wave >> 1) * 32;
    const int64_t r0 = blockIdx.y * p.per, r1 = min(p.r, r0 + p.per);
    f64x4 acc[2][2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) acc[x][y] = f64x4{0};
    for (int64_t rb = r0; rb < r1; rb += kGR) {
        for (int e = threadIdx.x; e < kGR * kGT; e += 256) {
            const int rr = WIDE ? e % kGR : e / kGT, c = WIDE ? e / kGR : e % kGT;
            const int64_t r = rb + rr;
            gi[rr][c] = r < r1 && ib * kGT + c < p.s ? elem<E, WIDE>(G, ld, r, ib * kGT + c) : 0.f;
            gj[rr][c] = r < r1 && jb * kGT + c < p.s ? elem<E, WIDE>(G, ld, r, jb * kGT + c) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kGR; k += 4) {
            double a[2], b[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                a[x] = static_cast<double>(gi[k + lk][wi + 16 * x + lc]);
                b[x] = static_cast<double>(gj[k + lk][wj + 16 * x + lc]);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) acc[x][y] = __builtin_amdgcn_mfma_f64_16x16x4f64(a[x], b[y], acc[x][y], 0, 0, 0);
        }
        __syncthreads();
    }
    double* o = part + (static_cast<int64_t>(blockIdx.y) * p.pairs + blockIdx.x) * kGT * kGT;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[(wi + 16 * x + 4 * e + lk) * kGT + wj + 16 * y + lc] = acc[x][y][e];
}

// the pieces' sum, in their order, to both triangles
__global__ __launch_bounds__(256) void ortho_gram_join_kernel(const double* __restrict__ part, OrthoPlan p, double* __restrict__ A) {
    int ib = 0, t = blockIdx.x;
    while (t > ib) t -= ++ib;
    const int jb = t;
    const int e = blockIdx.y * 256 + threadIdx.x;  // element of the tile
    double s = 0.0;
    for (int i = 0; i < p.splits; ++i) s += part[(static_cast<int64_t>(i) * p.pairs + blockIdx.x) * kGT * kGT + e];
    const int i = ib * kGT + e / kGT, j = jb * kGT + e % kGT;
    if (ib == jb && e / kGT < e % kGT) return;  // a diagonal tile's upper half is its lower half's mirror
    A[static_cast<int64_t>(i) * p.sp + j] = s;
    A[static_cast<int64_t>(j) * p.sp + i] = s;
}

// trace of A0 over a block of 256 threads (the same sum in every block)
__device__ __forceinline__ double block_trace(const double* A0, const OrthoPlan& p) {
    __shared__ double sm[4];
    double t = 0.0;
    for (int i = threadIdx.x; i < p.s; i += 256) t += A0[static_cast<int64_t>(i) * p.sp + i];
#pragma unroll
    for (int o = 32; o; o >>= 1) t += __shfl_xor(t, o);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = t;
    __syncthreads();
    t = sm[0] + sm[1] + sm[2] + sm[3];
    __syncthreads();
    return t;
}

// ---- S x S products of symmetric, commuting matrices: C = X Y, 32 x 32 per workgroup, 16 x 16 per wave --------------
struct ChainArgs {
    OrthoPlan p;
    const double* A0;        // unnormalised Gram matrix
    const double* X[2];
    const double* Y[2];      // blockIdx.z
    double* C[2];
    int normalise;           // C[0]'s product takes 1 / trace (first step)
    int poly;                // C[0] = a I + b X + c X Y (first step: X and Y divided by the trace)
    double a, b, c;
};

__global__ __launch_bounds__(256) void ortho_chain_kernel(ChainArgs q) {
    const int sp = q.p.sp, z = blockIdx.z;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lc = lane & 15, lk = lane >> 4;
    const int i0 = blockIdx.x * 32 + (wave & 1) * 16, j0 = blockIdx.y * 32 + (wave >> 1) * 16;
    const double *X = q.X[z], *Y = q.Y[z];
    double inv = 1.0;
    if (q.normalise && z == 0) {
        const double tr = block_trace(q.A0, q.p);
        inv = tr == 0.0 ? 0.0 : 1.0 / tr;
    }
    f64x4 acc = f64x4{0};
    // X and Y are symmetric: both operands are read along rows k
    for (int k = 0; k < sp; k += 32) {
        double a[8], b[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            a[u] = X[static_cast<int64_t>(k + 4 * u + lk) * sp + i0 + lc];
            b[u] = Y[static_cast<int64_t>(k + 4 * u + lk) * sp + j0 + lc];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(a[u], b[u], acc, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int i = i0 + 4 * e + lk, j = j0 + lc;
        const int64_t at = static_cast<int64_t>(i) * sp + j;
        double v = acc[e] * inv;
        if (q.poly && z == 0) v = (i == j ? q.a : 0.0) + q.b * X[at] * inv + q.c * (v * inv);
        q.C[z][at] = v;
    }
}

// ---- X = G T / |G| -------------------------------------------------------------------------------------------------
// NB: column tiles at most (each workgroup has all columns of its rows)
template <typename E, bool WIDE, int NB>
__global__ __launch_bounds__(256) void ortho_apply_kernel(const E* G, int64_t ldg, OrthoPlan p, const double* __restrict__ A0,
                                                         const double* __restrict__ T, E* X, int64_t ldx) {
    __shared__ float gs[32][kAR + 1], ts[32][kGT + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lc = lane & 31, half = lane >> 5;
    const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kAR;
    const double tr = block_trace(A0, p);
    const float inv = tr == 0.0 ? 0.f : static_cast<float>(1.0 / sqrt(tr));
    // every column tile of these rows, their sums kept until all are read: X may be G
    f32x16 acc[NB][2];
#pragma unroll
    for (int jb = 0; jb < NB; ++jb) acc[jb][0] = acc[jb][1] = f32x16{0};
    for (int k0 = 0; k0 < p.s; k0 += 32) {
        __syncthreads();
        for (int e = threadIdx.x; e < 32 * kAR; e += 256) {
            const int rr = WIDE ? e % kAR : e / 32, c = WIDE ? e / kAR : e % 32;
            gs[c][rr] = r0 + rr < p.r && k0 + c < p.s ? elem<E, WIDE>(G, ldg, r0 + rr, k0 + c) : 0.f;
        }
#pragma unroll
        for (int jb = 0; jb < NB; ++jb) {
            if (jb >= p.nb) break;
            __syncthreads();
            for (int e = threadIdx.x; e < 32 * kGT; e += 256)
                ts[e / kGT][e % kGT] = static_cast<float>(T[static_cast<int64_t>(k0 + e / kGT) * p.sp + jb * kGT + e % kGT]);
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
                const float g = gs[k + half][wave * 32 + lc];
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float t = ts[k + half][32 * y + lc];
                    // lanes run along the contiguous side of X
                    acc[jb][y] = WIDE ? __builtin_amdgcn_mfma_f32_32x32x2f32(t, g, acc[jb][y], 0, 0, 0)
                                      : __builtin_amdgcn_mfma_f32_32x32x2f32(g, t, acc[jb][y], 0, 0, 0);
                }
            }
        }
    }
#pragma unroll
    for (int jb = 0; jb < NB; ++jb)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int row = 8 * (e / 4) + 4 * half + e % 4;
                const int64_t r = r0 + wave * 32 + (WIDE ? lc : row);
                const int j = jb * kGT + 32 * y + (WIDE ? row : lc);
                if (r < p.r && j < p.s) X[WIDE ? j * ldx + r : r * ldx + j] = static_cast<E>(acc[jb][y][e] * inv);
            }
}

template <typename E, bool WIDE>
void run(const OrthoPlan& p, const E* G, int64_t ldg, int32_t steps, double a, double b, double c, E* X, int64_t ldx, char* ws,
         hipStream_t st) {
    double* part = reinterpret_cast<double*>(ws + p.o_part);
    double* mat[6];
    for (int i = 0; i < 6; ++i) mat[i] = reinterpret_cast<double*>(ws + p.o_mat[i]);
    double *A0 = mat[0], *M = mat[2], *U = mat[3], *T = mat[4], *T2 = mat[5];
    ortho_gram_kernel<E, WIDE><<<dim3(p.pairs, p.splits), 256, 0, st>>>(G, ldg, p, part);
    RS_HIP(hipGetLastError());
    ortho_gram_join_kernel<<<dim3(p.pairs, kGT * kGT / 256), 256, 0, st>>>(part, p, A0);
    RS_HIP(hipGetLastError());
    const uint32_t t = static_cast<uint32_t>(p.sp / 32);
    ChainArgs q{};
    q.p = p, q.A0 = A0, q.a = a, q.b = b, q.c = c;
    const double* A = A0;
    for (int j = 0; j < steps; ++j) {
        const bool last = j + 1 == steps;
        q.normalise = j == 0;
        double* Mj = j == 0 ? T : M;  // T = M_0
        q.poly = 1;
        q.X[0] = q.Y[0] = A, q.C[0] = Mj;
        ortho_chain_kernel<<<dim3(t, t, 1), 256, 0, st>>>(q);
        RS_HIP(hipGetLastError());
        q.poly = 0;
        // A M (not after the last step) and T M (not in the first)
        int z = 0;
        if (!last) q.X[z] = A, q.Y[z] = Mj, q.C[z] = U, ++z;
        if (j) q.X[z] = T, q.Y[z] = Mj, q.C[z] = T2, ++z;
        if (z) ortho_chain_kernel<<<dim3(t, t, static_cast<uint32_t>(z)), 256, 0, st>>>(q);
        RS_HIP(hipGetLastError());
        if (j) std::swap(T, T2);
        if (last) break;
        q.normalise = 0;
        q.X[0] = U, q.Y[0] = Mj, q.C[0] = mat[1];
        ortho_chain_kernel<<<dim3(t, t, 1), 256, 0, st>>>(q);
        RS_HIP(hipGetLastError());
        A = mat[1];
    }
    auto apply = [&](auto nb) {
        ortho_apply_kernel<E, WIDE, decltype(nb)::value><<<static_cast<uint32_t>(ceil_div(p.r, kAR)), 256, 0, st>>>(G, ldg, p, A0, T, X, ldx);
    };
    if (p.nb <= 1)
        apply(std::integral_constant<int, 1>{});
    else if (p.nb <= 2)
        apply(std::integral_constant<int, 2>{});
    else if (p.nb <= 4)
        apply(std::integral_constant<int, 4>{});
    else
        apply(std::integral_constant<int, 8>{});
    RS_HIP(hipGetLastError());
}

std::string check_sizes(int64_t rows, int64_t cols) {
    if (rows < 0 || rows > INT32_MAX - 1024) return "rows out of range";
    if (cols < 0 || cols > INT32_MAX - 1024) return "cols out of range";
    return std::string();
}

}  // namespace
}  // namespace rs

extern "C" int rs_orthogonalize_workspace(rs_ctx* ctx, int64_t rows, int64_t cols, int64_t* bytes) {
    if (!bytes) return rs::set_error(ctx, RS_ERR_INVALID, "bytes is NULL");
    *bytes = 0;
    const std::string bad = rs::check_sizes(rows, cols);
    if (!bad.empty()) return rs::set_error(ctx, RS_ERR_INVALID, bad);
    if (std::min(rows, cols) > RS_DENSE_MAX_FACTORS)
        return rs::set_error(ctx, RS_ERR_UNSUPPORTED, "the shorter side must be at most 512");
    if (rows && cols) *bytes = rs::make_plan(rows, cols).bytes;
    return RS_OK;
}

extern "C" int rs_orthogonalize(rs_ctx* ctx, int32_t type, int64_t rows, int64_t cols, const void* G, int64_t ldg, int32_t steps,
                                double a, double b, double c, void* X, int64_t ldx, void* ws, int64_t ws_bytes, void* stream) {
    using namespace rs;
    if (!type_ok(type)) return set_error(ctx, RS_ERR_INVALID, "type must be RS_TYPE_F32, RS_TYPE_BF16 or RS_TYPE_F16");
    const std::string bad = check_sizes(rows, cols);
    if (!bad.empty()) return set_error(ctx, RS_ERR_INVALID, bad);
    if (std::min(rows, cols) > RS_DENSE_MAX_FACTORS) return set_error(ctx, RS_ERR_UNSUPPORTED, "the shorter side must be at most 512");
    if (steps < 1 || steps > RS_ORTHO_MAX_STEPS) return set_error(ctx, RS_ERR_INVALID, "steps must be in [1, 16]");
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return set_error(ctx, RS_ERR_INVALID, "coefficients must be finite");
    if (rows == 0 || cols == 0) return RS_OK;
    for (const std::string& m : {check_matrix("G", G, cols, ldg, type_size(type)), check_matrix("X", X, cols, ldx, type_size(type))})
        if (!m.empty()) return set_error(ctx, RS_ERR_INVALID, m);
    if (G == X && ldg != ldx) return set_error(ctx, RS_ERR_INVALID, "X is G with another row stride");
    const OrthoPlan p = make_plan(rows, cols);
    if (!ws || reinterpret_cast<uintptr_t>(ws) % 16) return set_error(ctx, RS_ERR_INVALID, "ws is NULL or not 16-byte aligned");
    if (ws_bytes < p.bytes)
        return set_error(ctx, RS_ERR_INVALID, "ws holds " + std::to_string(ws_bytes) + " bytes, " + std::to_string(p.bytes) + " needed");
    return dense_guard(ctx, [&]() -> int {
        const hipStream_t st = pick_stream(ctx, stream);
        with_type(type, [&](auto e) {
            using E = typename decltype(e)::type;
            auto go = [&](auto wide) {
                run<E, decltype(wide)::value>(p, static_cast<const E*>(G), ldg, steps, a, b, c, static_cast<E*>(X), ldx, static_cast<char*>(ws), st);
            };
            if (rows >= cols)
                go(std::false_type{});
            else
                go(std::true_type{});
        });
        return RS_OK;
    });
}
