// ortho.hip -- the orthogonalised form of a factor table's update by Newton-Schulz products (gfx950).
//
// With G tall (long side R, short side S; a wide G is the same with its sides exchanged), X_{j+1} = X_j M_j,
// M_j = a I + b A_j + c A_j^2, A_j = X_j^T X_j: all of them are polynomials of the one S x S matrix A_0 = G^T G / |G|^2, so
//   X_steps = G T / |G|,  T = M_0 M_1 ...,  A_{j+1} = M_j A_j M_j,
// and the table is read once for A_0 (whose trace is |G|^2) and once for G T, instead of three products of the
// table per step.  The S x S chain runs in fp64: A_j's error grows by up to a^2 per step in the directions of small
// singular values, which fp32 sums would not stand.
//
// Bound by the table's bytes where it is large, by the chain's 14 dependent products where it is not: 1e6 x 256 fp32 0.91 ms
// (Gram pass 0.38 ms, 2.7 TB/s; product 0.59 ms, 3.5 TB/s read and written; chain 0.08), 26744 x 128 bf16 93 us (19, 12,
// 55), 6040 x 100 fp32 81 us (13, 9, 53), 1682 x 20 fp32 29 us in five launches.
#include <hip/hip_runtime.h>

#include <cmath>

#include "dense.hpp"

namespace rs {
namespace {

constexpr int kThreads = 512;     // the two passes over the table: 8 waves
constexpr int kStage = 8192;      // table elements of one stage of the Gram pass (per panel)
constexpr int kJoinGroups = 8;    // groups that many pieces of the Gram matrix are summed in first
constexpr int kJoinDirect = 24;   // up to so many pieces are joined at once
constexpr int kPieces64 = 16;     // pieces of the fp64 Gram pass at most
constexpr float kLowUp = 2048.f;  // the second pieces of G's fp16 pairs are held up by this in the last pass (first pieces: 11 bits)

struct OrthoPlan {
    int64_t r;       // long side
    int32_t s, sp;   // short side; padded to 64, 128, 256 or 512
    int32_t sm;      // side of the chain's matrices: 32, or sp
    int32_t panels;  // the Gram matrix is panels x panels blocks of at most 256 x 256
    int32_t splits;  // pieces of the long side, one per workgroup
    int64_t per;     // long-side rows of a piece
    int32_t blocks64, splits64;  // the fp64 Gram pass: 32 x 32 blocks of the lower triangle, pieces of the long side
    int64_t per64;               // (0: not taken)
    int64_t o_part, o_sum, o_pscale, o_mat[6], o_t, o_scale, bytes;  // A0, A, M, U, Ta, Tb; T's fp16 pieces and their scales
};

OrthoPlan make_plan(int64_t rows, int64_t cols) {
    OrthoPlan p{};
    p.r = std::max(rows, cols);
    p.s = static_cast<int32_t>(std::min(rows, cols));
    p.sp = p.s <= 64 ? 64 : p.s <= 128 ? 128 : p.s <= 256 ? 256 : 512;
    p.sm = p.s <= 32 ? 32 : p.sp;
    p.panels = p.sp > 256 ? 2 : 1;
    const int64_t kr = kStage / std::min(p.sp, 256) / p.panels, stages = ceil_div(p.r, kr);
    // One workgroup per CU at most; eight stages each, because the pieces' sums are written and read again, fewer where that
    // leaves only few pieces.
    const int64_t want = std::max<int64_t>(ceil_div(stages, 8), std::min<int64_t>(stages, kJoinDirect));
    p.splits = static_cast<int32_t>(std::min<int64_t>(256 / (p.panels * p.panels), want));
    p.per = ceil_div(stages, p.splits) * kr;
    p.splits = static_cast<int32_t>(ceil_div(p.r, p.per));
    // fp32 tables take their Gram matrix in fp64 where that costs little and the shape may be near-square (fp32 sums / fp64:
    // 1682 x 20 32.1 / 29.3 us, 512 x 512 256 / 253, 1024 x 512 261 / 263; but 6040 x 100 81 / 88, 4096 x 512 277 / 321,
    // 26744 x 128 91 / 141, and there both give the same X: a long side of four short ones and more has no small
    // singular values by chance)
    const int32_t side = p.sm / 32;
    p.blocks64 = side * (side + 1) / 2;
    if (p.r <= 2048) {
        const int64_t most = std::min(kPieces64, std::max(4, 512 / p.blocks64));
        p.per64 = round_up(ceil_div(p.r, most), 128);
        p.splits64 = static_cast<int32_t>(ceil_div(p.r, p.per64));
    }
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at += round_up(bytes, 256);
        return o;
    };
    p.o_part = take(std::max(static_cast<int64_t>(p.splits) * p.sp * p.sp * 4, static_cast<int64_t>(p.splits64) * p.sm * p.sm * 8));
    p.o_sum = take(p.splits > kJoinDirect ? static_cast<int64_t>(kJoinGroups) * p.sp * p.sp * 8 : 0);
    p.o_pscale = take(static_cast<int64_t>(p.splits) * p.panels * p.panels * 4);
    for (int64_t& o : p.o_mat) o = take(static_cast<int64_t>(p.sm) * p.sm * 8);
    p.o_t = take(static_cast<int64_t>(2) * p.sp * p.sp * 2);
    p.o_scale = take((p.sp + 1) * 4);
    p.bytes = at;
    return p;
}

// four elements of the table, consecutive along its contiguous side: long index r, short index i of the first
template <typename E, bool WIDE, bool VEC>
__device__ __forceinline__ f32x4 load4(const E* G, int64_t ld, int64_t r, int64_t r1, int i, int s) {
    typedef __attribute__((ext_vector_type(4))) E e4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (WIDE ? i >= s : r >= r1) return v;
    const E* src = G + (WIDE ? i * ld + r : r * ld + i);
    const int n = WIDE ? static_cast<int>(min<int64_t>(r1 - r, 4)) : min(s - i, 4);
    if (VEC && n >= 4) {
        const e4 x = *reinterpret_cast<const e4*>(src);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(x[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) v[e] = static_cast<float>(src[e]);
    }
    return v;
}

// element offset of a value in an LDS tile of W 16-bit columns
template <int W>
__device__ __forceinline__ int lds_at(int row, int col) {
    return LdsTile<W>::base(row, col >> 3) / 2 + (col & 7);
}

// ---- Gram matrix of a piece of the long side -----------------------------------------------------------------------
// On fp16 MFMAs, the table scaled by a power of two that follows the largest element seen (a stage four times
// larger than the last reference moves it, and the sums with it: both exact), so any magnitudes are right.  16-bit
// tables: G^T G by one product.  fp32 as pairs g = h + l: with B = h (h / 2 + l), two products, G^T G is B + B^T up to
// 2^-24 of its terms.  The long side is the contraction: the operands come from a row-major LDS stage by
// transposing reads.
// SP: columns of a panel (64, 128, 256); eight waves as WI x WJ blocks of 64 x 64 or (SP = 256) 64 x 128, NG groups
// of waves share a stage's rows.  PAN: 1, or 2 where blockIdx.y's block has different row and column panels (SP = 256).
template <typename E, bool WIDE, bool VEC, int SP, int PAN>
__global__ __launch_bounds__(kThreads) void ortho_gram_kernel(const E* __restrict__ G, int64_t ld, OrthoPlan p, float* __restrict__ part,
                                                             float* __restrict__ part_scale) {
#pragma clang fp contract(fast)
    constexpr int NP = std::is_same<E, float>::value ? 2 : 1;
    constexpr int KR = kStage / SP / PAN, WI = SP / 64, WJ = SP == 256 ? 2 : SP / 64, NG = 8 / (WI * WJ), BJ = SP / WJ / 32;
    constexpr int PIECE = KR * SP, BUF = PAN * NP * PIECE;  // 16-bit elements
    constexpr int PER = kStage / 4 / kThreads;              // groups of four elements a thread stages
    extern __shared__ __attribute__((aligned(16))) char smem[];
    _Float16* tile = reinterpret_cast<_Float16*>(smem);     // [2][PAN][NP][KR][SP]
    __shared__ uint32_t smax[2][8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lx = lane & 31, half = lane >> 5;
    const int grp = wave / (WI * WJ), wi = (wave % (WI * WJ)) / WJ * 64, wj = (wave % WJ) * (SP / WJ);
    const int pi = PAN == 2 ? blockIdx.y / p.panels : 0, pj = PAN == 2 ? blockIdx.y % p.panels : 0;
    const int64_t r0 = blockIdx.x * p.per, r1 = min(p.r, r0 + p.per);

    f32x4 sa[PER], sb[PER];  // two stages on their way: one is too little to cover memory's latency
    auto place = [&](int i, int& pan, int& row, int& col) {
        const int g = i * kThreads + threadIdx.x;
        pan = g / (PIECE / 4);
        const int q = g % (PIECE / 4);
        if (WIDE)
            row = q % (KR / 4) * 4, col = q / (KR / 4);
        else
            row = q / (SP / 4), col = q % (SP / 4) * 4;
    };
    auto fetch = [&](f32x4 (&st)[PER], int64_t rb) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int pan, row, col;
            place(i, pan, row, col);
            st[i] = load4<E, WIDE, VEC>(G, ld, rb + row, r1, (pan ? pj : pi) * 256 + col, p.s);
        }
    };
    // a stage's largest magnitude: each wave's share noted, and (a barrier later) the workgroup's
    auto note = [&](const f32x4 (&st)[PER], int slot) {
        float top = 0.f;  // (NaN passes by, an infinity makes the result one or NaN whatever the scale)
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(st[i][e]));
        const uint32_t m = wave_max_u32(__float_as_uint(top));
        if (lane == 0) smax[slot][wave] = m;
    };
    auto largest = [&](int slot) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, smax[slot][i]);
        return m;
    };
    auto put = [&](const f32x4 (&st)[PER], int b, float sc) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int pan, row, col;
            place(i, pan, row, col);
            _Float16* t = tile + b * BUF + pan * NP * PIECE;
            f16x4 h, l;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = st[i][e] * sc;  // (a power of two: exact, fused or not)
                h[e] = static_cast<_Float16>(x);
                l[e] = static_cast<_Float16>(x - static_cast<float>(h[e]));
            }
            if (WIDE) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    t[lds_at<SP>(row + e, col)] = h[e];
                    if (NP == 2) t[PIECE + lds_at<SP>(row + e, col)] = l[e];
                }
            } else {
                *reinterpret_cast<f16x4*>(t + lds_at<SP>(row, col)) = h;
                if (NP == 2) *reinterpret_cast<f16x4*>(t + PIECE + lds_at<SP>(row, col)) = l;
            }
        }
    };
    // operand: lane = column c0 + lane mod 32 of the stage, elements = its rows k0 + 8 half + (0..7)
    const int g4 = (lane & 15) >> 2, c4 = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    auto frag = [&](const _Float16* t, int k0, int c0) {
        auto rd = [&](int row) {
            return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(t + lds_at<SP>(row, c0 + c4)));
        };
        const s16x4 u = rd(k0 + 8 * half + g4), w = rd(k0 + 8 * half + 4 + g4);
        return __builtin_bit_cast(f16x8, __builtin_shufflevector(u, w, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    f32x16 acc[2][BJ];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < BJ; ++y) acc[x][y] = f32x16{0};
    // scale: 2^(12 - exponent of the reference); a stage's largest may reach 2^15.  Returns what the sums so far are to be
    // multiplied by (twice: they are products of two).
    float sc = 1.f;
    uint32_t limit = 0;  // bits of the largest magnitude the scale stands
    auto follow = [&](uint32_t m) {
        if (m <= limit) return 1.f;
        const int e = max(static_cast<int>(m >> 23), 1) - 127;
        limit = e + 3 > 127 ? 0x7F7FFFFFu : static_cast<uint32_t>(e + 3 + 127) << 23;
        const float next = __uint_as_float(static_cast<uint32_t>(min(12 - e, 126) + 127) << 23), f = next / sc;
        sc = next;
        return f;
    };
    auto multiply = [&](int b) {
        const _Float16 *ti = tile + b * BUF, *tj = ti + (PAN - 1) * NP * PIECE;
#pragma unroll
        for (int k = 0; k < KR / 16 / NG; ++k) {
            const int k0 = (k * NG + grp) * 16;
            f16x8 fi[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) fi[x] = frag(ti, k0, wi + 32 * x);
#pragma unroll
            for (int y = 0; y < BJ; ++y) {
                f16x8 j1 = frag(tj, k0, wj + 32 * y);
                if constexpr (NP == 2) j1 *= static_cast<_Float16>(0.5f);
#pragma unroll
                for (int x = 0; x < 2; ++x) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fi[x], j1, acc[x][y], 0, 0, 0);
                if constexpr (NP == 2) {
                    const f16x8 j2 = frag(tj + PIECE, k0, wj + 32 * y);
#pragma unroll
                    for (int x = 0; x < 2; ++x) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fi[x], j2, acc[x][y], 0, 0, 0);
                }
            }
        }
    };
    // Stage i in LDS, i + 1 in `ready` (its largest noted), i + 2 on its way in `other`: one barrier a stage.
    auto step = [&](int64_t rb, int b, f32x4 (&ready)[PER], f32x4 (&other)[PER]) {
        float f = 1.f;
        if (rb + KR < r1) {
            f = follow(largest(b ^ 1));
            put(ready, b ^ 1, sc);
            if (rb + 3 * KR < r1) fetch(ready, rb + 3 * KR);
        }
        multiply(b);
        if (f != 1.f)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int y = 0; y < BJ; ++y)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[x][y][i] = acc[x][y][i] * f * f;
        if (rb + 2 * KR < r1) note(other, b);
        __syncthreads();
    };
    fetch(sa, r0);
    if (r0 + KR < r1) fetch(sb, r0 + KR);
    note(sa, 0);
    __syncthreads();
    follow(largest(0));
    put(sa, 0, sc);
    if (r0 + 2 * KR < r1) fetch(sa, r0 + 2 * KR);
    if (r0 + KR < r1) note(sb, 1);
    __syncthreads();
    for (int64_t rb = r0; rb < r1; rb += 2 * KR) {
        step(rb, 0, sb, sa);
        if (rb + KR < r1) step(rb + KR, 1, sa, sb);
    }
    if (threadIdx.x == 0) part_scale[blockIdx.y * gridDim.x + blockIdx.x] = sc;
    // the groups' sums, halving their number through LDS
    float* red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int n = NG / 2; n; n /= 2) {
        float* slot = red + ((grp % n) * (SP * SP)) + ((wave % (WI * WJ)) * 2 * BJ) * 1024;
        if (grp >= n && grp < 2 * n)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int y = 0; y < BJ; ++y)
#pragma unroll
                    for (int e = 0; e < 16; ++e) slot[((x * BJ + y) * 16 + e) * 64 + lane] = acc[x][y][e];
        __syncthreads();
        if (grp < n)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int y = 0; y < BJ; ++y)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[x][y][e] += slot[((x * BJ + y) * 16 + e) * 64 + lane];
        __syncthreads();
    }
    if (grp) return;
    float* o = part + static_cast<int64_t>(blockIdx.x) * p.sp * p.sp + static_cast<int64_t>(pi * 256) * p.sp + pj * 256;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < BJ; ++y)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                o[static_cast<int64_t>(wi + 32 * x + 8 * (e / 4) + 4 * half + e % 4) * p.sp + wj + 32 * y + lx] = acc[x][y][e];
}

// Sums of groups of the pieces in fp64, where there are many: a thread per four entries, blockIdx.y a group.
__global__ __launch_bounds__(256) void ortho_gram_sum_kernel(const float* __restrict__ part, const float* __restrict__ part_scale, OrthoPlan p,
                                                            double* __restrict__ out) {
    const int64_t step = static_cast<int64_t>(p.sp) * p.sp, at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
    const int i = static_cast<int>(at / p.sp), j = static_cast<int>(at % p.sp);
    const float* sc = part_scale + (i / 256 * p.panels + j / 256) * p.splits;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    const int n0 = p.splits * static_cast<int>(blockIdx.y) / kJoinGroups, n1 = p.splits * (static_cast<int>(blockIdx.y) + 1) / kJoinGroups;
#pragma unroll 8
    for (int n = n0; n < n1; ++n) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(part + n * step + at);
        const double a = 1.0 / sc[n];  // (a power of two)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += static_cast<double>(x[e]) * (a * a);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) out[blockIdx.y * step + at + e] = s[e];
}

// A0 = sum of the pieces' B + B^T (16-bit tables: their half) in fp64, in the pieces' order; a 16 x 16 block and its
// mirror per workgroup, four groups of 256 threads share the pieces.  P: float pieces with their scales, or the sums of
// groups of them.
template <typename P>
__global__ __launch_bounds__(1024) void ortho_gram_join_kernel(const P* __restrict__ part, const float* __restrict__ part_scale,
                                                              OrthoPlan p, int pieces, double scale, double* __restrict__ A) {
    __shared__ double sm[2][4][16][17];
    int ib = 0, t = blockIdx.x;
    while (t > ib) t -= ++ib;  // block t of the lower triangle: row ib, column t
    const int jb = t, g = threadIdx.x >> 8, i = (threadIdx.x >> 4) & 15, j = threadIdx.x & 15;
    const P *u = part + static_cast<int64_t>(ib * 16 + i) * p.sp + jb * 16 + j, *v = part + static_cast<int64_t>(jb * 16 + i) * p.sp + ib * 16 + j;
    const float *us = part_scale + (ib / 16 * p.panels + jb / 16) * p.splits, *vs = part_scale + (jb / 16 * p.panels + ib / 16) * p.splits;
    const int64_t step = static_cast<int64_t>(p.sp) * p.sp;
    double su = 0.0, sv = 0.0;
    const int n0 = pieces * g / 4, n1 = pieces * (g + 1) / 4;
#pragma unroll 4
    for (int n = n0; n < n1; ++n) {
        double a = 1.0, b = 1.0;
        if constexpr (std::is_same<P, float>::value) a = 1.0 / us[n], b = 1.0 / vs[n];  // (powers of two)
        su += static_cast<double>(u[n * step]) * (a * a);
        sv += static_cast<double>(v[n * step]) * (b * b);
    }
    sm[0][g][i][j] = su;
    sm[1][g][i][j] = sv;
    __syncthreads();
    if (g) return;
    auto sum = [&](int w, int x, int y) { return ((sm[w][0][x][y] + sm[w][1][x][y]) + sm[w][2][x][y]) + sm[w][3][x][y]; };
    const double a = (sum(0, i, j) + sum(1, j, i)) * scale;
    A[static_cast<int64_t>(ib * 16 + i) * p.sm + jb * 16 + j] = a;
    if (ib != jb) A[static_cast<int64_t>(jb * 16 + j) * p.sm + ib * 16 + i] = a;
}

// ---- Gram matrix in fp64 (fp32 tables of a shorter long side) -------------------------------------------------------
// The products of fp32 elements are exact.  Small singular values are lost in fp32 sums: their share of a near-square
// update comes out up to a^steps = 486 times larger, with the sums' errors (random 10 x 12: 2.2e-6 of X with fp32 sums,
// 2.6e-7 with these; 40 x 40: 1.0e-5 and 8.0e-7; the steps themselves in fp32: 5.1e-7 and 9.0e-7).  A workgroup takes
// 32 x 32 entries of the lower triangle from a piece of the long side, its waves every fourth 32 rows, straight from
// memory: 32 loads feed 32 products of 64 cycles.
template <bool WIDE>
__global__ __launch_bounds__(256) void ortho_gram64_kernel(const float* __restrict__ G, int64_t ld, OrthoPlan p, double* __restrict__ part) {
    __shared__ double sm[3][16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lc = lane & 15, lk = lane >> 4;
    int ib = 0, t = blockIdx.x;
    while (t > ib) t -= ++ib;  // block t of the lower triangle: row ib, column t
    const int i0 = ib * 32, j0 = t * 32;
    const int64_t r0 = blockIdx.y * p.per64, r1 = min(p.r, r0 + p.per64);
    f64x4 acc[2][2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) acc[x][y] = f64x4{0};
    auto load = [&](int64_t r, int i) { return r < r1 && i < p.s ? G[WIDE ? i * ld + r : r * ld + i] : 0.f; };
    for (int64_t rb = r0 + wave * 32; rb < r1; rb += 128) {
        float a[2][8], b[2][8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int64_t r = rb + (WIDE ? lk * 8 + u : u * 4 + lk);  // (any order of the rows, the same for both)
                a[x][u] = load(r, i0 + 16 * x + lc);
                b[x][u] = load(r, j0 + 16 * x + lc);
            }
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y)
                    acc[x][y] = __builtin_amdgcn_mfma_f64_16x16x4f64(static_cast<double>(a[x][u]), static_cast<double>(b[y][u]), acc[x][y], 0, 0, 0);
    }
    if (wave)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int e = 0; e < 4; ++e) sm[wave - 1][(x * 2 + y) * 4 + e][lane] = acc[x][y][e];
    __syncthreads();
    if (wave) return;
    double* o = part + static_cast<int64_t>(blockIdx.y) * p.sm * p.sm;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int q = (x * 2 + y) * 4 + e;
                o[static_cast<int64_t>(i0 + 16 * x + 4 * e + lk) * p.sm + j0 + 16 * y + lc] = ((acc[x][y][e] + sm[0][q][lane]) + sm[1][q][lane]) + sm[2][q][lane];
            }
}

// A0 from the pieces' lower triangles, in their order; a thread per entry
__global__ __launch_bounds__(256) void ortho_join64_kernel(const double* __restrict__ part, OrthoPlan p, double* __restrict__ A) {
    const int at = blockIdx.x * 256 + threadIdx.x, i = at / p.sm, j = at % p.sm;
    const bool lower = i / 32 >= j / 32;
    const double* src = part + (lower ? at : static_cast<int64_t>(j) * p.sm + i);
    const int64_t step = static_cast<int64_t>(p.sm) * p.sm;
    double x[kPieces64], sum = 0.0;
#pragma unroll
    for (int n = 0; n < kPieces64; ++n) x[n] = n < p.splits64 ? src[n * step] : 0.0;
#pragma unroll
    for (int n = 0; n < kPieces64; ++n) sum += x[n];
    A[at] = sum;
}

// trace of A0 over a block of N threads (the same sum in every block)
template <int N>
__device__ __forceinline__ double block_trace(const double* A0, const OrthoPlan& p) {
    __shared__ double sm[N / 64];
    double t = 0.0;
    for (int i = threadIdx.x; i < p.s; i += N) t += A0[static_cast<int64_t>(i) * p.sm + i];
#pragma unroll
    for (int o = 32; o; o >>= 1) t += __shfl_xor(t, o);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = t;
    __syncthreads();
    t = 0.0;
#pragma unroll
    for (int i = 0; i < N / 64; ++i) t += sm[i];
    __syncthreads();
    return t;
}

// ---- S x S products of symmetric, commuting matrices: C = X Y, 16 x 16 per workgroup, its four waves share k.  C is
// symmetric too: of 512 x 512, where the operands' reads through L2 bound it, only the blocks of the lower triangle
// are formed and mirrored (all steps of a 512 x 512 update 253 -> 201 us; of 128 x 128 and 256 x 256, where latency
// does, all blocks: 81 us against 83 and 6.0 us a product against 6.2).
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

template <bool LOWER>  // only the lower triangle's blocks, by blockIdx.x
__global__ __launch_bounds__(256) void ortho_chain_kernel(ChainArgs q) {
    __shared__ double sm[3][4][64];
    const int sm_ = q.p.sm, z = blockIdx.z;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lc = lane & 15, lk = lane >> 4;
    int ib = blockIdx.x, jb = blockIdx.y;
    if (LOWER)  // block x of the lower triangle: row ib, column jb
        for (ib = 0, jb = blockIdx.x; jb > ib;) jb -= ++ib;
    const int i0 = ib * 16, j0 = jb * 16, kq = sm_ / 4;
    // X and Y are symmetric: both operands are read along rows k
    const double *X = q.X[z] + static_cast<int64_t>(wave * kq + lk) * sm_ + i0 + lc, *Y = q.Y[z] + static_cast<int64_t>(wave * kq + lk) * sm_ + j0 + lc;
    // (the epilogue's values of X are on their way during the product: 3.9 us a product of 128 x 128, 4.1 read after it)
    const int64_t out = static_cast<int64_t>(i0 + lk) * sm_ + j0 + lc;  // the lane's first entry, the others 4 rows apart
    double x[4] = {0.0, 0.0, 0.0, 0.0};
    if (q.poly && z == 0 && wave == 0)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = q.X[0][out + static_cast<int64_t>(4 * e) * sm_];
    f64x4 acc = f64x4{0};
    for (int k = 0; k < kq; k += 32) {
        double a[8], b[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (k + 4 * u < kq) {
                a[u] = X[static_cast<int64_t>(k + 4 * u) * sm_];
                b[u] = Y[static_cast<int64_t>(k + 4 * u) * sm_];
            }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (k + 4 * u < kq) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(a[u], b[u], acc, 0, 0, 0);
    }
    double inv = 1.0;
    if (q.normalise && z == 0) {
        const double tr = block_trace<256>(q.A0, q.p);
        inv = tr == 0.0 ? 0.0 : 1.0 / tr;
    }
    if (wave)
#pragma unroll
        for (int e = 0; e < 4; ++e) sm[wave - 1][e][lane] = acc[e];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        double v = (((acc[e] + sm[0][e][lane]) + sm[1][e][lane]) + sm[2][e][lane]) * inv;
        if (q.poly && z == 0) v = (i0 + 4 * e + lk == j0 + lc ? q.a : 0.0) + q.b * x[e] * inv + q.c * (v * inv);
        q.C[z][out + static_cast<int64_t>(4 * e) * sm_] = v;
        if (LOWER && i0 != j0) q.C[z][static_cast<int64_t>(j0 + lc) * sm_ + i0 + 4 * e + lk] = v;
    }
}

// The whole chain in one workgroup, its matrices in LDS: SM = 32 (four waves), 64 (sixteen), a 16 x 16 block each.  The
// steps between products cost a barrier instead of a launch.
template <int SM>
__global__ __launch_bounds__(SM * SM / 4) void ortho_small_chain_kernel(OrthoPlan p, const double* A0, double* T, int steps, double a, double b, double c) {
    constexpr int N = SM * SM / 4, LD = SM + 1;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    double* mat = reinterpret_cast<double*>(smem);  // A, M, U, T of SM x LD
    double *A = mat, *M = mat + SM * LD, *U = M + SM * LD, *Tl = U + SM * LD;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lc = lane & 15, lk = lane >> 4;
    const int i0 = wave / (SM / 16) * 16, j0 = wave % (SM / 16) * 16;
    const double tr = block_trace<N>(A0, p), inv = tr == 0.0 ? 0.0 : 1.0 / tr;
    for (int e = threadIdx.x; e < SM * SM; e += N) A[e / SM * LD + e % SM] = A0[e] * inv;
    __syncthreads();
    auto product = [&](const double* X, const double* Y) {
        f64x4 acc = f64x4{0};
#pragma unroll
        for (int k = 0; k < SM; k += 4) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(X[(k + lk) * LD + i0 + lc], Y[(k + lk) * LD + j0 + lc], acc, 0, 0, 0);
        return acc;
    };
    auto write = [&](double* C, f64x4 v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) C[(i0 + 4 * e + lk) * LD + j0 + lc] = v[e];
    };
    for (int j = 0; j < steps; ++j) {
        f64x4 v = product(A, A);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int x = i0 + 4 * e + lk, y = j0 + lc;
            v[e] = (x == y ? a : 0.0) + b * A[x * LD + y] + c * v[e];
        }
        write(M, v);
        if (j == 0) write(Tl, v);
        __syncthreads();
        const bool last = j + 1 == steps;
        f64x4 u = f64x4{0}, t = f64x4{0};
        if (!last) u = product(A, M);
        if (j) t = product(Tl, M);
        if (!last) write(U, u);
        __syncthreads();
        if (j) write(Tl, t);
        if (!last) v = product(U, M), write(A, v);
        __syncthreads();
    }
    for (int e = threadIdx.x; e < SM * SM; e += N) T[e] = Tl[e / SM * LD + e % SM];
}

// T as two fp16 pieces, each row (T is symmetric: each column) scaled by a power of two to below 2^14; scale[j] takes an
// element of G T back and divides by |G|, scale[sp] is the power of two that brings G below 2^14.  A wave per row.
__global__ __launch_bounds__(64) void ortho_pack_kernel(OrthoPlan p, const double* __restrict__ A0, const double* __restrict__ T,
                                                       _Float16* __restrict__ tp, float* __restrict__ scale) {
    const int j = blockIdx.x, lane = threadIdx.x;
    double tr = 0.0;
    for (int i = lane; i < p.s; i += 64) tr += A0[static_cast<int64_t>(i) * p.sm + i];
#pragma unroll
    for (int o = 32; o; o >>= 1) tr += __shfl_xor(tr, o);
    const double norm = sqrt(tr);
    auto power = [](int e) { return __uint_as_float(static_cast<uint32_t>(min(max(e, -126), 127) + 127) << 23); };
    int eg = 0;
    if (norm > 0.0 && norm < 1e300) eg = 13 - ilogb(norm);
    eg = min(max(eg, -126), 126);
    double m = 0.0;
    if (j < p.sm)
        for (int i = lane; i < p.sm; i += 64) m = fmax(m, fabs(T[static_cast<int64_t>(j) * p.sm + i]));
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmax(m, __shfl_xor(m, o));
    int et = 0;
    if (m > 0.0 && m < 1e300) et = 13 - ilogb(m);
    et = min(max(et, -120), 120);
    const double st = ldexp(1.0, et);
    for (int i = lane; i < p.sp; i += 64) {
        const double v = j < p.sm && i < p.sm ? T[static_cast<int64_t>(j) * p.sm + i] * st : 0.0;
        const _Float16 h = static_cast<_Float16>(static_cast<float>(v));
        tp[static_cast<int64_t>(j) * p.sp + i] = h;
        tp[static_cast<int64_t>(p.sp + j) * p.sp + i] = static_cast<_Float16>(static_cast<float>(v - static_cast<double>(static_cast<float>(h))));
    }
    if (lane == 0) {
        // G = 0: X = 0.  The product of the two powers and 1 / |G| is near 1 / (2^13 2^13): formed in fp64.
        scale[j] = norm == 0.0 ? 0.f : static_cast<float>(ldexp(1.0, -et - eg) / norm);
        if (j == 0) scale[p.sp] = power(eg);
    }
}

// ---- X = G T / |G| -------------------------------------------------------------------------------------------------
// Each wave keeps 32 columns of T in registers (both pieces) for all its rows of G; a tile of G passes through LDS as fp16
// (fp32: pairs) that all waves read: the table is read once from memory and X written once.  Products: hi T1 + hi T2
// + lo T1.  G has one scale, so lo is held kLowUp times its value and meets T1 / kLowUp: fp16 ends at 2^-24, and rows of
// 2^-15 of |G| and less would lose their second piece there (to 2^-38 of |G|; now 2^-49).  Sums of their own for the
// small products instead: 200000 x 512 fp32 1.49 ms against 1.29.  SP: short side; KS = SP / 16 steps; WC waves cover the
// columns of a workgroup (all of them up to 256).
template <typename E, bool WIDE, bool VEC, int SP, int THREADS>
__global__ __launch_bounds__(THREADS) void ortho_apply_kernel(const E* G, int64_t ldg, OrthoPlan p, const _Float16* __restrict__ tp,
                                                             const float* __restrict__ scale, E* X, int64_t ldx) {
#pragma clang fp contract(fast)
    constexpr int NP = std::is_same<E, float>::value ? 2 : 1;
    constexpr int WAVES = THREADS / 64, WC = SP / 32 < WAVES ? SP / 32 : WAVES, NG = WAVES / WC, KS = SP / 16;
    constexpr int TR = 32 * NG, PIECE = TR * SP, PER = PIECE / 4 / THREADS;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    _Float16* tile = reinterpret_cast<_Float16*>(smem);  // [2][NP][TR][SP]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lx = lane & 31, half = lane >> 5;
    const int grp = wave / WC, j0 = blockIdx.y * (WC * 32) + wave % WC * 32;
    const float gscale = scale[p.sp];
    f16x8 t[2][KS];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int k = 0; k < KS; ++k) t[q][k] = *reinterpret_cast<const f16x8*>(tp + (static_cast<int64_t>(q) * SP + j0 + lx) * SP + k * 16 + half * 8);
    constexpr bool kTwo = SP <= 256;  // two tiles on their way; SP = 512: T takes the registers, one
    f32x4 sa[PER], sb[kTwo ? PER : 1];
    auto place = [&](int i, int& row, int& col) {
        const int g = i * THREADS + threadIdx.x;
        if (WIDE)
            row = g % (TR / 4) * 4, col = g / (TR / 4);
        else
            row = g / (SP / 4), col = g % (SP / 4) * 4;
    };
    auto fetch = [&](f32x4 (&st)[PER], int64_t r0) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int row, col;
            place(i, row, col);
            st[i] = load4<E, WIDE, VEC>(G, ldg, r0 + row, p.r, col, p.s);
        }
    };
    auto put = [&](const f32x4 (&st)[PER], int b) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int row, col;
            place(i, row, col);
            _Float16* d = tile + b * NP * PIECE;
            f16x4 h, l;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = st[i][e] * gscale;  // (a power of two: exact, fused or not)
                h[e] = static_cast<_Float16>(x);
                l[e] = static_cast<_Float16>((x - static_cast<float>(h[e])) * kLowUp);
            }
            if (WIDE) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    d[lds_at<SP>(row + e, col)] = h[e];
                    if (NP == 2) d[PIECE + lds_at<SP>(row + e, col)] = l[e];
                }
            } else {
                *reinterpret_cast<f16x4*>(d + lds_at<SP>(row, col)) = h;
                if (NP == 2) *reinterpret_cast<f16x4*>(d + PIECE + lds_at<SP>(row, col)) = l;
            }
        }
    };
    const int64_t tiles = (p.r + TR - 1) / TR, hop = gridDim.x;
    const float back = scale[j0 + lx];  // what takes a column's sums back
    // a tile in LDS, the next one in `ready`, the one after it fetched into `other`
    auto step = [&](int64_t it, int b, f32x4 (&ready)[PER], f32x4 (&other)[PER]) {
        const int64_t ahead = it + (kTwo ? 2 : 1) * hop;
        if (ahead < tiles) fetch(other, ahead * TR);
        // (both bases taken anew for every tile: kept for all 16 stores and the reads they would cost the registers of T)
        int rb = LdsTile<SP>::base(grp * 32 + lx, half) + b * NP * PIECE * 2;
        E* out = X + (WIDE ? (j0 + 4 * half) * ldx + it * TR + grp * 32 + lx : (it * TR + grp * 32 + 4 * half) * ldx + j0 + lx);
        asm volatile("" : "+v"(rb), "+v"(out));
        f32x16 acc = f32x16{0};
        // lanes run along the contiguous side of X
        auto mm = [&](f16x8 u, f16x8 v) {
            acc = WIDE ? __builtin_amdgcn_mfma_f32_32x32x16_f16(v, u, acc, 0, 0, 0) : __builtin_amdgcn_mfma_f32_32x32x16_f16(u, v, acc, 0, 0, 0);
        };
        int down = 0x1000;  // 1 / kLowUp, unknown to the compiler: it would keep T times it beside T
        asm volatile("" : "+v"(down));
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            f16x8 g[NP];
#pragma unroll
            for (int q = 0; q < NP; ++q) g[q] = *reinterpret_cast<const f16x8*>(smem + q * PIECE * 2 + LdsTile<SP>::at(rb, 2 * k));
            mm(g[0], t[0][k]);
            mm(g[0], t[1][k]);
            if constexpr (NP == 2) mm(g[1], t[0][k] * __builtin_bit_cast(_Float16, static_cast<short>(down)));
        }
        if (it + hop < tiles) put(ready, b ^ 1);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int o = 8 * (e / 4) + e % 4;  // rows (WIDE: columns) past the first of the lane's
            const int64_t r = it * TR + grp * 32 + (WIDE ? lx : 4 * half + o);
            const int j = j0 + (WIDE ? 4 * half + o : lx);
            if (r < p.r && j < p.s) out[o * ldx] = static_cast<E>(acc[e] * (WIDE ? scale[j] : back));
        }
        __syncthreads();
    };
    const int64_t first = blockIdx.x;
    if (first < tiles) fetch(sa, first * TR);
    if constexpr (kTwo)
        if (first + hop < tiles) fetch(sb, (first + hop) * TR);
    if (first < tiles) put(sa, 0);
    __syncthreads();
    for (int64_t it = first; it < tiles; it += 2 * hop) {
        if constexpr (kTwo) {
            step(it, 0, sb, sa);
            if (it + hop < tiles) step(it + hop, 1, sa, sb);
        } else {
            step(it, 0, sa, sa);
            if (it + hop < tiles) step(it + hop, 1, sa, sa);
        }
    }
}

template <typename K, typename... A>
void launch_lds(K kern, dim3 grid, int threads, int lds, hipStream_t st, A... args) {
    if (lds > 64 * 1024)
        RS_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    kern<<<grid, threads, lds, st>>>(args...);
    RS_HIP(hipGetLastError());
}

template <typename E, bool WIDE, bool VEC>
void run(const OrthoPlan& p, const E* G, int64_t ldg, int32_t steps, double a, double b, double c, E* X, int64_t ldx, char* ws,
         hipStream_t st) {
    constexpr bool kF32 = std::is_same<E, float>::value;
    float* part = reinterpret_cast<float*>(ws + p.o_part);
    float* part_scale = reinterpret_cast<float*>(ws + p.o_pscale);
    double* mat[6];
    for (int i = 0; i < 6; ++i) mat[i] = reinterpret_cast<double*>(ws + p.o_mat[i]);
    double *A0 = mat[0], *M = mat[2], *U = mat[3], *T = mat[4], *T2 = mat[5];
    _Float16* tp = reinterpret_cast<_Float16*>(ws + p.o_t);
    float* scale = reinterpret_cast<float*>(ws + p.o_scale);

    const uint32_t t = static_cast<uint32_t>(p.sm / 16);
    bool exact = false;
    if constexpr (kF32) {
        exact = p.per64 > 0;
        if (exact) {
            ortho_gram64_kernel<WIDE><<<dim3(static_cast<uint32_t>(p.blocks64), static_cast<uint32_t>(p.splits64)), 256, 0, st>>>(
                G, ldg, p, reinterpret_cast<double*>(part));
            RS_HIP(hipGetLastError());
            ortho_join64_kernel<<<static_cast<uint32_t>(p.sm * p.sm / 256), 256, 0, st>>>(reinterpret_cast<const double*>(part), p, A0);
            RS_HIP(hipGetLastError());
        }
    }
    if (!exact) {
        const int glds = 2 * (kF32 ? 2 : 1) * kStage * 2;
        const dim3 ggrid(static_cast<uint32_t>(p.splits), static_cast<uint32_t>(p.panels * p.panels));
        // (the groups' sums take up to 64 KB of the same LDS)
        if (p.sp == 64)
            launch_lds(ortho_gram_kernel<E, WIDE, VEC, 64, 1>, ggrid, kThreads, std::max(glds, 65536), st, G, ldg, p, part, part_scale);
        else if (p.sp == 128)
            launch_lds(ortho_gram_kernel<E, WIDE, VEC, 128, 1>, ggrid, kThreads, std::max(glds, 65536), st, G, ldg, p, part, part_scale);
        else if (p.sp == 256)
            launch_lds(ortho_gram_kernel<E, WIDE, VEC, 256, 1>, ggrid, kThreads, glds, st, G, ldg, p, part, part_scale);
        else
            launch_lds(ortho_gram_kernel<E, WIDE, VEC, 256, 2>, ggrid, kThreads, glds, st, G, ldg, p, part, part_scale);
        if (p.splits > kJoinDirect) {
            double* sums = reinterpret_cast<double*>(ws + p.o_sum);
            ortho_gram_sum_kernel<<<dim3(static_cast<uint32_t>(p.sp * p.sp / 1024), kJoinGroups), 256, 0, st>>>(part, part_scale, p, sums);
            RS_HIP(hipGetLastError());
            ortho_gram_join_kernel<double><<<t * (t + 1) / 2, 1024, 0, st>>>(sums, part_scale, p, kJoinGroups, kF32 ? 1.0 : 0.5, A0);
        } else {
            ortho_gram_join_kernel<float><<<t * (t + 1) / 2, 1024, 0, st>>>(part, part_scale, p, p.splits, kF32 ? 1.0 : 0.5, A0);
        }
        RS_HIP(hipGetLastError());
    }

    if (p.sm == 32) {
        launch_lds(ortho_small_chain_kernel<32>, dim3(1), 256, 4 * 32 * 33 * 8, st, p, static_cast<const double*>(A0), T, steps, a, b, c);
    } else if (p.sm == 64) {
        launch_lds(ortho_small_chain_kernel<64>, dim3(1), 1024, 4 * 64 * 65 * 8, st, p, static_cast<const double*>(A0), T, steps, a, b, c);
    } else {
        ChainArgs q{};
        q.p = p, q.A0 = A0, q.a = a, q.b = b, q.c = c;
        auto product = [&](int z) {
            if (p.sm == 512)
                ortho_chain_kernel<true><<<dim3(t * (t + 1) / 2, 1, static_cast<uint32_t>(z)), 256, 0, st>>>(q);
            else
                ortho_chain_kernel<false><<<dim3(t, t, static_cast<uint32_t>(z)), 256, 0, st>>>(q);
            RS_HIP(hipGetLastError());
        };
        const double* A = A0;
        for (int j = 0; j < steps; ++j) {
            const bool last = j + 1 == steps;
            q.normalise = j == 0;
            double* Mj = j == 0 ? T : M;  // T = M_0
            q.poly = 1;
            q.X[0] = q.Y[0] = A, q.C[0] = Mj;
            product(1);
            q.poly = 0;
            // A M (not after the last step) and T M (not in the first)
            int z = 0;
            if (!last) q.X[z] = A, q.Y[z] = Mj, q.C[z] = U, ++z;
            if (j) q.X[z] = T, q.Y[z] = Mj, q.C[z] = T2, ++z;
            if (z) product(z);
            if (j) std::swap(T, T2);
            if (last) break;
            q.normalise = 0;
            q.X[0] = U, q.Y[0] = Mj, q.C[0] = mat[1];
            product(1);
            A = mat[1];
        }
    }
    ortho_pack_kernel<<<static_cast<uint32_t>(p.sp), 64, 0, st>>>(p, A0, T, tp, scale);
    RS_HIP(hipGetLastError());

    auto apply = [&](auto sp, auto threads) {
        constexpr int SP = decltype(sp)::value, N = decltype(threads)::value;
        constexpr int WC = SP / 32 < N / 64 ? SP / 32 : N / 64, TR = 32 * (N / 64 / WC);
        const uint32_t blocks = static_cast<uint32_t>(std::min<int64_t>(ceil_div(p.r, TR), SP == 512 ? 64 : 256));
        launch_lds(ortho_apply_kernel<E, WIDE, VEC, SP, N>, dim3(blocks, SP / (WC * 32)), N, 2 * (kF32 ? 2 : 1) * TR * SP * 2, st, G, ldg, p,
                   static_cast<const _Float16*>(tp), static_cast<const float*>(scale), X, ldx);
    };
    using std::integral_constant;
    if (p.sp == 64)
        apply(integral_constant<int, 64>{}, integral_constant<int, 512>{});
    else if (p.sp == 128)
        apply(integral_constant<int, 128>{}, integral_constant<int, 512>{});
    else if (p.sp == 256)
        apply(integral_constant<int, 256>{}, integral_constant<int, 512>{});
    else
        apply(integral_constant<int, 512>{}, integral_constant<int, 256>{});
}

// whether two matrices share memory (columns of one table beside each other do not)
bool overlap(const void* G, int64_t ldg, const void* X, int64_t ldx, int64_t rows, int64_t cols, int64_t elem) {
    const uintptr_t g = reinterpret_cast<uintptr_t>(G), x = reinterpret_cast<uintptr_t>(X);
    const uintptr_t ge = g + ((rows - 1) * ldg + cols) * elem, xe = x + ((rows - 1) * ldx + cols) * elem;
    if (g >= xe || x >= ge) return false;
    if (ldg != ldx) return true;
    const int64_t m = static_cast<int64_t>((x > g ? x - g : g - x) / elem) % ldg;
    return m < cols || m > ldg - cols;
}

std::string check_sizes(int64_t rows, int64_t cols) {
    if (rows < 0 || rows > INT32_MAX - 1024) return "rows out of range";
    if (cols < 0 || cols > INT32_MAX - 1024) return "cols out of range";
    return std::string();
}

}  // namespace
}  // namespace rs

extern "C" int rs_orthogonalize_workspace(rs_ctx* ctx, int64_t rows, int64_t cols, int64_t* bytes) {
    return rs::no_throw([&]() -> int {
        if (!bytes) return rs::set_error(ctx, RS_ERR_INVALID, "bytes is NULL");
        *bytes = 0;
        const std::string bad = rs::check_sizes(rows, cols);
        if (!bad.empty()) return rs::set_error(ctx, RS_ERR_INVALID, bad);
        if (std::min(rows, cols) > RS_DENSE_MAX_FACTORS)
            return rs::set_error(ctx, RS_ERR_UNSUPPORTED, "the shorter side must be at most 512");
        if (rows && cols) *bytes = rs::make_plan(rows, cols).bytes;
        return RS_OK;
    });
}

extern "C" int rs_orthogonalize(rs_ctx* ctx, int32_t type, int64_t rows, int64_t cols, const void* G, int64_t ldg, int32_t steps,
                                double a, double b, double c, void* X, int64_t ldx, void* ws, int64_t ws_bytes, void* stream) {
    return rs::no_throw([&]() -> int {
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
        if (G != X && overlap(G, ldg, X, ldx, rows, cols, type_size(type)))
            return set_error(ctx, RS_ERR_INVALID, "X overlaps G");
        if (G == X && std::min(rows, cols) > 256) return set_error(ctx, RS_ERR_UNSUPPORTED, "X may be G only where the shorter side is at most 256");
        const OrthoPlan p = make_plan(rows, cols);
        if (!ws || reinterpret_cast<uintptr_t>(ws) % 16) return set_error(ctx, RS_ERR_INVALID, "ws is NULL or not 16-byte aligned");
        if (ws_bytes < p.bytes)
            return set_error(ctx, RS_ERR_INVALID, "ws holds " + std::to_string(ws_bytes) + " bytes, " + std::to_string(p.bytes) + " needed");
        return dense_guard(ctx, [&]() -> int {
            const hipStream_t st = pick_stream(ctx, stream);
            with_type(type, [&](auto e) {
                using E = typename decltype(e)::type;
                // four elements at once where every row starts on a multiple of four
                const bool vec = reinterpret_cast<uintptr_t>(G) % (4 * sizeof(E)) == 0 && ldg % 4 == 0;
                auto go = [&](auto wide, auto v) {
                    run<E, decltype(wide)::value, decltype(v)::value>(p, static_cast<const E*>(G), ldg, steps, a, b, c, static_cast<E*>(X), ldx,
                                                                      static_cast<char*>(ws), st);
                };
                if (rows >= cols)
                    vec ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
                else
                    vec ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
            });
            return RS_OK;
        });
    });
}
