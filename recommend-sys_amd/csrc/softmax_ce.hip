// softmax_ce.hip -- softmax cross entropy over the item catalogue and its gradient, no logits kept (gfx950).
//
// Mathematics.  With x the "stationary" rows held by a wave and y the rows that stream past:
//   forward: x = users' rows, y = items.  S[y, x] = W_y . H_x; a running maximum m_x and sum s_x of 2^(l2 - m_x), l2 the
//     logit in base 2, and (for the gradient) O_x = sum_y 2^(l2 - m_x) W_y, all three rescaled when m_x grows.  So one
//     pass over the catalogue gives lse and dH = weight (O / s - W_target).
//   dW: x = items, y = users' rows.  S is computed again, c = weight (2^(l2 - lse2) - [target]) and dW_x += sum_y c H_y.
// Both are one kernel: S = Y X^T, then acc[k, x] += Y^T f(S).  S comes out of the matrix unit with x over lanes and y
// over registers, which is (up to an order of y, the same for both operands) what the second product takes as its
// second operand: f(S) never leaves the registers.  Its first operand Y^T comes from the same LDS tile as Y by
// transposing LDS reads.
//
// Operands are packed into the workspace first: rows padded to tiles and columns to KP with zeros, withdrawn items
// and rows without a known target zeroed (so NaN or garbage in them reaches no product), as fp16 of the matrix scaled by
// a power of two.  bf16's 8 bits fit fp16's 11: the products are those of bf16, but the coefficients f(S) keep 11 bits
// where bf16 MFMAs would round them to 8 (dW's error then was 1.5 times that of its own rounding).  fp32 is split into
// two pieces hi + lo (each rounds its rest: 2^-24 of the element is left); the product of two such is
// hi hi + hi lo + lo hi, three fp16 MFMAs (2.5 PF / 3) where an fp32 MFMA would run at 157 TF.
#include <hip/hip_runtime.h>

#include <cmath>

#include "dense.hpp"

namespace rs {
namespace {

constexpr int kTileX = 128;      // stationary rows of a workgroup (4 waves of 32)
constexpr int kTileY = 32;       // streamed rows of a step
constexpr int kMaxBlocks = 256;  // blocks of the maxima pass, per matrix
constexpr float kShift = 14.f;   // p is held as 2^14 p: fp16's range below 1 is short
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

enum Mode { kLoss = 0, kLossGrad = 1, kItems = 2 };

// Device scalars (ws): the powers of two that scale H, W and the weights, and what undoes them.
struct Scal {
    float hs, wsc, cs;   // H, W, weights are multiplied by these
    float logit;         // S -> base-2 logit: log2(e) / (hs wsc)
    float inv_w;         // 1 / wsc
    float inv_dw;        // 1 / (cs hs)
    float inv_cs;        // 1 / cs
};

struct CePlan {
    int64_t n, v, n_pad, v_pad;
    int32_t k, kp, np, oc, z, type, grad;
    int32_t splits_f, tiles_f, splits_w, tiles_w;  // splits of the streamed rows and their tiles each
    int64_t o_max, o_scal, o_h, o_w, o_bias, o_m, o_s, o_lse2, o_wv, o_tgt, o_part, o_db, bytes;
};

CePlan make_plan(int32_t type, int64_t n, int64_t v, int32_t k, int32_t grad) {
    CePlan p{};
    p.n = n, p.v = v, p.k = k, p.type = type, p.grad = grad;
    p.kp = k <= 32 ? 32 : k <= 64 ? 64 : k <= 128 ? 128 : k <= 256 ? 256 : 512;
    p.np = type == RS_TYPE_F32 ? 2 : 1;
    p.oc = std::min(p.kp, 256);
    p.z = p.kp / p.oc;
    p.n_pad = round_up(n, kTileX);
    p.v_pad = round_up(v, kTileX);
    auto split = [](int64_t tx, int64_t ty, int32_t* splits, int32_t* tiles) {
        const int64_t want = std::max<int64_t>(1, ceil_div(512, tx));        // two workgroups per CU
        int64_t per = std::max<int64_t>(ceil_div(ty, want), std::min<int64_t>(ty, 2));
        *tiles = static_cast<int32_t>(per);
        *splits = static_cast<int32_t>(ceil_div(ty, per));
    };
    split(p.n_pad / kTileX, p.v_pad / kTileY, &p.splits_f, &p.tiles_f);
    split(p.v_pad / kTileX, p.n_pad / kTileY, &p.splits_w, &p.tiles_w);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at += round_up(bytes, 256);
        return o;
    };
    p.o_max = take(3 * kMaxBlocks * 4);
    p.o_scal = take(sizeof(Scal));
    p.o_h = take(p.n_pad * p.kp * 2 * p.np);
    p.o_w = take(p.v_pad * p.kp * 2 * p.np);
    p.o_bias = take(p.v_pad * 4);
    p.o_m = take(p.splits_f * p.n_pad * 4);
    p.o_s = take(p.splits_f * p.n_pad * 4);
    if (grad) {
        p.o_lse2 = take(p.n_pad * 4);
        p.o_wv = take(p.n_pad * 4);
        p.o_tgt = take(p.n_pad * 4);
        const int64_t of = p.splits_f * p.n_pad * p.kp * 4, ow = p.splits_w > 1 ? p.splits_w * p.v_pad * p.kp * 4 : 0;
        p.o_part = take(std::max(of, ow));  // O partials, read before dW's are written
        p.o_db = take(p.splits_w > 1 ? p.splits_w * p.v_pad * 4 : 0);
    }
    p.bytes = at;
    return p;
}

struct CeArgs {
    const void *H, *W;
    int64_t ldh, ldw;
    const float *bias, *weight;
    const int32_t* target;
    float *loss, *lse, *dbias;
    void *dH, *dW;
    int64_t lddh, lddw;
    char* ws;
    CePlan p;
    template <typename T>
    __host__ __device__ T* at(int64_t off) const {
        return reinterpret_cast<T*>(ws + off);
    }
};

__device__ __forceinline__ bool row_known(const CeArgs& a, int64_t n) {
    return n < a.p.n && static_cast<uint64_t>(static_cast<int64_t>(a.target[n])) < static_cast<uint64_t>(a.p.v);
}
__device__ __forceinline__ bool item_there(const CeArgs& a, int64_t v) {
    return v < a.p.v && !(a.bias && a.bias[v] == -INFINITY);
}

// ---- largest finite magnitudes of H, W and the weights (blockIdx.y = 0, 1, 2), one value per block ----------------
template <typename E>
__global__ __launch_bounds__(256) void ce_max_kernel(CeArgs a) {
    const int which = blockIdx.y;
    uint32_t m = 0;
    auto see = [&](float x) {
        const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
        if (b < 0x7F800000u && b > m) m = b;
    };
    if (which < 2) {
        const E* X = static_cast<const E*>(which ? a.W : a.H);
        const int64_t rows = which ? a.p.v : a.p.n, ld = which ? a.ldw : a.ldh;
        // a wave per row
        for (int64_t r = blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += gridDim.x * 4) {
            if (!(which ? item_there(a, r) : row_known(a, r))) continue;
            for (int c = threadIdx.x & 63; c < a.p.k; c += 64) see(static_cast<float>(X[r * ld + c]));
        }
    } else if (a.weight) {
        for (int64_t r = blockIdx.x * 256 + threadIdx.x; r < a.p.n; r += gridDim.x * 256)
            if (row_known(a, r)) see(a.weight[r]);
    }
    m = wave_max_u32(m);
    __shared__ uint32_t sm[4];
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0)
        a.at<uint32_t>(a.p.o_max)[which * kMaxBlocks + blockIdx.x] = max(max(sm[0], sm[1]), max(sm[2], sm[3]));
}

// 2^e with max * 2^e in [2^13, 2^14), e bounded so that the power and its inverse are normal numbers
__device__ __forceinline__ float scale_for(uint32_t max_bits) {
    if (max_bits == 0) return 1.f;
    int e = static_cast<int>(max_bits >> 23) - 127;
    e = 13 - e;
    e = min(max(e, -100), 100);
    return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// ---- packing -------------------------------------------------------------------------------------------------------
template <typename E, int NP>
__global__ __launch_bounds__(256) void ce_pack_kernel(CeArgs a, int max_blocks) {
    __shared__ uint32_t sm[3];
    if (threadIdx.x < 192) {
        const int which = threadIdx.x >> 6;
        uint32_t m = 0;
        for (int i = threadIdx.x & 63; i < max_blocks; i += 64) m = max(m, a.at<uint32_t>(a.p.o_max)[which * kMaxBlocks + i]);
        m = wave_max_u32(m);
        if ((threadIdx.x & 63) == 0) sm[which] = m;
    }
    __syncthreads();
    constexpr bool kScaled = !std::is_same<E, _Float16>::value;
    const float hs = kScaled ? scale_for(sm[0]) : 1.f, wsc = kScaled ? scale_for(sm[1]) : 1.f;
    // coefficients c = weight (p - [target]): |c| <= |weight| cs < 2^14
    const float cs = scale_for(a.weight ? sm[2] : 0x3F800000u);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        Scal s;
        s.hs = hs, s.wsc = wsc, s.cs = cs;
        s.logit = kLog2e / hs / wsc;
        s.inv_w = 1.f / wsc;
        s.inv_dw = 1.f / cs / hs;
        s.inv_cs = 1.f / cs;
        *a.at<Scal>(a.p.o_scal) = s;
    }
    const int64_t per_row = a.p.kp / 8, chunks = (a.p.n_pad + a.p.v_pad) * per_row;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < chunks; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = i / per_row;
        const int c0 = static_cast<int>(i % per_row) * 8;
        const bool w = row >= a.p.n_pad;
        const int64_t r = w ? row - a.p.n_pad : row;
        const bool there = w ? item_there(a, r) : row_known(a, r);
        if (w && c0 == 0) {
            const float b = r < a.p.v ? (a.bias ? a.bias[r] : 0.f) : -INFINITY;
            a.at<float>(a.p.o_bias)[r] = b * kLog2e;
        }
        const E* src = static_cast<const E*>(w ? a.W : a.H) + (there ? r * (w ? a.ldw : a.ldh) : 0);
        const float sc = w ? wsc : hs;
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = there && c0 + e < a.p.k ? static_cast<float>(src[c0 + e]) : 0.f;
            const float y = x * sc;  // (a power of two: exact)
            hi[e] = static_cast<_Float16>(y);
            if (NP == 2) lo[e] = static_cast<_Float16>(y - static_cast<float>(hi[e]));
        }
        _Float16* dst = a.at<_Float16>(w ? a.p.o_w : a.p.o_h) + r * a.p.kp + c0;
        *reinterpret_cast<f16x8*>(dst) = hi;
        if (NP == 2) *reinterpret_cast<f16x8*>(dst + (w ? a.p.v_pad : a.p.n_pad) * a.p.kp) = lo;
    }
}

// ---- the products --------------------------------------------------------------------------------------------------
__device__ __forceinline__ f32x16 mfma16(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// 16-byte chunk c of row r of an LDS tile sits at chunk c ^ (r mod 16) of the row (fewer where a row has fewer
// chunks): the row-wise and the transposing reads both spread over the banks.
template <int KP>
__device__ __forceinline__ int lds_chunk(int row, int c) {
    constexpr int C = KP / 8, M = C < 16 ? C - 1 : 15;
    return row * C + (c ^ (row & M));
}

// MODE kLoss / kLossGrad: x = users' rows, y = items; kItems: x = items, y = users' rows.
template <typename E, int NP, int KP, int MODE>
__global__ __launch_bounds__(256) void ce_main_kernel(CeArgs a) {
#pragma clang fp contract(fast)
    constexpr int OC = KP < 256 ? KP : 256, NB = OC / 32, KS = KP / 16, C = KP / 8;
    constexpr int PIECE = kTileY * KP;                     // elements of one piece of a tile
    constexpr int CHUNKS = kTileY * C * NP, PER = (CHUNKS + 255) / 256;
    constexpr int NM = MODE == kItems ? 3 : 1;             // values per streamed row
    extern __shared__ __attribute__((aligned(16))) char smem[];
    _Float16* tile = reinterpret_cast<_Float16*>(smem);          // [2][NP][kTileY][KP]
    float* meta = reinterpret_cast<float*>(smem + 2 * NP * PIECE * 2);       // [2][NM][kTileY]

    const CePlan& p = a.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lx = lane & 31, half = lane >> 5;
    const bool items = MODE == kItems;
    const int64_t x_pad = items ? p.v_pad : p.n_pad, y_pad = items ? p.n_pad : p.v_pad;
    const _Float16* X = a.at<_Float16>(items ? p.o_w : p.o_h);
    const _Float16* Y = a.at<_Float16>(items ? p.o_h : p.o_w);
    const int per = items ? p.tiles_w : p.tiles_f;
    const int split = blockIdx.y, oc0 = blockIdx.z * OC;
    const int64_t x = static_cast<int64_t>(blockIdx.x) * kTileX + wave * 32 + lx;
    const int t0 = split * per, t1 = static_cast<int>(min<int64_t>(y_pad / kTileY, t0 + per));
    const Scal sc = *a.at<Scal>(p.o_scal);

    f16x8 xf[NP][KS];
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int s = 0; s < KS; ++s)
            xf[q][s] = *reinterpret_cast<const f16x8*>(X + (q * x_pad + x) * KP + s * 16 + half * 8);

    f16x8 stage[PER];
    float stage_meta = 0.f;
    auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int ch = i * 256 + threadIdx.x;
            if (CHUNKS % 256 == 0 || ch < CHUNKS) {
                const int q = ch / (kTileY * C), r = ch / C % kTileY, c = ch % C;
                stage[i] = *reinterpret_cast<const f16x8*>(Y + (q * y_pad + static_cast<int64_t>(t) * kTileY + r) * KP + c * 8);
            }
        }
        if (threadIdx.x < NM * kTileY) {
            const int64_t y = static_cast<int64_t>(t) * kTileY + (threadIdx.x & 31);
            const int which = threadIdx.x >> 5;
            stage_meta = a.at<float>(!items ? p.o_bias : which == 0 ? p.o_lse2 : which == 1 ? p.o_wv : p.o_tgt)[y];
        }
    };
    auto put = [&](int b) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int ch = i * 256 + threadIdx.x;
            if (CHUNKS % 256 == 0 || ch < CHUNKS) {
                const int q = ch / (kTileY * C), r = ch / C % kTileY, c = ch % C;
                *reinterpret_cast<f16x8*>(tile + (b * NP + q) * PIECE + lds_chunk<KP>(r, c) * 8) = stage[i];
            }
        }
        if (threadIdx.x < NM * kTileY) meta[b * NM * kTileY + threadIdx.x] = stage_meta;
    };

    f32x16 acc[MODE == kLoss ? 1 : NB];
#pragma unroll
    for (int b = 0; b < (MODE == kLoss ? 1 : NB); ++b) acc[b] = f32x16{0};
    float m_run = -INFINITY, sum = 0.f;
    float bias_x = 0.f;
    if (items) bias_x = a.at<float>(p.o_bias)[x];

    fetch(t0);
    put(0);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int b = (t - t0) & 1;
        if (t + 1 < t1) fetch(t + 1);
        const _Float16* tl = tile + b * NP * PIECE;
        const float* mt = meta + b * NM * kTileY;

        f32x16 s = f32x16{0};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const f16x8 y0 = *reinterpret_cast<const f16x8*>(tl + lds_chunk<KP>(lx, ks * 2 + half) * 8);
            s = mfma16(y0, xf[0][ks], s);
            if constexpr (NP == 2) {
                const f16x8 y1 = *reinterpret_cast<const f16x8*>(tl + PIECE + lds_chunk<KP>(lx, ks * 2 + half) * 8);
                s = mfma16(y0, xf[1][ks], s);
                s = mfma16(y1, xf[0][ks], s);
            }
        }
        // lane: column x; register i: row y = 8 (i / 4) + 4 half + i mod 4 of the tile
        if constexpr (MODE != kItems) {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 bv = *reinterpret_cast<const f32x4*>(mt + 8 * j + 4 * half);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // a withdrawn item's row is zeros: 0 + (-inf)
                    s[4 * j + e] = s[4 * j + e] * sc.logit + bv[e];
                    top = fmaxf(top, s[4 * j + e]);
                }
            }
            top = fmaxf(top, __shfl_xor(top, 32));
            if (__any(top > m_run)) {  // rare after the first tiles: the maximum of a column grows about log(items) times
                const float m_new = fmaxf(m_run, top);
                const float f = m_new == -INFINITY ? 1.f : exp2f(m_run - m_new);
                m_run = m_new;
                sum *= f;
                if constexpr (MODE == kLossGrad) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[nb][i] *= f;
                }
            }
            const float off = m_run == -INFINITY ? 0.f : m_run - kShift;
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = exp2f(s[i] - off);
                part += s[i];
            }
            sum += part;
        } else {
            float part = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 ls = *reinterpret_cast<const f32x4*>(mt + 8 * j + 4 * half);
                const f32x4 wv = *reinterpret_cast<const f32x4*>(mt + kTileY + 8 * j + 4 * half);
                const i32x4 tg = __builtin_bit_cast(i32x4, *reinterpret_cast<const f32x4*>(mt + 2 * kTileY + 8 * j + 4 * half));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // a row that takes no part has lse2 = +inf and weight 0
                    const float pr = exp2f(s[4 * j + e] * sc.logit + bias_x - ls[e]);
                    s[4 * j + e] = wv[e] * (pr - (tg[e] == static_cast<int32_t>(x) ? 1.f : 0.f));
                    part += s[4 * j + e];
                }
            }
            sum += part;
        }
        if constexpr (MODE != kLoss) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f16x8 c0, c1;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float f = s[8 * j + e];
                    // the fp32 value itself is what both pieces come from: fused into the rounding of one of them, the
                    // product before it would round to another hi now and then
                    if (NP == 2) asm("" : "+v"(f));
                    c0[e] = static_cast<_Float16>(f);
                    if (NP == 2) c1[e] = static_cast<_Float16>(f - static_cast<float>(c0[e]));
                }
                // Y^T: lane = column of Y, elements e = rows 16 j + 8 (e / 4) + 4 half + e mod 4, as c0's.  A transposing
                // read hands lane i of a group of 16 the column i of the 4 x 16 block whose rows its lanes address.
                const int g = lane & 15, row = 16 * j + 4 * half + (g >> 2), col = oc0 + 16 * ((lane >> 4) & 1) + 4 * (g & 3);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    f16x8 yt[NP];
#pragma unroll
                    for (int q = 0; q < NP; ++q) {
                        const int cc = col + nb * 32;
                        auto rd = [&](int r) {
                            return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
                                tl + q * PIECE + lds_chunk<KP>(r, cc >> 3) * 8 + (cc & 7)));
                        };
                        const s16x4 u = rd(row), w = rd(row + 8);
                        yt[q] = __builtin_bit_cast(f16x8, __builtin_shufflevector(u, w, 0, 1, 2, 3, 4, 5, 6, 7));
                    }
                    acc[nb] = mfma16(yt[0], c0, acc[nb]);
                    if constexpr (NP == 2) {
                        acc[nb] = mfma16(yt[0], c1, acc[nb]);
                        acc[nb] = mfma16(yt[1], c0, acc[nb]);
                    }
                }
            }
        }
        if (t + 1 < t1) put(b ^ 1);
        __syncthreads();
    }

    sum += __shfl_xor(sum, 32);
    if constexpr (MODE != kItems) {
        if (blockIdx.z == 0 && half == 0) {
            a.at<float>(p.o_m)[split * p.n_pad + x] = m_run;
            a.at<float>(p.o_s)[split * p.n_pad + x] = sum;
        }
        if constexpr (MODE == kLossGrad) {
            float* O = a.at<float>(p.o_part) + (split * p.n_pad + x) * KP + oc0;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f32x4 o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = acc[nb][4 * j + e];
                    *reinterpret_cast<f32x4*>(O + nb * 32 + 8 * j + 4 * half) = o;
                }
        }
    } else if (p.splits_w > 1) {
        if (blockIdx.z == 0 && half == 0) a.at<float>(p.o_db)[split * p.v_pad + x] = sum;
        float* O = a.at<float>(p.o_part) + (split * p.v_pad + x) * KP + oc0;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = acc[nb][4 * j + e];
                *reinterpret_cast<f32x4*>(O + nb * 32 + 8 * j + 4 * half) = o;
            }
    } else if (x < p.v) {
        if (blockIdx.z == 0 && half == 0) a.dbias[x] = sum * sc.inv_cs;
        E* O = static_cast<E*>(a.dW) + x * a.lddw;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int col = oc0 + nb * 32 + 8 * (i / 4) + 4 * half + i % 4;
                if (col < p.k) O[col] = static_cast<E>(acc[nb][i] * sc.inv_dw);
            }
    }
}

// ---- joining the splits of the catalogue: lse, loss, dH and what the dW pass reads of each row; a wave per row -----
template <typename E>
__global__ __launch_bounds__(256) void ce_join_kernel(CeArgs a) {
    const CePlan& p = a.p;
    const int lane = threadIdx.x & 63;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int64_t rows = p.grad ? p.n_pad : p.n;
    if (n >= rows) return;
    const Scal sc = *a.at<Scal>(p.o_scal);
    const bool known = row_known(a, n);
    float m = -INFINITY, s = 0.f;
    if (known)
        for (int i = lane; i < p.splits_f; i += 64) m = fmaxf(m, a.at<float>(p.o_m)[i * p.n_pad + n]);
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (known)
        for (int i = lane; i < p.splits_f; i += 64) {
            const float mi = a.at<float>(p.o_m)[i * p.n_pad + n], si = a.at<float>(p.o_s)[i * p.n_pad + n];
            s += m == -INFINITY ? si : si * exp2f(mi - m);
        }
    s = wave_sum_f32(s);
    const int32_t tg = known ? a.target[n] : 0;
    const bool there = known && item_there(a, tg);
    float lt = 0.f;
    if (there)
        for (int c = lane; c < p.k; c += 64)
            lt = fmaf(static_cast<float>(static_cast<const E*>(a.H)[n * a.ldh + c]),
                      static_cast<float>(static_cast<const E*>(a.W)[tg * a.ldw + c]), lt);
    lt = wave_sum_f32(lt);
    if (there && a.bias) lt += a.bias[tg];
    // every item withdrawn: m stays -inf and s is 0
    const bool empty = m == -INFINITY && s == 0.f;
    const float l2 = m + (log2f(s) - kShift);
    const float lse = empty ? -INFINITY : m * kLn2 + logf(s) - kShift * kLn2;
    if (lane == 0 && n < p.n) {
        a.lse[n] = known ? lse : 0.f;
        a.loss[n] = !known || empty ? 0.f : there ? lse - lt : INFINITY;
    }
    if (!p.grad) return;
    const bool live = there && !empty;
    const float w = live ? (a.weight ? a.weight[n] : 1.f) : 0.f;
    if (lane == 0) {
        a.at<float>(p.o_lse2)[n] = live ? l2 : INFINITY;
        a.at<float>(p.o_wv)[n] = w * sc.cs;
        a.at<int32_t>(p.o_tgt)[n] = live ? tg : -1;
    }
    if (n >= p.n) return;
    E* out = static_cast<E*>(a.dH) + n * a.lddh;
    const float inv = sc.inv_w / s;
    for (int c = lane; c < p.k; c += 64) {
        float g = 0.f;
        if (live) {
            float o = 0.f;
            for (int i = 0; i < p.splits_f; ++i)
                o += a.at<float>(p.o_part)[(i * p.n_pad + n) * p.kp + c] * exp2f(a.at<float>(p.o_m)[i * p.n_pad + n] - m);
            g = w * (o * inv - static_cast<float>(static_cast<const E*>(a.W)[tg * a.ldw + c]));
        }
        out[c] = static_cast<E>(g);
    }
}

// dW and dbias from the splits of the users' rows, in their order
template <typename E>
__global__ __launch_bounds__(256) void ce_items_join_kernel(CeArgs a) {
    const CePlan& p = a.p;
    const Scal sc = *a.at<Scal>(p.o_scal);
    const int64_t total = p.v * p.k;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t v = i / p.k;
        const int c = static_cast<int>(i % p.k);
        float o = 0.f;
        for (int s = 0; s < p.splits_w; ++s) o += a.at<float>(p.o_part)[(s * p.v_pad + v) * p.kp + c];
        static_cast<E*>(a.dW)[v * a.lddw + c] = static_cast<E>(o * sc.inv_dw);
        if (c == 0) {
            float d = 0.f;
            for (int s = 0; s < p.splits_w; ++s) d += a.at<float>(p.o_db)[s * p.v_pad + v];
            a.dbias[v] = d * sc.inv_cs;
        }
    }
}

template <typename E, int NP, int KP, int MODE>
void launch_main(const CeArgs& a, hipStream_t st) {
    const CePlan& p = a.p;
    constexpr int NM = MODE == kItems ? 3 : 1;
    constexpr int lds = 2 * NP * kTileY * KP * 2 + 2 * NM * kTileY * 4;
    auto kern = ce_main_kernel<E, NP, KP, MODE>;
    if (lds > 64 * 1024)
        RS_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    const dim3 grid(static_cast<uint32_t>((MODE == kItems ? p.v_pad : p.n_pad) / kTileX),
                    static_cast<uint32_t>(MODE == kItems ? p.splits_w : p.splits_f), MODE == kLoss ? 1u : static_cast<uint32_t>(p.z));
    kern<<<grid, 256, lds, st>>>(a);
    RS_HIP(hipGetLastError());
}

template <typename E, int NP>
void launch_all(const CeArgs& a, hipStream_t st) {
    const CePlan& p = a.p;
    int blocks = 0;
    if (!std::is_same<E, _Float16>::value || (p.grad && a.weight)) {
        blocks = static_cast<int>(std::min<int64_t>(kMaxBlocks, ceil_div(std::max(p.n, p.v), 4)));
        ce_max_kernel<E><<<dim3(static_cast<uint32_t>(blocks), 3), 256, 0, st>>>(a);
        RS_HIP(hipGetLastError());
    }
    const int64_t chunks = (p.n_pad + p.v_pad) * (p.kp / 8);
    ce_pack_kernel<E, NP><<<static_cast<uint32_t>(std::min<int64_t>(ceil_div(chunks, 256), 4096)), 256, 0, st>>>(a, blocks);
    RS_HIP(hipGetLastError());
    auto mode = [&](auto m) {
        constexpr int M = decltype(m)::value;
        switch (p.kp) {
            case 32: return launch_main<E, NP, 32, M>(a, st);
            case 64: return launch_main<E, NP, 64, M>(a, st);
            case 128: return launch_main<E, NP, 128, M>(a, st);
            case 256: return launch_main<E, NP, 256, M>(a, st);
            default: return launch_main<E, NP, 512, M>(a, st);
        }
    };
    if (p.grad)
        mode(std::integral_constant<int, kLossGrad>{});
    else
        mode(std::integral_constant<int, kLoss>{});
    ce_join_kernel<E><<<static_cast<uint32_t>(ceil_div(p.grad ? p.n_pad : p.n, 4)), 256, 0, st>>>(a);
    RS_HIP(hipGetLastError());
    if (!p.grad) return;
    mode(std::integral_constant<int, kItems>{});
    if (p.splits_w > 1) {
        ce_items_join_kernel<E><<<static_cast<uint32_t>(std::min<int64_t>(ceil_div(p.v * p.k, 256), 8192)), 256, 0, st>>>(a);
        RS_HIP(hipGetLastError());
    }
}

// the sizes both entry points take; an empty string or the complaint
std::string check_sizes(int32_t type, int64_t n, int64_t v, int32_t k) {
    if (!type_ok(type)) return "type must be RS_TYPE_F32, RS_TYPE_BF16 or RS_TYPE_F16";
    if (n < 0 || n > INT32_MAX - 1024) return "n_rows out of range";
    if (v < 0 || v > INT32_MAX - 1024) return "n_items out of range";
    if (k < 1) return "n_factors must be at least 1";
    return std::string();
}

}  // namespace
}  // namespace rs

extern "C" int rs_softmax_ce_workspace(rs_ctx* ctx, int32_t type, int64_t n_rows, int64_t n_items, int32_t n_factors,
                                       int32_t with_grad, int64_t* bytes) {
    if (!bytes) return rs::set_error(ctx, RS_ERR_INVALID, "bytes is NULL");
    *bytes = 0;
    const std::string bad = rs::check_sizes(type, n_rows, n_items, n_factors);
    if (!bad.empty()) return rs::set_error(ctx, RS_ERR_INVALID, bad);
    if (n_factors > RS_DENSE_MAX_FACTORS) return rs::set_error(ctx, RS_ERR_UNSUPPORTED, "n_factors must be at most 512");
    if (n_rows && n_items) *bytes = rs::make_plan(type, n_rows, n_items, n_factors, with_grad).bytes;
    return RS_OK;
}

extern "C" int rs_softmax_ce(rs_ctx* ctx, int32_t type, int64_t n_rows, int64_t n_items, int32_t n_factors, const void* H,
                             int64_t ldh, const void* W, int64_t ldw, const float* bias, const int32_t* target,
                             const float* weight, float* loss, float* lse, void* dH, int64_t lddh, void* dW, int64_t lddw,
                             float* dbias, void* ws, int64_t ws_bytes, void* stream) {
    using namespace rs;
    std::string bad = check_sizes(type, n_rows, n_items, n_factors);
    if (!bad.empty()) return set_error(ctx, RS_ERR_INVALID, bad);
    if (n_factors > RS_DENSE_MAX_FACTORS) return set_error(ctx, RS_ERR_UNSUPPORTED, "n_factors must be at most 512");
    const int grads = (dH != nullptr) + (dW != nullptr) + (dbias != nullptr);
    if (grads != 0 && grads != 3 && n_rows && n_items)
        return set_error(ctx, RS_ERR_INVALID, "dH, dW and dbias are given together or not at all");
    if (n_rows == 0 && n_items == 0) return RS_OK;
    if (n_rows == 0 || n_items == 0)
        return set_error(ctx, RS_ERR_INVALID, n_rows ? "n_items is 0" : "n_rows is 0");
    const int64_t e = type_size(type);
    for (const std::string& b : {check_matrix("H", H, n_factors, ldh, e), check_matrix("W", W, n_factors, ldw, e),
                                 check_matrix("target", target, 1, 1, 4), check_matrix("loss", loss, 1, 1, 4),
                                 check_matrix("lse", lse, 1, 1, 4),
                                 grads ? check_matrix("dH", dH, n_factors, lddh, e) : std::string(),
                                 grads ? check_matrix("dW", dW, n_factors, lddw, e) : std::string(),
                                 grads ? check_matrix("dbias", dbias, 1, 1, 4) : std::string(),
                                 bias ? check_matrix("bias", bias, 1, 1, 4) : std::string(),
                                 weight ? check_matrix("weight", weight, 1, 1, 4) : std::string()})
        if (!b.empty()) return set_error(ctx, RS_ERR_INVALID, b);
    CeArgs a{};
    a.p = make_plan(type, n_rows, n_items, n_factors, grads == 3);
    if (!ws || reinterpret_cast<uintptr_t>(ws) % 16) return set_error(ctx, RS_ERR_INVALID, "ws is NULL or not 16-byte aligned");
    if (ws_bytes < a.p.bytes)
        return set_error(ctx, RS_ERR_INVALID, "ws holds " + std::to_string(ws_bytes) + " bytes, " + std::to_string(a.p.bytes) + " needed");
    a.H = H, a.W = W, a.ldh = ldh, a.ldw = ldw, a.bias = bias, a.target = target, a.weight = weight;
    a.loss = loss, a.lse = lse, a.dH = dH, a.dW = dW, a.lddh = lddh, a.lddw = lddw, a.dbias = dbias;
    a.ws = static_cast<char*>(ws);
    return dense_guard(ctx, [&]() -> int {
        const hipStream_t st = pick_stream(ctx, stream);
        if (type == RS_TYPE_F32)
            launch_all<float, 2>(a, st);
        else if (type == RS_TYPE_BF16)
            launch_all<__bf16, 1>(a, st);
        else
            launch_all<_Float16, 1>(a, st);
        return RS_OK;
    });
}
