// softmax_ce.hip -- softmax cross entropy over the item catalogue and its gradient, no logits kept (gfx950).
//
// Mathematics.  With x the "stationary" rows held by a wave and y the rows that stream past:
//   forward: x = users' rows, y = items but the row's target.  S[y, x] = W_y . H_x; a running maximum m_x and sum s_x of
//     2^(l2 - m_x), l2 the logit in base 2, and (for the gradient) O_x = sum_y 2^(l2 - m_x) W_y, all three rescaled when
//     m_x grows.  The target joins at the end: with its own term t = 2^(l2_target - m_x), one pass over the catalogue
//     gives lse and dH = weight (O - s W_target) / (s + t).  (With the target inside the sums dH would be the difference
//     O / (s + t) - W_target of two near vectors where its probability is near one: 2^-12 of W_target, against 2^-12 of
//     dH; the loss keeps its small values in the same way.)
//   dW: x = items, y = users' rows.  S is computed again, c = weight (2^(l2 - m_y) / (s_y + t_y) - [target]) and
//     dW_x += sum_y c H_y.
// Both are one kernel: S = Y X^T, then acc[k, x] += Y^T f(S).  S comes out of the matrix unit with x over lanes and y
// over registers, which is (up to an order of y, the same for both operands) what the second product takes as its
// second operand: f(S) never leaves the registers.  Its first operand Y^T comes from the same LDS tile as Y by
// transposing LDS reads.
//
// Operands are packed into the workspace first: rows padded to tiles and columns to KP with zeros, withdrawn items
// and rows without a known target zeroed (so NaN or garbage in them reaches no product), as fp16 of the matrix scaled by
// a power of two.  bf16's 8 bits fit fp16's 11: the products are those of bf16, but the coefficients f(S) keep 11 bits
// where bf16 MFMAs would round them to 8 (dW's error then was 1.5 times that of its own rounding).  fp16's gradients keep
// 11 bits themselves, so its coefficients are two pieces (405 us on 8192 x 26744 x 128; one piece takes 306 and leaves up
// to 2 times the error of dW's own rounding where it sums a few rows).  fp32 is split into two pieces hi + lo (each
// rounds its rest: at most 2^-23 of the element is left); the product of two such is hi hi + hi lo + lo hi, three fp16
// MFMAs (2.5 PF / 3) where an fp32 MFMA would run at 157 TF.  lo lo, at most 2^-22 of the product, of either sign and
// about 2^-24.6 in the mean square, is left out.
//
// With gradients, bound by the instruction mix of the two passes: 16 MFMAs of 32 cycles beside about 40 cycles of exponential,
// sums, maxima and packing for each of a lane's 16 logits (KP = 128: the matrix units are busy 41 and 39 % of the time, the
// vector ones 51 and 56 %).  1024 x 1e6 x 256 bf16 2.4 ms: passes 1.03 and 1.20 ms (1.02 and 0.87 PFLOP/s), largest
// elements and packing 0.38; 8192 x 26744 x 128 bf16 0.317 ms; 4096 x 3706 x 100 fp32 92 us; 128 x 1682 x 20 fp32 29 us,
// five launches.
#include <hip/hip_runtime.h>

#include <cmath>

#include "dense.hpp"

namespace rs {
namespace {

constexpr int kPad = 256;        // rows are padded to this: a multiple of what a workgroup holds or a stage streams
constexpr int kTileY = 128;      // streamed rows are split over workgroups in multiples of this
// rows that the table is read for as it is, without gradients: 4 / 5 rows (as it is / packed) against 108944 x 320 bf16 52 /
// 122 us, 1e6 x 256 bf16 216 / 460, 26744 x 100 fp32 16 / 30.  One launch holds four (a lane's registers); packed, 5 to 64
// rows take the same time
constexpr int kFewRows = 4;
constexpr int kFewItems = 128;   // items that a workgroup has on their way then: 8 waves x 4 x 4
constexpr int kMaxBlocks = 1024;  // blocks of the maxima pass at most, per matrix
// p = 2^(l2 - m) is held as 2^shift_of(m) p (fp16's range below 1 is short; beside a large m the shift would be lost in
// the difference), and m may lag the maximum by kLag: moving it at each new maximum costs a pass over the sums in most
// tiles (32 columns a wave, each with its own records)
constexpr float kLag = 8.f;
// a column's coefficients in the items' pass, weight p / s, are held times a power of two that brings the largest so far
// to [2^kCoefAt, 2^15]: whatever the item's probabilities and the weights, none is rounded by more than its 11 bits (two
// pieces: 22) or 2^-25, 2^-33 of the largest (one scale for the batch left nothing of an item that no row thinks likely).
// Brought to 2^11: the items' pass of 1024 x 1e6 x 256 bf16 1.34 ms, 1.20 with 2^8, where the scale moves less often.
constexpr int kCoefAt = 8;
__device__ __forceinline__ float shift_of(float m) { return fabsf(m) < 32768.f ? 7.f : 0.f; }
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

enum Mode { kLoss = 0, kLossGrad = 1, kItems = 2 };

// Shape of a workgroup: waves of 32 stationary rows each, streamed rows of a stage (between two barriers) in blocks of
// 32, waves per SIMD asked of the compiler.  Measured on 8192 x 26744 x 128 and 1024 x 1e6 x 256 (bf16), 4096 x 3706 x 100
// (fp32), times of the two passes (users / items):
//   KP = 128, one piece: 8 waves 149 / 186 us, 4 waves 171 / 196 and twice the pieces to join; stages of 4 blocks for the
//     users' pass (of 2: 150 when they were chosen, 137 now that the target stays out of the sums), 2 for the items' (4 spill)
//   KP = 256, one piece: 8 waves 1028 / 1200 us, 4 waves 1349 / 1323 (8 waves read the streamed tile once for 256 rows)
//   KP = 128, two pieces: 4 waves 35.9 / 36.5 us, 8 waves 34.1 / 34.7 (before the items' maxima)
//   wider: the row and its sums take more than half the registers: one wave per SIMD
struct Shape {
    int waves, blocks, occ;
};
constexpr Shape shape_for(int np, int kp, int mode) {
    if (np * kp >= 512) return {4, 1, 1};
    if (np * kp == 256) return np == 1 ? Shape{8, 1, 2} : Shape{4, 1, 2};
    if (np * kp == 128) return np == 2 ? Shape{4, 2, 2} : mode == kItems ? Shape{8, 2, 2} : Shape{8, 4, 2};
    return {4, 2, 2};
}

// Device scalars (ws): the powers of two that scale H and W.  They and their inverses may be no fp32 numbers (a largest
// element of 2^-140, or of 2^127 in both): only exponents are kept, and undone by ldexp.
struct Scal {
    int eh, ew;   // H, W are multiplied by 2^eh, 2^ew
    float logit;  // S -> base-2 logit: log2(e) 2^-(eh + ew)
};

struct CePlan {
    int64_t n, v, n_pad, v_pad;
    int32_t k, kp, np, oc, z, type, grad;
    int32_t few;  // ce_few_kernel: no packed tables
    int32_t splits_f, tiles_f, splits_w, tiles_w;  // splits of the streamed rows and their tiles each
    int64_t o_max, o_scal, o_h, o_w, o_bias, o_m, o_s, o_row, o_part, o_db, bytes;
};

CePlan make_plan(int32_t type, int64_t n, int64_t v, int32_t k, int32_t grad) {
    CePlan p{};
    p.n = n, p.v = v, p.k = k, p.type = type, p.grad = grad;
    p.kp = k <= 32 ? 32 : k <= 64 ? 64 : k <= 128 ? 128 : k <= 256 ? 256 : 512;
    p.np = type == RS_TYPE_F32 ? 2 : 1;
    p.oc = std::min(p.kp, 256);
    p.z = p.kp / p.oc;
    p.n_pad = round_up(n, kPad);
    p.v_pad = round_up(v, kPad);
    // Splits of the streamed rows: enough to fill the chip, against the sums that every split writes and the join reads.
    // In microseconds, by the measured rates of the passes: a tile of kTileY rows at 3.4 TFLOP/s a CU where one
    // workgroup has it (whole rounds of 256 workgroups), 2.4 where two share it (they end at different times: half a
    // workgroup's time is lost at the end), 3 for a workgroup's start and end, the sums at 8 TB/s.
    auto split = [&](int64_t rows_x, int64_t rows_y, int mode, int32_t* splits, int32_t* tiles) {
        const Shape sh = shape_for(p.np, p.kp, mode);
        const int64_t tx = ceil_div(rows_x, 32 * sh.waves) * p.z, ty = ceil_div(rows_y, kTileY);
        const bool alone = sh.waves == 8 || sh.occ == 1;
        const double tile = static_cast<double>(kTileY) * 32 * sh.waves * (p.kp + p.oc) * 2 * (p.np == 2 ? 3.0 : type == RS_TYPE_F16 ? 1.5 : 1.0) / (alone ? 3.4e6 : 2.4e6);
        const double sums = static_cast<double>(rows_x) * p.kp * 8 / 8e6;
        double best = 0.0;
        for (int64_t s = 1, per = ty; s == 1 || tx * s <= 4096; s = ceil_div(ty, per)) {  // each length of a split once
            const double one = static_cast<double>(per) * tile;
            double cost = alone ? static_cast<double>(ceil_div(tx * s, 256)) * (one + 3.0)
                                : static_cast<double>(std::max<int64_t>(tx * s, 256)) / 256 * (one + 2.0) + 0.5 * one;
            if (s > 1 || mode != kItems) cost += static_cast<double>(s) * sums;
            if (s > 1 && mode == kItems) cost += 5.0;  // the join's launch
            if (mode != kItems) cost += 0.05 * static_cast<double>(s);  // a row's pieces are read one after the other
            if (s == 1 || cost < best) best = cost, *splits = static_cast<int32_t>(s), *tiles = static_cast<int32_t>(per);
            if (per == 1) break;
            per = ceil_div(ty, ceil_div(ty, per - 1));
        }
    };
    split(n, v, kLossGrad, &p.splits_f, &p.tiles_f);
    split(v, n, kItems, &p.splits_w, &p.tiles_w);
    p.few = !grad && n <= kFewRows;
    if (p.few) p.splits_f = static_cast<int32_t>(std::min<int64_t>(512, ceil_div(v, kFewItems)));
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at += round_up(bytes, 256);
        return o;
    };
    p.o_max = take(2 * kMaxBlocks * 4);
    p.o_scal = take(sizeof(Scal));
    p.o_h = take(p.few ? 0 : p.n_pad * p.kp * 2 * p.np);
    p.o_w = take(p.few ? 0 : p.v_pad * p.kp * 2 * p.np);
    p.o_bias = take(p.few ? 0 : p.v_pad * 4);
    p.o_m = take(p.splits_f * p.n_pad * 4);
    p.o_s = take(p.splits_f * p.n_pad * 4);
    if (grad) {
        p.o_row = take(4 * p.n_pad * 4);
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
__device__ __forceinline__ float bounded_bias(float b) {
    return fabsf(b) < INFINITY ? fminf(fmaxf(b, -0x1p120f), 0x1p120f) : b;
}
__device__ __forceinline__ bool item_there(const CeArgs& a, int64_t v) {
    return v < a.p.v && !(a.bias && a.bias[v] == -INFINITY);
}

// Eight elements of a row from column c on as fp32, zeros past column k.  VEC: rows start at 16-byte addresses.
template <typename E, bool VEC>
__device__ __forceinline__ void load8(const E* row, int c, int k, float (&v)[8]) {
    constexpr int V = 16 / sizeof(E);
    typedef __attribute__((ext_vector_type(V))) E vec;
    if (VEC && c + 8 <= k) {
#pragma unroll
        for (int h = 0; h < 8 / V; ++h) {
            const vec w = *reinterpret_cast<const vec*>(row + c + h * V);
#pragma unroll
            for (int e = 0; e < V; ++e) v[h * V + e] = static_cast<float>(w[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < k ? static_cast<float>(row[c + e]) : 0.f;
    }
}

// e with max * 2^e in [2^13, 2^14): -114 to 162
__device__ __forceinline__ int scale_for(uint32_t max_bits) {
    return max_bits ? 14 - __builtin_amdgcn_frexp_expf(__uint_as_float(max_bits)) : 0;
}

// Past 2^126 the logits leave fp32 with their factor (S is a multiple of 2^-48: 2^78 at least, or 0); below 2^-126 they
// vanish beside any bias (S is below 2^37), but the factor stays above 0: a target left out is -inf times it.
__device__ __forceinline__ Scal scales(int eh, int ew) { return {eh, ew, __builtin_amdgcn_ldexpf(kLog2e, max(min(-(eh + ew), 126), -126))}; }

// frexp's exponent of the power of two that takes x to [2^kCoefAt, 2^(kCoefAt + 1))
__device__ __forceinline__ int coef_exponent(float x) { return min(kCoefAt + 2 - __builtin_amdgcn_frexp_expf(x), 127); }

__device__ __forceinline__ void see_largest(uint32_t& m, float x) {
    const uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
    if (b < 0x7F800000u && b > m) m = b;
}

// ---- largest finite magnitudes of H and W (blockIdx.y = 0, 1), one value per block ---------------------------------
template <typename E, bool VEC>
__global__ __launch_bounds__(256) void ce_max_kernel(CeArgs a) {
    const CePlan& p = a.p;
    const int which = blockIdx.y;
    uint32_t m = 0;
    const E* X = static_cast<const E*>(which ? a.W : a.H);
    const int64_t rows = which ? p.v : p.n, ld = which ? a.ldw : a.ldh;
    const int lanes = p.kp / 8, at = threadIdx.x / lanes, c = threadIdx.x % lanes * 8;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (256 / lanes);
#pragma unroll 4
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * (256 / lanes) + at; r < rows; r += step) {
        if (c >= p.k) continue;
        float v[8];
        load8<E, VEC>(X + r * ld, c, p.k, v);
        uint32_t t = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) see_largest(t, v[e]);
        if (t > m && (which ? item_there(a, r) : row_known(a, r))) m = t;  // (looked up for new records only)
    }
    m = wave_max_u32(m);
    __shared__ uint32_t sm[4];
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) a.at<uint32_t>(p.o_max)[which * kMaxBlocks + blockIdx.x] = max(max(sm[0], sm[1]), max(sm[2], sm[3]));
}

// ---- packing: a thread per eight columns ---------------------------------------------------------------------------
template <typename E, int NP, bool VEC>
__global__ __launch_bounds__(256) void ce_pack_kernel(CeArgs a, int max_blocks) {
    constexpr bool kScaled = !std::is_same<E, _Float16>::value;
    const CePlan& p = a.p;
    __shared__ uint32_t sm[2];
    if (kScaled && threadIdx.x < 128) {
        const int which = threadIdx.x >> 6;
        uint32_t m = 0;
        for (int i = threadIdx.x & 63; i < max_blocks; i += 64) m = max(m, a.at<uint32_t>(p.o_max)[which * kMaxBlocks + i]);
        m = wave_max_u32(m);
        if ((threadIdx.x & 63) == 0) sm[which] = m;
    }
    __syncthreads();
    const int eh = kScaled ? scale_for(sm[0]) : 0, ew = kScaled ? scale_for(sm[1]) : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.at<Scal>(p.o_scal) = scales(eh, ew);
    const int lanes = p.kp / 8, at = threadIdx.x / lanes, c0 = threadIdx.x % lanes * 8, step = 256 / lanes;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * step + at; row < p.n_pad + p.v_pad; row += static_cast<int64_t>(gridDim.x) * step) {
        const bool w = row >= p.n_pad;
        const int64_t r = w ? row - p.n_pad : row;
        const bool there = w ? item_there(a, r) : row_known(a, r);
        if (w && c0 == 0) {
            // base-2 biases.  Finite ones are held to +-2^120: the type's lowest value is no withdrawal.
            const float b = r < p.v ? (a.bias ? a.bias[r] : 0.f) : -INFINITY;
            a.at<float>(p.o_bias)[r] = bounded_bias(b) * kLog2e;
        }
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (there) load8<E, VEC>(static_cast<const E*>(w ? a.W : a.H) + r * (w ? a.ldw : a.ldh), c0, p.k, v);
        const int sc = w ? ew : eh;
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float y = __builtin_amdgcn_ldexpf(v[e], sc);
            hi[e] = static_cast<_Float16>(y);
            if (NP == 2) lo[e] = static_cast<_Float16>(y - static_cast<float>(hi[e]));
        }
        _Float16* dst = a.at<_Float16>(w ? p.o_w : p.o_h) + r * p.kp + c0;
        *reinterpret_cast<f16x8*>(dst) = hi;
        if (NP == 2) *reinterpret_cast<f16x8*>(dst + (w ? p.v_pad : p.n_pad) * p.kp) = lo;
    }
}

// ---- the products --------------------------------------------------------------------------------------------------
__device__ __forceinline__ f32x16 mfma16(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Each wave holds 32 stationary rows; a stage of streamed rows passes through LDS, the next one on its way in registers.
// MODE kLoss / kLossGrad: x = users' rows, y = items; kItems: x = items, y = users' rows.
template <typename E, int NP, int KP, int MODE, int WAVES, int SUB, int OCC>
__global__ __launch_bounds__(WAVES * 64, OCC) void ce_main_kernel(CeArgs a) {
#pragma clang fp contract(fast)
    constexpr bool items = MODE == kItems;
    constexpr int THREADS = WAVES * 64;
    constexpr int OC = KP < 256 ? KP : 256, NB = MODE == kLoss ? 1 : OC / 32, KS = KP / 16, C = KP / 8;
    constexpr int NC = std::is_same<E, __bf16>::value ? 1 : 2;  // pieces of a coefficient
    constexpr int ROWS = 32 * SUB;                         // rows of a stage
    constexpr int PIECE = ROWS * KP;                       // elements of one piece of a stage
    constexpr int CHUNKS = ROWS * C * NP, PER = (CHUNKS + THREADS - 1) / THREADS;
    constexpr int NM = items ? 4 : 1;                      // values per streamed row: bias, or m, weight / s, target, its coefficient
    extern __shared__ __attribute__((aligned(16))) char smem[];
    // smem: [2][NP][ROWS][KP] fp16
    float* meta = reinterpret_cast<float*>(smem + 2 * NP * PIECE * 2);  // [2][NM][ROWS]

    const CePlan& p = a.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lx = lane & 31, half = lane >> 5;
    const int64_t x_pad = items ? p.v_pad : p.n_pad, y_pad = items ? p.n_pad : p.v_pad;
    const _Float16* X = a.at<_Float16>(items ? p.o_w : p.o_h);
    const _Float16* Y = a.at<_Float16>(items ? p.o_h : p.o_w);
    const int per = (items ? p.tiles_w : p.tiles_f) * (kTileY / ROWS);
    const int split = blockIdx.y, oc0 = blockIdx.z * OC;
    const int64_t x0 = (static_cast<int64_t>(blockIdx.x) * WAVES + wave) * 32, x = x0 + lx;  // the wave's first row, the lane's
    const int t0 = split * per, t1 = static_cast<int>(min<int64_t>(((items ? p.n : p.v) + ROWS - 1) / ROWS, t0 + per));
    const Scal sc = *a.at<Scal>(p.o_scal);

    f16x8 xf[NP][KS];
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int s = 0; s < KS; ++s) xf[q][s] = *reinterpret_cast<const f16x8*>(X + (q * x_pad + x) * KP + s * 16 + half * 8);

    // A stage is contiguous in memory, piece by piece: chunk i THREADS + thread of it is this thread's i-th.
    static_assert(CHUNKS % THREADS == 0 && (ROWS * C) % THREADS == 0, "a thread's i-th chunk is in one piece for all threads");
    f16x8 stage[PER];
    float stage_meta = 0.f;
    auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            constexpr int per_piece = ROWS * C / THREADS;
            const char* src = reinterpret_cast<const char*>(Y + (i / per_piece * y_pad + static_cast<int64_t>(t) * ROWS) * KP) + i % per_piece * (THREADS * 16);
            stage[i] = *reinterpret_cast<const f16x8*>(src + threadIdx.x * 16u);
        }
        if (threadIdx.x < NM * ROWS) {
            const int64_t y = static_cast<int64_t>(t) * ROWS + threadIdx.x % ROWS;
            const int which = threadIdx.x / ROWS;
            stage_meta = a.at<float>(!items ? p.o_bias : p.o_row + which * p.n_pad * 4)[y];
        }
    };
    constexpr int LINES_T = THREADS / C;  // rows that the threads' chunks cover
    const int put_base = LdsTile<KP>::base(threadIdx.x / C, threadIdx.x % C);
    auto put = [&](int b) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            // rows a multiple of 16 further have the same chunk order
            const int r = i * LINES_T, at = LINES_T % 16 == 0 ? put_base + r * KP * 2 : LdsTile<KP>::base(r + threadIdx.x / C, threadIdx.x % C);
            *reinterpret_cast<f16x8*>(smem + b * NP * PIECE * 2 + at) = stage[i];
        }
        if (threadIdx.x < NM * ROWS) meta[b * NM * ROWS + threadIdx.x] = stage_meta;
    };

    f32x16 acc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = f32x16{0};
    float m_run = -INFINITY, sum = 0.f;
    float coef = 0x1p126f;  // items: what a column's coefficients are held times
    const float bias_x = items ? a.at<float>(p.o_bias)[x] : 0.f;
    const int target_x = !items && x < p.n ? a.target[x] : -1;

    // row-wise reads: row lx, chunk half + 2 ks.  Transposing reads hand lane i of a group of 16 the column i of the
    // 4 x 16 block whose rows its lanes address: row 4 half + (i / 4) of 8, chunk 2 (group mod 2) + (i mod 4) / 2.
    const int g4 = lane & 15, row_base = LdsTile<KP>::base(lx, half);
    const int tr_row = 4 * half + (g4 >> 2), tr_chunk = oc0 / 8 + 2 * ((lane >> 4) & 1) + ((g4 & 3) >> 1);
    const int tr_base[2] = {LdsTile<KP>::base(tr_row, tr_chunk) + (g4 & 1) * 8, LdsTile<KP>::base(tr_row + 8, tr_chunk) + (g4 & 1) * 8};

    // The sums times f.  Where a wave has a SIMD for itself they stay in accumulator registers, which only matrix instructions
    // work on, and are taken out one at a time: left to the compiler, all of them move to other registers for this rare step,
    // and those to scratch (2048 x 26744 x 512 fp32 1.50 ms against 3.36, 512 bf16 0.62 against 0.68).  The waits stand for the
    // compiler's, which does not look inside.
    auto rescale = [&](float f) {
        if constexpr (OCC == 1) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                asm volatile("s_nop 15\n\ts_nop 15" : "+a"(acc[nb]));  // (from a product to the read of its result: 19 at most)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float t;
                    asm volatile("v_accvgpr_read_b32 %1, %0\n\ts_nop 1\n\tv_mul_f32 %1, %1, %2\n\ts_nop 1\n\tv_accvgpr_write_b32 %0, %1"
                                 : "+a"(acc[nb][i]), "=&v"(t)
                                 : "v"(f));
                }
                asm volatile("s_nop 15" : "+a"(acc[nb]));
            }
        } else {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[nb][i] *= f;
        }
    };

    // 32 streamed rows from first_y on: the byte offset of their LDS tile and their values
    auto block = [&](int first_y, int tile, const float* mt) {
        // the tile's offset has none of the bits that the chunks are mixed in: it joins the bases.  Wide rows take the
        // addresses anew for every block, or the compiler keeps all of them in registers and spills others (KP = 256: 168
        // bytes, 1221 / 2067 us against 1072 / 1215); narrow ones keep them (KP = 128: 126 us against 154)
        int rb = row_base + tile, tb[2] = {tr_base[0] + tile, tr_base[1] + tile};
        if (KP >= 256) {
            asm volatile("" : "+v"(rb), "+v"(tb[0]));
            tb[1] = tb[0] ^ 128;  // (the chunks' order eight rows on; the rows themselves are a constant)
        }
        constexpr int kEight = KP >= 256 ? 8 * KP * 2 : 0;
        f32x16 s = f32x16{0};
        // A lane's target is not for these sums: its logit becomes -inf.  Asked for between the products where the registers
        // allow it (8192 x 26744 x 128 without gradients: 100 us, 108 in the maximum's branch, 99 if it were left in),
        // otherwise in the maximum's branch (1024 x 1e6 x 256 with gradients: 2440 us; 2472 between the products and the
        // maximum, 2513 early, 2418 if it were left in)
        constexpr bool kEarly = !items && NP * KP < 256;
        const bool target_here = !items && __any(static_cast<uint32_t>(target_x - first_y) < 32u);
        auto leave_out = [&] {
            if (!target_here) return;
            const int tg = target_x - first_y - 4 * half;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = tg == 8 * (i / 4) + i % 4 ? -INFINITY : s[i];
        };
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const f16x8 y0 = *reinterpret_cast<const f16x8*>(smem + LdsTile<KP>::at(rb, ks * 2));
            s = mfma16(y0, xf[0][ks], s);
            if constexpr (NP == 2) {
                const f16x8 y1 = *reinterpret_cast<const f16x8*>(smem + PIECE * 2 + LdsTile<KP>::at(rb, ks * 2));
                s = mfma16(y0, xf[1][ks], s);
                s = mfma16(y1, xf[0][ks], s);
            }
            if constexpr (kEarly)
                if (ks == 0) leave_out();
        }
        // lane: column x; register i: row y = 8 (i / 4) + 4 half + i mod 4 of the block
        float off = 0.f;
        bool here = false;
        if constexpr (!items) {
            float top = -INFINITY;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 bv = *reinterpret_cast<const f32x4*>(mt + 8 * q + 4 * half);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // a withdrawn item's row is zeros: 0 + (-inf)
                    s[4 * q + e] = s[4 * q + e] * sc.logit + bv[e];
                    top = fmaxf(top, s[4 * q + e]);
                }
            }
            top = fmaxf(top, __shfl_xor(top, 32));
            const bool over = __any(top > m_run + kLag);  // the first block, and rarely after it
            if (over || (!kEarly && target_here)) {
                if constexpr (!kEarly) leave_out();
                if (over) {
                    if constexpr (!kEarly) {
                        top = s[0];
#pragma unroll
                        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
                        top = fmaxf(top, __shfl_xor(top, 32));
                    }
                    const float m_new = top > m_run + kLag ? top : m_run;
                    const float f = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_run - m_new) + (shift_of(m_new) - shift_of(m_run)));
                    m_run = m_new;
                    sum *= f;
                    if constexpr (MODE == kLossGrad) rescale(f);
                }
            }
            off = m_run == -INFINITY ? 0.f : m_run - shift_of(m_run);
        } else {
            // which of the rows have their target among the wave's columns (few: one in items / 32)
            here = __any(static_cast<uint32_t>(__float_as_int(mt[2 * ROWS + lx]) - static_cast<int>(x0)) < 32u);
        }
        // f(S) and its product.  Wide rows leave few registers: 16 rows of the block at a time (KP = 256: the items'
        // pass 2001 -> 1536 us); otherwise all 32, which gives the scheduler more to run beside the products (KP = 128:
        // 145 us against 166)
        constexpr int HALVES = NP * KP >= 256 ? 2 : 1, Q = 4 / HALVES;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            if constexpr (items) {
#pragma unroll
                for (int q = Q * h; q < Q * h + Q; ++q) {
                    const f32x4 m = *reinterpret_cast<const f32x4*>(mt + 8 * q + 4 * half);
#pragma unroll
                    for (int e = 0; e < 4; ++e)  // a row that takes no part has m = +inf and weight 0
                        s[4 * q + e] = __builtin_amdgcn_exp2f((s[4 * q + e] * sc.logit + bias_x) - m[e]);  // (rounded as the users' pass rounds it)
                }
#pragma unroll
                for (int q = Q * h; q < Q * h + Q; ++q) {
                    const f32x4 ws = *reinterpret_cast<const f32x4*>(mt + ROWS + 8 * q + 4 * half);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[4 * q + e] *= ws[e];
                }
                if (here) {
#pragma unroll
                    for (int q = Q * h; q < Q * h + Q; ++q) {
                        const i32x4 t = *reinterpret_cast<const i32x4*>(mt + 2 * ROWS + 8 * q + 4 * half);
                        const f32x4 w = *reinterpret_cast<const f32x4*>(mt + 3 * ROWS + 8 * q + 4 * half);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[4 * q + e] = t[e] == static_cast<int>(x) ? w[e] : s[4 * q + e];
                    }
                }
                float top = 0.f;
#pragma unroll
                for (int i = 4 * Q * h; i < 4 * Q * (h + 1); ++i) top = fmaxf(top, fabsf(s[i]));
                if (__any(top * coef > 0x1p15f)) {  // the first block, and rarely after it
                    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                    top = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
                    const int down = top * coef > 0x1p15f ? coef_exponent(top) - __builtin_amdgcn_frexp_expf(coef) : 0;
                    coef = __builtin_amdgcn_ldexpf(coef, down);
                    rescale(__builtin_amdgcn_ldexpf(1.f, down));
                }
            } else {
#pragma unroll
                for (int i = 4 * Q * h; i < 4 * Q * (h + 1); ++i) s[i] = __builtin_amdgcn_exp2f(s[i] - off);
            }
            float part = 0.f;
#pragma unroll
            for (int i = 4 * Q * h; i < 4 * Q * (h + 1); ++i) part += s[i];
            sum += part;
            if constexpr (MODE != kLoss) {
#pragma unroll
                for (int j = 2 * h / HALVES; j < 2 * (h + 1) / HALVES; ++j) {
                    f16x8 c[NC];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float f = s[8 * j + e];
                        // the fp32 value itself is what both pieces come from: fused into the rounding of one of them, the
                        // product before it would round to another hi now and then (a power of two may be: it is exact)
                        if (NC == 2) asm("" : "+v"(f));
                        if (items) f *= coef;
                        c[0][e] = static_cast<_Float16>(f);
                        if (NC == 2) c[NC - 1][e] = static_cast<_Float16>(f - static_cast<float>(c[0][e]));
                    }
                    // Y^T: lane = column of Y, elements e = rows 16 j + 8 (e / 4) + 4 half + e mod 4, as c's
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        f16x8 yt[NP];
#pragma unroll
                        for (int q = 0; q < NP; ++q) {
                            auto rd = [&](int k) {
                                return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
                                    smem + q * PIECE * 2 + j * (32 * KP) + LdsTile<KP>::at(tb[k], nb * 4) + k * kEight));
                            };
                            const s16x4 u = rd(0), w = rd(1);
                            yt[q] = __builtin_bit_cast(f16x8, __builtin_shufflevector(u, w, 0, 1, 2, 3, 4, 5, 6, 7));
                        }
                        acc[nb] = mfma16(yt[0], c[0], acc[nb]);
                        if constexpr (NC == 2) acc[nb] = mfma16(yt[0], c[1], acc[nb]);
                        if constexpr (NP == 2) acc[nb] = mfma16(yt[1], c[0], acc[nb]);
                    }
                }
            }
        }
    };

    fetch(t0);
    put(0);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int b = (t - t0) & 1;
        if (t + 1 < t1) fetch(t + 1);
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) block(t * ROWS + sub * 32, b * NP * PIECE * 2 + sub * (64 * KP), meta + b * NM * ROWS + sub * 32);
        if (t + 1 < t1) put(b ^ 1);
        __syncthreads();
    }

    float total = sum + __shfl_xor(sum, 32);
    // a withdrawn item's coefficients are exp2(-inf), NaN beside a row that is not finite: it takes no part
    if (items && bias_x == -INFINITY) {
        total = 0.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) acc[nb] = f32x16{0};
    }
    const int back = 127 - static_cast<int>(__float_as_uint(coef) >> 23) - sc.eh;  // (items)
    // a split's sums, times 2^back: four columns of row x at a time
    auto partial = [&](int64_t rows, int back) {
        float* O = a.at<float>(p.o_part) + (split * rows + x) * KP + oc0;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f32x4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __builtin_amdgcn_ldexpf(acc[nb][4 * q + e], back);
                *reinterpret_cast<f32x4*>(O + nb * 32 + 8 * q + 4 * half) = o;
            }
    };
    if constexpr (!items) {
        if (blockIdx.z == 0 && half == 0) {
            a.at<float>(p.o_m)[split * p.n_pad + x] = m_run;
            a.at<float>(p.o_s)[split * p.n_pad + x] = total;
        }
        if constexpr (MODE == kLossGrad) partial(p.n_pad, 0);
    } else if (p.splits_w > 1) {
        if (blockIdx.z == 0 && half == 0) a.at<float>(p.o_db)[split * p.v_pad + x] = total;
        partial(p.v_pad, back);
    } else {
        if (x < p.v && blockIdx.z == 0 && half == 0) a.dbias[x] = total;
        // dW through LDS, so that a row's stores are contiguous: OW columns at a time, 16-byte chunk c of row r at
        // chunk c ^ (r mod the row's chunks)
        constexpr int OW = OC < 128 / static_cast<int>(sizeof(E)) ? OC : 128 / static_cast<int>(sizeof(E));
        constexpr int kRow = OW * static_cast<int>(sizeof(E)), CH = kRow / 16, V = 16 / sizeof(E), LINES = 64 / CH;
        typedef __attribute__((ext_vector_type(4))) E e4;
        typedef __attribute__((ext_vector_type(sizeof(E)))) int words;  // (stored as it is read: integers)
        typedef __attribute__((ext_vector_type(V))) E ev;
        char* mine = smem + wave * 32 * kRow;
        const bool aligned = (reinterpret_cast<uintptr_t>(a.dW) | static_cast<uintptr_t>(a.lddw * static_cast<int64_t>(sizeof(E)))) % 16 == 0;
#pragma unroll
        for (int w0 = 0; w0 < OC; w0 += OW) {
#pragma unroll
            for (int q = 0; q < OW / 8; ++q) {
                e4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = static_cast<E>(__builtin_amdgcn_ldexpf(acc[(w0 + 8 * q) / 32][4 * (q % 4) + e], back));
                const int byte = (8 * q + 4 * half) * static_cast<int>(sizeof(E));
                *reinterpret_cast<words*>(mine + lx * kRow + (((byte >> 4) ^ (lx & (CH - 1))) << 4) + (byte & 15)) = __builtin_bit_cast(words, v);
            }
            wave_lds_fence();
#pragma unroll
            for (int r = 0; r < 32; r += LINES) {
                const int row = r + lane / CH, ch = lane % CH, col = oc0 + w0 + ch * V;
                const i32x4 w = *reinterpret_cast<const i32x4*>(mine + row * kRow + ((ch ^ (row & (CH - 1))) << 4));
                if (x0 + row >= p.v) continue;
                E* o = static_cast<E*>(a.dW) + (x0 + row) * a.lddw + col;
                if (aligned && col + V <= p.k) {
                    *reinterpret_cast<i32x4*>(o) = w;
                } else {
                    const ev y = __builtin_bit_cast(ev, w);
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (col + e < p.k) o[e] = y[e];
                }
            }
            wave_lds_fence();
        }
    }
}

// ---- a few rows without gradients: the table is read once, as it is ------------------------------------------------
// Packing it for four rows would cost more than its products (2 x 108938 x 317 bf16, rows not aligned: 90 us in all, 173
// packed; aligned, 4 x 108944 x 320 43 us and the join's 9, one row 19 and 9: 3.7 TB/s).  The rows
// stay in registers in fp32; sixteen lanes take an item, eight columns each at a time, and sum its products by shuffles;
// lane l keeps the running maximum and sum of row l mod R (one row, or
// up to four).  KC: 128 columns each.
template <typename E, bool VEC, int KC, int R>
__global__ __launch_bounds__(512) void ce_few_kernel(CeArgs a) {
#pragma clang fp contract(fast)
    const CePlan& p = a.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, sub = lane >> 4, row = l & (R - 1);
    const E *H = static_cast<const E*>(a.H), *W = static_cast<const E*>(a.W);
    float h[R][KC][8];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < KC; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) h[r][j][e] = 0.f;
            if (r < p.n && l * 8 + j * 128 < p.k) load8<E, VEC>(H + r * a.ldh, l * 8 + j * 128, p.k, h[r][j]);
        }
    constexpr int U = KC == 4 ? 2 : 4;  // items of a lane on their way (four of 512 columns would not fit the registers)
    const int64_t target = row < p.n ? a.target[row] : -1;
    float m = -INFINITY, s = 0.f;
    for (int64_t v0 = static_cast<int64_t>(blockIdx.x) * kFewItems + wave * 16; v0 < p.v; v0 += static_cast<int64_t>(gridDim.x) * kFewItems) {
#pragma unroll 1
        for (int q = 0; q < 4; q += U) {
            float w[U][KC][8], b[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t v = min(v0 + (q + u) * 4 + sub, p.v - 1);
                b[u] = bounded_bias(a.bias ? a.bias[v] : 0.f) * kLog2e;
#pragma unroll
                for (int j = 0; j < KC; ++j) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[u][j][e] = 0.f;
                    if (l * 8 + j * 128 < p.k) load8<E, VEC>(W + v * a.ldw, l * 8 + j * 128, p.k, w[u][j]);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t v = v0 + (q + u) * 4 + sub;
                float dot[R];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    dot[r] = 0.f;
#pragma unroll
                    for (int j = 0; j < KC; ++j)
#pragma unroll
                        for (int e = 0; e < 8; ++e) dot[r] = fmaf(h[r][j][e], w[u][j][e], dot[r]);
#pragma unroll
                    for (int o = 8; o; o >>= 1) dot[r] += __shfl_xor(dot[r], o);
                }
                const float mine = R == 1 || row == 0 ? dot[0] : row == 1 ? dot[1 % R] : row == 2 ? dot[2 % R] : dot[3 % R];
                // a withdrawn item may hold anything; the row's target joins at the end
                const float l2 = v >= p.v || b[u] == -INFINITY || v == target ? -INFINITY : fmaf(mine, kLog2e, b[u]);
                const float top = fmaxf(m, l2);
                if (top > -INFINITY || l2 != l2) {
                    s = s * __builtin_amdgcn_exp2f(m - top) + __builtin_amdgcn_exp2f(l2 - top);
                    m = top;
                }
            }
        }
    }
    // the four items at a time, then the waves
    auto meet = [&](float m2, float s2) {
        const float top = fmaxf(m, m2);
        s = top == -INFINITY ? s + s2 : s * __builtin_amdgcn_exp2f(m - top) + s2 * __builtin_amdgcn_exp2f(m2 - top);
        m = top;
    };
    meet(__shfl_xor(m, 16), __shfl_xor(s, 16));
    meet(__shfl_xor(m, 32), __shfl_xor(s, 32));
    __shared__ float sm[2][8][R];
    if (lane < R) sm[0][wave][lane] = m, sm[1][wave][lane] = s;
    __syncthreads();
    if (threadIdx.x < R) {
        for (int w = 1; w < 8; ++w) meet(sm[0][w][lane], sm[1][w][lane]);
        const int64_t at = blockIdx.x * p.n_pad + lane;
        a.at<float>(p.o_m)[at] = m;
        a.at<float>(p.o_s)[at] = s * __builtin_amdgcn_exp2f(shift_of(m));  // (as the passes keep it)
    }
}

// ---- joining the splits of the catalogue: lse, loss, dH and what the dW pass reads of each row --------------------
// W waves per row: one, or where few rows have many splits the eight of a workgroup, which share the splits (27 x 635201
// x 92 fp32, 709 splits: all of a call 432 us, 534 with one; 1024 x 1e6 x 256 bf16, 64 splits: the join 18 us and 30).
template <typename E, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void ce_join_kernel(CeArgs a) {
    const CePlan& p = a.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n = W == 1 ? wide_block() * 4 + wave : wide_block();
    const int64_t rows = p.grad ? p.n_pad : p.n;
    if (n >= rows) return;
    const Scal sc = *a.at<Scal>(p.o_scal);
    const bool known = row_known(a, n);
    const float *pm = a.at<float>(p.o_m) + n, *ps = a.at<float>(p.o_s) + n;
    // (the first 64 splits' values and the target's are asked for together)
    const float m0 = lane < p.splits_f ? pm[lane * p.n_pad] : -INFINITY, s0 = lane < p.splits_f ? ps[lane * p.n_pad] : 0.f;
    const int32_t tg = known ? a.target[n] : 0;
    const bool there = known && item_there(a, tg);
    float m = known ? m0 : -INFINITY, s = 0.f;
    if (known)
        for (int i = lane + 64; i < p.splits_f; i += 64) m = fmaxf(m, pm[i * p.n_pad]);
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const E *h = static_cast<const E*>(a.H) + n * a.ldh, *wt = static_cast<const E*>(a.W) + tg * a.ldw;
    float lt = 0.f;
    if (there)
        for (int c = lane; c < p.k; c += 64) lt = fmaf(static_cast<float>(h[c]), static_cast<float>(wt[c]), lt);
    lt = wave_sum_f32(lt);
    // the target's logit in base 2, rounded as the passes round theirs; the maximum over all items
    const float lt2 = there ? fmaf(lt, kLog2e, bounded_bias(a.bias ? a.bias[tg] : 0.f) * kLog2e) : -INFINITY;
    const bool first = lt2 >= m;
    if (first) m = lt2;
    auto share = [&](float mi, float si) { return m == -INFINITY ? si : si * __builtin_amdgcn_exp2f((mi - m) - shift_of(mi)); };
    if (known) {
        if (lane < p.splits_f) s = share(m0, s0);
        for (int i = lane + 64; i < p.splits_f; i += 64) s += share(pm[i * p.n_pad], ps[i * p.n_pad]);
    }
    const float rest = wave_sum_f32(s);  // the others' sum
    // every item withdrawn: m stays -inf and the sum is 0
    const bool empty = m == -INFINITY && rest == 0.f;
    s = there ? rest + __builtin_amdgcn_exp2f(lt2 - m) : rest;
    // lse = m ln 2 + ls, in two parts: where m is large they must not be joined before the target's logit goes
    const float ls = first ? log1pf(rest) : log2f(s) * kLn2;
    if (lane == 0 && (W == 1 || wave == 0) && n < p.n) {
        a.lse[n] = !known ? 0.f : empty ? -INFINITY : fmaf(m, kLn2, ls);
        a.loss[n] = !known || empty ? 0.f : there ? fmaf(m - lt2, kLn2, ls) : INFINITY;
    }
    if (!p.grad) return;
    const bool live = there && !empty;
    const float w = live ? (a.weight ? a.weight[n] : 1.f) : 0.f;
    if (lane == 0 && (W == 1 || wave == 0)) {
        float* row = a.at<float>(p.o_row) + n;
        row[0] = live ? m : INFINITY;
        row[p.n_pad] = live ? w / s : 0.f;
        row[2 * p.n_pad] = __int_as_float(live ? tg : -1);
        row[3 * p.n_pad] = live ? -w * (rest / s) : 0.f;  // the target's coefficient, weight (p - 1)
    }
    if (n >= p.n) return;
    E* out = static_cast<E*>(a.dH) + n * a.lddh;
    // weight (O / s - W_target rest / s), in W's scale; the weight's exponent goes with the scale's at the end, so that no
    // step before the last leaves fp32
    const float inv = 1.f / s, share_rest = rest / s, w_frac = __builtin_amdgcn_frexp_mantf(w);
    const int back = __builtin_amdgcn_frexp_expf(w) - sc.ew;
    // four columns a lane; where a row has fewer than 256, groups of lanes share the splits
    const int quads = p.kp / 4, lanes = quads < 64 ? quads : 64, groups = 64 / lanes, grp = lane / lanes;
    const float* O = a.at<float>(p.o_part) + n * p.kp;
    const int64_t step = p.n_pad * p.kp;
    const int share_w = (p.splits_f + W - 1) / W, i_first = W == 1 ? 0 : wave * share_w, i_last = min(p.splits_f, i_first + share_w);
    for (int c = lane % lanes * 4; c < p.kp; c += 256) {
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        if (live)
            for (int i0 = i_first; i0 < i_last; i0 += 64) {
                // the factors of 64 splits, one a lane
                float f = 0.f;
                if (i0 + lane < i_last) {
                    const float mi = i0 ? pm[(i0 + lane) * p.n_pad] : m0;
                    f = __builtin_amdgcn_exp2f((mi - m) - shift_of(mi));
                }
                const int count = min(64, i_last - i0);
#pragma unroll 8
                for (int i = 0; i < count; i += groups) {  // (as often in every lane: a shuffle reads active lanes only)
                    const float fi = __shfl(f, i + grp);
                    if (i + grp >= count) continue;
                    const f32x4 x = *reinterpret_cast<const f32x4*>(O + (i0 + i + grp) * step + c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], fi, o[e]);
                }
            }
        for (int g = lanes; g < 64; g <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], g);
        if constexpr (W > 1) {
            __shared__ f32x4 sums[W - 1][64];
            if (wave) sums[wave - 1][lane] = o;
            __syncthreads();
            if (wave == 0)
#pragma unroll
                for (int w = 0; w < W - 1; ++w)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] += sums[w][lane][e];
            __syncthreads();
        }
        if (grp == 0 && (W == 1 || wave == 0))
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < p.k) {
                    const float t = __builtin_amdgcn_ldexpf(static_cast<float>(wt[c + e]), sc.ew);
                    out[c + e] = static_cast<E>(live ? __builtin_amdgcn_ldexpf(w_frac * (o[e] * inv - share_rest * t), back) : 0.f);
                }
    }
}

// dW and dbias from the splits of the users' rows, in their order; a thread per four columns
template <typename E>
__global__ __launch_bounds__(256) void ce_items_join_kernel(CeArgs a) {
    const CePlan& p = a.p;
    const int quads = p.kp / 4;  // (a power of two)
    const int64_t i = wide_block() * 256 + threadIdx.x, v = i >> __builtin_ctz(quads);
    const int c = (static_cast<int>(i) & (quads - 1)) * 4;
    if (v >= p.v || c >= p.k) return;
    const float* O = a.at<float>(p.o_part) + v * p.kp + c;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    // eight splits' loads at a time: a split is read where it was just written, far from this CU
    for (int s0 = 0; s0 < p.splits_w; s0 += 8) {
        f32x4 x[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) x[s] = s0 + s < p.splits_w ? *reinterpret_cast<const f32x4*>(O + (s0 + s) * p.v_pad * p.kp) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += x[s][e];
    }
    E* out = static_cast<E*>(a.dW) + v * a.lddw;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e < p.k) out[c + e] = static_cast<E>(o[e]);
    if (c == 0) {
        float d = 0.f;
        for (int s = 0; s < p.splits_w; ++s) d += a.at<float>(p.o_db)[s * p.v_pad + v];
        a.dbias[v] = d;
    }
}

template <typename E, int NP, int KP, int MODE>
void launch_main(const CeArgs& a, hipStream_t st) {
    const CePlan& p = a.p;
    constexpr Shape sh = shape_for(NP, KP, MODE);
    constexpr int NM = MODE == kItems ? 4 : 1, OC = KP < 256 ? KP : 256;
    constexpr int row = OC * static_cast<int>(sizeof(E)) < 128 ? OC * static_cast<int>(sizeof(E)) : 128;
    // two stages and their rows' values; dW leaves through the same memory
    constexpr int rows = 32 * sh.blocks, tiles = 2 * NP * rows * KP * 2 + 2 * NM * rows * 4, out = MODE == kItems ? sh.waves * 32 * row : 0;
    constexpr int lds = tiles > out ? tiles : out, kTileX = sh.waves * 32;
    static_assert(lds <= 160 * 1024 && kPad % kTileX == 0 && kTileY % rows == 0, "the shape fits the LDS and the padding");
    auto kern = ce_main_kernel<E, NP, KP, MODE, sh.waves, sh.blocks, sh.occ>;
    if (lds > 64 * 1024)
        RS_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    const dim3 grid(static_cast<uint32_t>(ceil_div(MODE == kItems ? p.v : p.n, kTileX)),
                    static_cast<uint32_t>(MODE == kItems ? p.splits_w : p.splits_f), MODE == kLoss ? 1u : static_cast<uint32_t>(p.z));
    kern<<<grid, sh.waves * 64, lds, st>>>(a);
    RS_HIP(hipGetLastError());
}

template <typename E, int NP>
void launch_all(const CeArgs& a, hipStream_t st) {
    const CePlan& p = a.p;
    const bool vec = (reinterpret_cast<uintptr_t>(a.H) | reinterpret_cast<uintptr_t>(a.W) |
                      static_cast<uintptr_t>((a.ldh | a.ldw) * static_cast<int64_t>(sizeof(E)))) % 16 == 0;
    auto prepare = [&](auto v) {
        constexpr bool VEC = decltype(v)::value;
        const int64_t step = 256 / (p.kp / 8);  // rows of a block at a time
        int blocks = 0;
        if (!std::is_same<E, _Float16>::value) {
            blocks = static_cast<int>(std::min<int64_t>(kMaxBlocks, ceil_div(std::max(p.n, p.v), step)));
            ce_max_kernel<E, VEC><<<dim3(static_cast<uint32_t>(blocks), 2), 256, 0, st>>>(a);
            RS_HIP(hipGetLastError());
        }
        ce_pack_kernel<E, NP, VEC><<<static_cast<uint32_t>(std::min<int64_t>(ceil_div(p.n_pad + p.v_pad, step), 8192)), 256, 0, st>>>(a, blocks);
        RS_HIP(hipGetLastError());
    };
    if (p.few) {
        auto few = [&](auto v, auto kc) {
            constexpr bool VEC = decltype(v)::value;
            constexpr int KC = decltype(kc)::value;
            if (p.n == 1)
                ce_few_kernel<E, VEC, KC, 1><<<static_cast<uint32_t>(p.splits_f), 512, 0, st>>>(a);
            else
                ce_few_kernel<E, VEC, KC, kFewRows><<<static_cast<uint32_t>(p.splits_f), 512, 0, st>>>(a);
            RS_HIP(hipGetLastError());
        };
        auto wide = [&](auto v) {
            if (p.k <= 128)
                few(v, std::integral_constant<int, 1>{});
            else if (p.k <= 256)
                few(v, std::integral_constant<int, 2>{});
            else
                few(v, std::integral_constant<int, 4>{});
        };
        vec ? wide(std::true_type{}) : wide(std::false_type{});
        ce_join_kernel<E, 1><<<wide_grid(ceil_div(p.n, 4)), 256, 0, st>>>(a);
        RS_HIP(hipGetLastError());
        return;
    }
    if (vec)
        prepare(std::true_type{});
    else
        prepare(std::false_type{});
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
    if (p.grad && p.splits_f >= 16 && p.n <= 2048)
        ce_join_kernel<E, 8><<<wide_grid(p.grad ? p.n_pad : p.n), 512, 0, st>>>(a);
    else
        ce_join_kernel<E, 1><<<wide_grid(ceil_div(p.grad ? p.n_pad : p.n, 4)), 256, 0, st>>>(a);
    RS_HIP(hipGetLastError());
    if (!p.grad) return;
    mode(std::integral_constant<int, kItems>{});
    if (p.splits_w > 1) {
        ce_items_join_kernel<E><<<wide_grid(ceil_div(p.v * (p.kp / 4), 256)), 256, 0, st>>>(a);
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
    return rs::no_throw([&]() -> int {
        if (!bytes) return rs::set_error(ctx, RS_ERR_INVALID, "bytes is NULL");
        *bytes = 0;
        const std::string bad = rs::check_sizes(type, n_rows, n_items, n_factors);
        if (!bad.empty()) return rs::set_error(ctx, RS_ERR_INVALID, bad);
        if (n_factors > RS_DENSE_MAX_FACTORS) return rs::set_error(ctx, RS_ERR_UNSUPPORTED, "n_factors must be at most 512");
        if (n_rows && n_items) *bytes = rs::make_plan(type, n_rows, n_items, n_factors, with_grad).bytes;
        return RS_OK;
    });
}

extern "C" int rs_softmax_ce(rs_ctx* ctx, int32_t type, int64_t n_rows, int64_t n_items, int32_t n_factors, const void* H,
                             int64_t ldh, const void* W, int64_t ldw, const float* bias, const int32_t* target,
                             const float* weight, float* loss, float* lse, void* dH, int64_t lddh, void* dW, int64_t lddw,
                             float* dbias, void* ws, int64_t ws_bytes, void* stream) {
    return rs::no_throw([&]() -> int {
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
    });
}
