// int8.hip -- rows quantised to 8 bits and the int8 matrix product with a scale per row and per channel (gfx950).
//
// C_mn = a_m b_n sum_k A_mk B_nk + ...: the sums run on the int8 matrix unit (exact in int32), the scales and biases in
// the epilogue.  Two kernels: for few rows of A one pass over B straight from HBM to registers (bound by B's bytes);
// for many rows LDS tiles (bound by the product, or for short rows by writing C).
#include <hip/hip_runtime.h>

#include "dense.hpp"

namespace rs {
namespace {

// ---- quantising rows -----------------------------------------------------------------------------------------------
// |x| / s to the nearest integer, ties to even, as if the quotient were exact: the fp32 quotient gives its floor r (or an
// integer beside it where the quotient is near one, far from the tie), the sign of the remainder |x| - (r + 1/2) s decides:
// one fused multiply-add keeps that sign, and zero, exact.
__device__ __forceinline__ int quantize(float ax, float s, float inv) {
    const float r = floorf(ax * inv);
    const int ri = static_cast<int>(r), d = static_cast<int>(__float_as_uint(fmaf(-(r + 0.5f), s, ax)));
    return ri + (d + (ri & 1) > 0);  // above the tie, or on it beside an odd r
}

// Lanes of a row: 16 up to 128 columns, 32 up to 256 (1e6 x 256 fp32 210 us, 6.1 TB/s; 412 with a wave a row), a wave, or
// past kWideRow columns the four of a workgroup (64 x 32768 bf16 12 us, 46 with a wave; but 8192 x 1024 13 us, 8 with a
// wave; 2048 columns give the same).  Bound by the bytes: 2048 x 4096 bf16 8 us with the launch.  Eight elements a lane
// at a time; rows of up to eight times that stay in registers between the maximum and the rounding, longer ones are read
// again.  VEC: rows of X start at 16-byte addresses, rows of q at 8-byte ones.
constexpr int kWideRow = 2048;
template <typename E, bool VEC, int LANES>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const E* __restrict__ X, int64_t ldx, int64_t rows, int64_t cols,
                                                           int8_t* __restrict__ q, int64_t ldq, float* __restrict__ scale) {
    typedef __attribute__((ext_vector_type(16 / sizeof(E)))) E vec;
    constexpr int V = 16 / sizeof(E), STEP = 8 * LANES, kKeep = LANES < 64 ? 1 : 8;
    const int at = threadIdx.x % LANES * 8;
    const int64_t r = wide_block() * (256 / LANES) + threadIdx.x / LANES;
    if (r >= rows) return;
    const E* x = X + r * ldx;
    int8_t* o = q + r * ldq;
    auto load = [&](int64_t c, float (&v)[8]) {
        if (VEC && c + 8 <= cols) {
#pragma unroll
            for (int h = 0; h < 8 / V; ++h) {
                const vec w = *reinterpret_cast<const vec*>(x + c + h * V);
#pragma unroll
                for (int e = 0; e < V; ++e) v[h * V + e] = static_cast<float>(w[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? static_cast<float>(x[c + e]) : 0.f;
        }
    };
    uint32_t m = 0;
    auto see = [&](const float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t b = __float_as_uint(v[e]) & 0x7FFFFFFFu;
            m = b > m ? b : m;
        }
    };
    float kept[kKeep][8];
    const bool fits = cols <= STEP * kKeep;
    if (fits) {
#pragma unroll
        for (int i = 0; i < kKeep; ++i)
            if (i * STEP < cols) load(i * STEP + at, kept[i]), see(kept[i]);
    } else {
        for (int64_t c = at; c < cols; c += STEP) {
            float v[8];
            load(c, v);
            see(v);
        }
    }
    if constexpr (LANES < 64) {
#pragma unroll
        for (int l = LANES / 2; l; l >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), l)));
    } else {
        m = wave_max_u32(m);
    }
    if constexpr (LANES == 256) {
        __shared__ uint32_t tops[4];
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
        __syncthreads();
        m = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    }
    const bool finite = m < 0x7F800000u;
    const float s = finite ? __uint_as_float(m) * (1.f / 127.f) : __uint_as_float(0x7FC00000u);
    if (at == 0) scale[r] = s;
    // a row of small numbers is scaled up (exactly) first, so that no remainder and no 1 / s leaves the normal numbers
    const float pre = s > 7.9e-31f ? 1.f : 0x1p96f, sp = s * pre, inv = 1.f / sp;
    const uint32_t some = finite && s > 0.f ? ~0u : 0u;
    auto write = [&](int64_t c, const float (&v)[8]) {
        if (c >= cols) return;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // (a subnormal scale may be rounded down by a third of itself: the quotient of the row's largest then passes 127)
            const int n = min(quantize(fabsf(v[e]) * pre, sp, inv), 127);
            w[e / 4] |= static_cast<uint32_t>((v[e] < 0.f ? -n : n) & 255) << (8 * (e % 4));
        }
        w[0] &= some, w[1] &= some;
        if (VEC && c + 8 <= cols) {
            *reinterpret_cast<uint2*>(o + c) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < cols) o[c + e] = static_cast<int8_t>(w[e / 4] >> (8 * (e % 4)));
        }
    };
    if (fits) {
#pragma unroll
        for (int i = 0; i < kKeep; ++i)
            if (i * STEP < cols) write(i * STEP + at, kept[i]);
    } else {
        for (int64_t c = at; c < cols; c += STEP) {
            float v[8];
            load(c, v);
            write(c, v);
        }
    }
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

// Few rows of A (m <= 64): they sit in LDS as MT tiles of 16; each wave takes 16 rows of B at a time straight from HBM
// into 16x16x64 MFMAs (first operand B's rows, second A's), so B is read once.  Bound by B's bytes: one row against 1e6 x 256
// 52 us, 4.9 TB/s.
constexpr int kFewRows = 64;
constexpr int kFewLds = 64 * 1024;
template <typename E, bool VEC, int MT>
__global__ __launch_bounds__(256) void i8_few_kernel(I8Args a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lk = lane >> 4;
    const int kc = static_cast<int>(ceil_div(a.k, 64));  // steps of 64
    i32x4* xs = reinterpret_cast<i32x4*>(smem);          // [kc][MT][64 lanes]
    for (int i = threadIdx.x; i < kc * MT * 64; i += 256) {
        const int64_t row = (i >> 6) % MT * 16 + (i & 15);
        xs[i] = row < a.m ? load16<VEC>(a.A + row * a.lda, static_cast<int64_t>((i >> 6) / MT) * 64 + ((i & 63) >> 4) * 16, a.k) : i32x4{0, 0, 0, 0};
    }
    __syncthreads();
    float sa[MT], rb[MT];
#pragma unroll
    for (int x = 0; x < MT; ++x) {
        const int64_t m = x * 16 + lr;
        sa[x] = m < a.m ? a.a_scale[m] : 0.f;
        rb[x] = m < a.m && a.row_bias ? a.row_bias[m] : 0.f;
    }
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + wave; t * 16 < a.n; t += static_cast<int64_t>(gridDim.x) * 4) {
        const int64_t n = t * 16 + lr;
        const int8_t* row = a.B + (n < a.n ? n : a.n - 1) * a.ldb;
        i32x4 acc[MT];
#pragma unroll
        for (int x = 0; x < MT; ++x) acc[x] = i32x4{0, 0, 0, 0};
        for (int s = 0; s < kc; ++s) {
            const i32x4 b = load16<VEC>(row, static_cast<int64_t>(s) * 64 + lk * 16, a.k);
#pragma unroll
            for (int x = 0; x < MT; ++x) acc[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, xs[(s * MT + x) * 64 + lane], acc[x], 0, 0, 0);
        }
        // lane: row m = 16 x + lr of A, registers: rows 4 lk + e of B
#pragma unroll
        for (int x = 0; x < MT; ++x)
            if (x * 16 + lr < a.m) {
                const int o[4] = {acc[x][0], acc[x][1], acc[x][2], acc[x][3]};
                store_scores<E>(a, x * 16 + lr, t * 16 + 4 * lk, o, sa[x], rb[x]);
            }
    }
}

// Many rows: TM x TN tiles of C, waves of WM x WN (32x32x32 MFMAs, first operand B's rows), steps of 64 along k through a
// double-buffered LDS tile; the next step's rows are on their way in registers during the MFMAs.  C leaves through
// LDS, so that a row's stores are contiguous.  OUT16: C's rows start at 16-byte addresses.
// 2048 x 8192 x 4096 to bf16 84 us, 1.64 POP/s (a large product reaches 2.0); 4096 x 26744 x 128 to bf16 75 us, bound by
// writing C at 2.9 TB/s (two steps on their way, or a workgroup that fetches its next tile while this one leaves, changed
// nothing; 128 x 128 tiles 90 us).
constexpr int kStep = 64;
template <typename E, bool VEC, bool OUT16, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__((TM / WM) * (TN / WN) * 64) void i8_tile_kernel(I8Args a, int tiles_m, int tiles_n) {
#pragma clang fp contract(fast)
    constexpr int THREADS = (TM / WM) * (TN / WN) * 64, CH = (TM + TN) * 4, PER = CH / THREADS, MB = WM / 32, NB = WN / 32;
    static_assert(CH % THREADS == 0, "chunks are dealt evenly");
    constexpr int kBuf = (TM + TN) * kStep;
    __shared__ __attribute__((aligned(16))) char smem[2 * kBuf];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 31, half = lane >> 5;
    const int wm = wave % (TM / WM) * WM, wn = wave / (TM / WM) * WN;
    // workgroups go round the eight XCDs: each XCD takes a contiguous part of the tiles (rows of A fastest), whose
    // operands its L2 then holds
    const int total = tiles_m * tiles_n, xcd = blockIdx.x & 7, nth = blockIdx.x >> 3;
    const int tile = xcd * (total >> 3) + min(xcd, total & 7) + nth;
    const int64_t m0 = static_cast<int64_t>(tile % tiles_m) * TM, n0 = static_cast<int64_t>(tile / tiles_m) * TN;
    const int steps = static_cast<int>(ceil_div(a.k, kStep));
    // 16-byte chunk c of row r sits at chunk c ^ ((r / 2) mod 4)
    auto at = [](int r, int c) { return (r * 4 + (c ^ ((r >> 1) & 3))) * 16; };
    i32x4 st[PER];
    const int8_t* src[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {  // rows past the end repeat the last one: their products are not stored
        const int ch = i * THREADS + threadIdx.x, r = ch >> 2;
        src[i] = r < TM ? a.A + min(m0 + r, a.m - 1) * a.lda : a.B + min(n0 + r - TM, a.n - 1) * a.ldb;
    }
    auto fetch = [&](int s) {
#pragma unroll
        for (int i = 0; i < PER; ++i) st[i] = load16<VEC>(src[i], static_cast<int64_t>(s) * kStep + (threadIdx.x & 3) * 16, a.k);
    };
    auto put = [&](int buf) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int ch = i * THREADS + threadIdx.x;
            *reinterpret_cast<i32x4*>(smem + buf * kBuf + at(ch >> 2, ch & 3)) = st[i];
        }
    };
    i32x16 acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = i32x16{0};
    fetch(0);
    put(0);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        if (s + 1 < steps) fetch(s + 1);
        const char* t = smem + (s & 1) * kBuf;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i32x4 fa[MB], fb[NB];
#pragma unroll
            for (int j = 0; j < MB; ++j) fa[j] = *reinterpret_cast<const i32x4*>(t + at(wm + 32 * j + lr, 2 * h + half));
#pragma unroll
            for (int i = 0; i < NB; ++i) fb[i] = *reinterpret_cast<const i32x4*>(t + at(TM + wn + 32 * i + lr, 2 * h + half));
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int j = 0; j < MB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[i], fa[j], acc[i][j], 0, 0, 0);
        }
        if (s + 1 < steps) put((s + 1) & 1);
        __syncthreads();
    }
    // 32 rows of C at a time through the wave's part of the tile: WN values a row, 16-byte chunk c of row r at
    // chunk c ^ (r mod the row's chunks)
    constexpr int kRow = WN * static_cast<int>(sizeof(E)), kRowCh = kRow / 16;
    static_assert((TM / WM) * (TN / WN) * 32 * kRow <= 2 * kBuf, "the waves' parts fit the tile");
    char* mine = smem + wave * 32 * kRow;
    auto out_at = [](int r, int byte) { return r * kRow + (((byte >> 4) ^ (r & (kRowCh - 1))) << 4) + (byte & 15); };
    float sb[NB][4][4], cb[NB][4][4];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t n = n0 + wn + 32 * i + 8 * g + 4 * half + e;
                sb[i][g][e] = n < a.n ? a.b_scale[n] : 0.f;
                cb[i][g][e] = n < a.n && a.col_bias ? a.col_bias[n] : 0.f;
            }
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        const int64_t mb = m0 + wm + 32 * j, m = mb + lr;
        const float sa = m < a.m ? a.a_scale[m] : 0.f, rb = m < a.m && a.row_bias ? a.row_bias[m] : 0.f;
        typedef __attribute__((ext_vector_type(4))) E e4;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                e4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = static_cast<E>(static_cast<float>(acc[i][j][4 * g + e]) * (sa * sb[i][g][e]) + rb + cb[i][g][e]);
                typedef __attribute__((ext_vector_type(sizeof(E)))) int words;  // (stored as it is read: integers)
                *reinterpret_cast<words*>(mine + out_at(lr, (32 * i + 8 * g + 4 * half) * static_cast<int>(sizeof(E)))) = __builtin_bit_cast(words, v);
            }
        wave_lds_fence();
        constexpr int V = 16 / sizeof(E), LANES = WN / V, ROWS = 64 / LANES;  // lanes along a row, rows at a time
#pragma unroll
        for (int r = 0; r < 32; r += ROWS) {
            const int row = r + lane / LANES, c = lane % LANES * V;
            const i32x4 w = *reinterpret_cast<const i32x4*>(mine + out_at(row, c * static_cast<int>(sizeof(E))));
            const int64_t n = n0 + wn + c;
            if (mb + row >= a.m) continue;
            E* o = static_cast<E*>(a.C) + (mb + row) * a.ldc + n;
            if (OUT16 && n + V <= a.n) {
                *reinterpret_cast<i32x4*>(o) = w;
            } else {
                typedef __attribute__((ext_vector_type(V))) E ev;
                const ev x = __builtin_bit_cast(ev, w);
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (n + e < a.n) o[e] = x[e];
            }
        }
        wave_lds_fence();
    }
}

template <typename E, bool VEC>
void launch_i8(const I8Args& a, hipStream_t st) {
    const int64_t kc = ceil_div(a.k, 64);
    const int mt = a.m <= 16 ? 1 : a.m <= 32 ? 2 : 4;
    if (a.m <= kFewRows && kc * mt * 1024 <= kFewLds) {
        const int lds = static_cast<int>(kc) * mt * 1024;
        const uint32_t blocks = static_cast<uint32_t>(std::min<int64_t>(ceil_div(a.n, 64), 2048));
        if (mt == 1)
            i8_few_kernel<E, VEC, 1><<<blocks, 256, lds, st>>>(a);
        else if (mt == 2)
            i8_few_kernel<E, VEC, 2><<<blocks, 256, lds, st>>>(a);
        else
            i8_few_kernel<E, VEC, 4><<<blocks, 256, lds, st>>>(a);
        RS_HIP(hipGetLastError());
        return;
    }
    const bool out16 = (reinterpret_cast<uintptr_t>(a.C) | static_cast<uintptr_t>(a.ldc * static_cast<int64_t>(sizeof(E)))) % 16 == 0;
    auto go = [&](auto tm, auto tn, auto wm, auto wn, auto o16) {
        constexpr int TM = decltype(tm)::value, TN = decltype(tn)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
        const int64_t tiles_m = ceil_div(a.m, TM), tiles_n = ceil_div(a.n, TN);
        i8_tile_kernel<E, VEC, decltype(o16)::value, TM, TN, WM, WN><<<static_cast<uint32_t>(tiles_m * tiles_n), (TM / WM) * (TN / WN) * 64, 0, st>>>(
            a, static_cast<int>(tiles_m), static_cast<int>(tiles_n));
    };
    using std::integral_constant;
    auto size = [&](auto o16) {
        // 256 x 256 tiles where they fill the chip: half the LDS reads per product
        if (ceil_div(a.m, 256) * ceil_div(a.n, 256) >= 192)
            go(integral_constant<int, 256>{}, integral_constant<int, 256>{}, integral_constant<int, 128>{}, integral_constant<int, 64>{}, o16);
        else
            go(integral_constant<int, 128>{}, integral_constant<int, 128>{}, integral_constant<int, 64>{}, integral_constant<int, 64>{}, o16);
    };
    if (out16)
        size(std::true_type{});
    else
        size(std::false_type{});
    RS_HIP(hipGetLastError());
}

}  // namespace
}  // namespace rs

extern "C" int rs_quantize_rows(rs_ctx* ctx, int32_t type, int64_t n_rows, int64_t n_cols, const void* X, int64_t ldx, int8_t* q,
                                int64_t ldq, float* scale, void* stream) {
    return rs::no_throw([&]() -> int {
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
                const bool vec = (reinterpret_cast<uintptr_t>(X) | static_cast<uintptr_t>(ldx * static_cast<int64_t>(sizeof(E)))) % 16 == 0 &&
                                 (reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(ldq)) % 8 == 0;
                auto go = [&](auto v, auto lanes) {
                    constexpr int LANES = decltype(lanes)::value;
                    quantize_rows_kernel<E, decltype(v)::value, LANES><<<wide_grid(ceil_div(n_rows, 256 / LANES)), 256, 0, st>>>(
                        static_cast<const E*>(X), ldx, n_rows, n_cols, q, ldq, scale);
                };
                auto width = [&](auto v) {
                    if (n_cols > kWideRow)
                        go(v, std::integral_constant<int, 256>{});
                    else if (n_cols > 256)
                        go(v, std::integral_constant<int, 64>{});
                    else if (n_cols > 128)
                        go(v, std::integral_constant<int, 32>{});
                    else
                        go(v, std::integral_constant<int, 16>{});
                };
                vec ? width(std::true_type{}) : width(std::false_type{});
            });
            RS_HIP(hipGetLastError());
            return RS_OK;
        });
    });
}

extern "C" int rs_i8_matmul(rs_ctx* ctx, int64_t m, int64_t n, int64_t k, const int8_t* A, int64_t lda, const float* a_scale,
                            const int8_t* B, int64_t ldb, const float* b_scale, const float* row_bias, const float* col_bias,
                            int32_t out_type, void* C, int64_t ldc, void* stream) {
    return rs::no_throw([&]() -> int {
        using namespace rs;
        if (!type_ok(out_type)) return set_error(ctx, RS_ERR_INVALID, "out_type must be RS_TYPE_F32, RS_TYPE_BF16 or RS_TYPE_F16");
        if (m < 0 || m > INT32_MAX) return set_error(ctx, RS_ERR_INVALID, "m out of range");
        if (n < 0 || n > INT32_MAX) return set_error(ctx, RS_ERR_INVALID, "n out of range");
        if (ceil_div(m, 128) * ceil_div(n, 128) > INT32_MAX / 512) return set_error(ctx, RS_ERR_UNSUPPORTED, "m x n is too large for one call");
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
    });
}
