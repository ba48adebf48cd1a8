// dense.hpp -- what the dense operators over factor tables share (softmax_ce.hip, int8.hip, ortho.hip): element
// types and their roundings, MFMA operand types, the device scope and the checks of device matrices.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "common.hpp"
#include "wave.hpp"
#include "rsgpu_dense.h"

namespace rs {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) double f64x4;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(16))) int i32x16;

// Element types: RS_TYPE_F32 / _BF16 / _F16 as C++ types.  Conversions from float round to nearest, ties to even.
template <int TYPE>
struct Elem;
template <>
struct Elem<RS_TYPE_F32> { using type = float; };
template <>
struct Elem<RS_TYPE_BF16> { using type = __bf16; };
template <>
struct Elem<RS_TYPE_F16> { using type = _Float16; };

inline int64_t type_size(int32_t type) { return type == RS_TYPE_F32 ? 4 : 2; }
inline bool type_ok(int32_t type) { return type == RS_TYPE_F32 || type == RS_TYPE_BF16 || type == RS_TYPE_F16; }

// f(Elem<...>) for the runtime type (checked by type_ok before)
template <typename F>
void with_type(int32_t type, F&& f) {
    if (type == RS_TYPE_F32)
        f(Elem<RS_TYPE_F32>{});
    else if (type == RS_TYPE_BF16)
        f(Elem<RS_TYPE_BF16>{});
    else
        f(Elem<RS_TYPE_F16>{});
}

__host__ __device__ inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
__host__ __device__ inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// A launch holds fewer than 2^32 threads along an axis: many workgroups (of up to 1024 threads) are laid over two, and a
// kernel asks for its number (workgroups past the end find no row and leave).
inline dim3 wide_grid(int64_t workgroups) {
    const int64_t x = std::min<int64_t>(workgroups, int64_t{1} << 21);
    return dim3(static_cast<uint32_t>(x), static_cast<uint32_t>(ceil_div(workgroups, x)));
}
__device__ __forceinline__ int64_t wide_block() { return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x; }

// The caller's current device is put back when an operator returns (its tensors may live on another device than the
// one that is current in the calling thread).
struct DeviceScope {
    int prev = -1;
    explicit DeviceScope(int device) {
        RS_HIP(hipGetDevice(&prev));
        if (prev != device)
            RS_HIP(hipSetDevice(device));
        else
            prev = -1;
    }
    ~DeviceScope() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
};

// Operator entry points: the device scope, and exceptions turned into status codes.
template <typename F>
int dense_guard(rs_ctx* ctx, F&& body) {
    if (!ctx) return set_error(nullptr, RS_ERR_INVALID, "ctx is NULL");
    try {
        DeviceScope scope(ctx->device);
        return body();
    } catch (const HipError& e) {
        return set_error(ctx, e.code == hipErrorOutOfMemory ? RS_ERR_NOMEM : RS_ERR_HIP, e.what);
    } catch (const std::bad_alloc&) {
        return set_error(ctx, RS_ERR_NOMEM, "host allocation failed");
    } catch (const std::exception& e) {
        return set_error(ctx, RS_ERR_INVALID, e.what());
    }
}

// A C entry's whole body: no exception leaves it, the argument checks' strings included (which then have no message).
template <typename F>
int no_throw(F&& body) {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return RS_ERR_NOMEM;
    } catch (...) {
        return RS_ERR_INVALID;
    }
}

// NULL: the ctx stream (as everywhere in the C-ABI); RS_STREAM_DEFAULT: the device's null stream
inline hipStream_t pick_stream(rs_ctx* ctx, void* stream) {
    if (stream == RS_STREAM_DEFAULT) return nullptr;
    return stream ? static_cast<hipStream_t>(stream) : ctx->stream;
}

// A device matrix argument: non-null, aligned to its element, its row stride at least its columns.  Returns the
// complaint, or an empty string.
inline std::string check_matrix(const char* name, const void* p, int64_t cols, int64_t ld, int64_t elem) {
    if (!p) return std::string(name) + " is NULL";
    if (reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(elem))
        return std::string(name) + " is not aligned to its element type";
    if (ld < cols) return std::string(name) + ": row stride below its columns";
    return std::string();
}

// LDS tile of rows of KP 16-bit values: 16-byte chunk c of row r sits at chunk c ^ mix(r), the row's low three bits
// rotated.  A row-wise read (8 rows, one chunk at a time) and a transposing one (4 rows, two neighbouring chunks) then
// both meet every bank once; c ^ (r mod 16) had neighbouring rows share their chunk pairs (half of the LDS cycles were
// conflicts).  Byte offset: what a lane adds is one base, the constant part of c goes in by XOR (bits the rows do not
// reach: by addition), so a few registers hold all the addresses of a tile.
template <int KP>
struct LdsTile {
    static constexpr int C = KP / 8, M = C < 16 ? C - 1 : 15;
    static __device__ __forceinline__ int mix(int row) {
        return KP == 32 ? (row & 2) | ((row >> 2) & 1) : (((row & 3) << 1) | ((row >> 2) & 1) | (row & 8)) & M;
    }
    static __device__ __forceinline__ int base(int row, int c) { return row * (KP * 2) + ((c ^ mix(row)) & M) * 16 + (c & ~M) * 16; }
    // base(row, c) with the constant dc joined to c (no common bits)
    static __device__ __forceinline__ int at(int base, int dc) { return (base ^ ((dc & M) * 16)) + (dc & ~M) * 16; }
};

// LDS written by lanes of a wave before this is read by its other lanes after it
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// maximum over the wave (64 lanes): inside rows of 16 lanes by DPP, the four rows by scalar reads
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto step = [&](auto ctrl) {
        const uint32_t w = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ctrl)::value, 0xF, 0xF, false));
        v = v > w ? v : w;
    };
    step(std::integral_constant<int, DPP_QUAD_XOR1>{});
    step(std::integral_constant<int, DPP_QUAD_XOR2>{});
    step(std::integral_constant<int, DPP_ROW_HALF_MIRROR>{});
    step(std::integral_constant<int, DPP_ROW_MIRROR>{});
    auto lane = [&](int l) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), l)); };
    return max(max(lane(0), lane(16)), max(lane(32), lane(48)));
}
__device__ __forceinline__ float wave_sum_f32(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

}  // namespace rs
