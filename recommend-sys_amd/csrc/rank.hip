// rank.hip -- the dense operators on a plan's resident factors: a training step for ranking over the whole catalogue
// (softmax cross entropy, its gradient, the orthogonalised update of the item table) and the whole catalogue's scores
// in 8 bits.  The plan's rows are [factors, bias, padding] of stride ld; the operators read the factor columns in place.
#include <hip/hip_runtime.h>

#include <cmath>
#include <numeric>

#include "dense.hpp"
#include "sgd_plan.hpp"

namespace rs {
namespace {

// dst row r = the factors of users[r], zeros for an unknown one; a wave per row
__global__ __launch_bounds__(256) void rank_gather_kernel(const float* __restrict__ P, int32_t ld, int32_t k, int32_t n_users, int64_t n,
                                                         const int32_t* __restrict__ users, float* __restrict__ dst) {
    const int lane = threadIdx.x & 63;
    const int64_t r = wide_block() * 4 + (threadIdx.x >> 6);
    if (r >= n) return;
    const int32_t u = users[r];
    const bool known = static_cast<uint32_t>(u) < static_cast<uint32_t>(n_users);
    for (int c = lane; c < k; c += 64) dst[r * k + c] = known ? P[static_cast<int64_t>(u) * ld + c] : 0.f;
}

// the bias column of a table
__global__ __launch_bounds__(256) void rank_bias_kernel(const float* __restrict__ T, int32_t ld, int32_t k, int64_t rows, float* __restrict__ out) {
    const int64_t r = wide_block() * 256 + threadIdx.x;
    if (r < rows) out[r] = T[r * ld + k];
}

// GlobalBias + b_u (unknown users: GlobalBias)
__global__ __launch_bounds__(256) void rank_row_bias_kernel(const float* __restrict__ P, int32_t ld, int32_t k, int32_t n_users, int64_t n,
                                                           const int32_t* __restrict__ users, const double* __restrict__ gb, float* __restrict__ out) {
    const int64_t r = wide_block() * 256 + threadIdx.x;
    if (r >= n) return;
    const int32_t u = users[r];
    const bool known = static_cast<uint32_t>(u) < static_cast<uint32_t>(n_users);
    out[r] = static_cast<float>(gb[0] + (known ? static_cast<double>(P[static_cast<int64_t>(u) * ld + k]) : 0.0));
}

// A value's step.  APPLY: it is written, unless the step was found to make some finite value no number; otherwise that is
// found out (*bad), and nothing written.
template <bool APPLY>
__device__ __forceinline__ void take_step(float* at, float next, int32_t* bad) {
    if (APPLY)
        *at = next;
    else if (!(fabsf(next) < INFINITY) && fabsf(*at) < INFINITY)
        *bad = 1;
}

// one user of the batch a wave: its rows of dH in batch order, then its step
template <bool APPLY>
__global__ __launch_bounds__(256) void rank_users_kernel(float* __restrict__ P, int32_t ld, int32_t k, const int32_t* __restrict__ seg,
                                                        const int32_t* __restrict__ seg_user, const int32_t* __restrict__ rows, int64_t n_seg,
                                                        const float* __restrict__ dH, float lr, float decay, int32_t* bad) {
    const int lane = threadIdx.x & 63;
    const int64_t s = wide_block() * 4 + (threadIdx.x >> 6);
    if (s >= n_seg || (APPLY && *bad)) return;
    const int32_t a = seg[s], b = seg[s + 1];
    float* p = P + static_cast<int64_t>(seg_user[s]) * ld;
    const float shrink = decay * static_cast<float>(b - a);
    for (int c = lane; c < k; c += 64) {
        float g = 0.f;
        for (int32_t i = a; i < b; ++i) g += dH[static_cast<int64_t>(rows[i]) * k + c];
        take_step<APPLY>(p + c, p[c] - lr * (g + shrink * p[c]), bad);
    }
}

// Q -= q_lr (O + reg Q), b -= lr db
template <bool APPLY>
__global__ __launch_bounds__(256) void rank_items_kernel(float* __restrict__ Q, int32_t ld, int32_t k, int64_t n_items, const float* __restrict__ O,
                                                        const float* __restrict__ db, float lr, float q_lr, float reg, int32_t* bad) {
    const int lane = threadIdx.x & 63;
    const int64_t v = wide_block() * 4 + (threadIdx.x >> 6);
    if (v >= n_items || (APPLY && *bad)) return;
    float* q = Q + v * ld;
    for (int c = lane; c < k; c += 64) take_step<APPLY>(q + c, q[c] - q_lr * (O[v * k + c] + reg * q[c]), bad);
    if (lane == 0) take_step<APPLY>(q + k, q[k] - lr * db[v], bad);
}

// a piece of the plan's workspace at a time
struct Carver {
    int64_t at = 0;
    int64_t take(int64_t bytes) {
        const int64_t o = at;
        at += round_up(bytes, 256);
        return o;
    }
};

char* workspace(rs_svd_plan* pl, int64_t bytes) {
    if (!pl->rank_ws.p || pl->rank_ws.n < static_cast<size_t>(bytes)) pl->rank_ws.alloc(static_cast<size_t>(bytes));
    return pl->rank_ws.p;
}

void check(rs_svd_plan* pl, int status) {  // an operator's refusal, as this call's
    if (status == RS_OK) return;
    if (status == RS_ERR_HIP || status == RS_ERR_NOMEM) throw HipError{status == RS_ERR_NOMEM ? hipErrorOutOfMemory : hipErrorUnknown, pl->ctx->err};
    throw std::invalid_argument(pl->ctx->err);
}

void rank_step(rs_svd_plan* pl, int64_t n, const int32_t* users, const int32_t* items, float lr, float q_lr, float reg, double* loss) {
    const int32_t k = pl->k, ld = pl->ld;
    const int64_t V = pl->n_items;
    // the known interactions by user, in batch order inside a user
    std::vector<int32_t> target(static_cast<size_t>(n), -1), rows;
    for (int64_t r = 0; r < n; ++r)
        if (static_cast<uint32_t>(users[r]) < static_cast<uint32_t>(pl->n_users) && static_cast<uint32_t>(items[r]) < static_cast<uint32_t>(pl->n_items)) {
            target[static_cast<size_t>(r)] = items[r];
            rows.push_back(static_cast<int32_t>(r));
        }
    if (loss) *loss = std::nan("");
    const int64_t m = static_cast<int64_t>(rows.size());
    if (m == 0) return;
    std::stable_sort(rows.begin(), rows.end(), [&](int32_t a, int32_t b) { return users[a] < users[b]; });
    std::vector<int32_t> seg, seg_user;
    for (int64_t i = 0; i < m; ++i)
        if (i == 0 || users[rows[i]] != users[rows[i - 1]]) {
            seg.push_back(static_cast<int32_t>(i));
            seg_user.push_back(users[rows[i]]);
        }
    const int64_t n_seg = static_cast<int64_t>(seg_user.size());
    seg.push_back(static_cast<int32_t>(m));
    const std::vector<float> weight(static_cast<size_t>(n), static_cast<float>(1.0 / static_cast<double>(m)));

    int64_t ce_bytes = 0, or_bytes = 0;
    check(pl, rs_softmax_ce_workspace(pl->ctx, RS_TYPE_F32, n, V, k, 1, &ce_bytes));
    check(pl, rs_orthogonalize_workspace(pl->ctx, V, k, &or_bytes));
    const bool in_place = std::min<int64_t>(V, k) <= 256;
    Carver c;
    const int64_t o_users = c.take(n * 4), o_tgt = c.take(n * 4), o_w = c.take(n * 4), o_rows = c.take(m * 4), o_seg = c.take((n_seg + 1) * 4),
                  o_su = c.take(n_seg * 4), o_bad = c.take(4), o_loss = c.take(n * 4), o_lse = c.take(n * 4), o_h = c.take(n * k * 4), o_dh = c.take(n * k * 4),
                  o_bias = c.take(V * 4), o_db = c.take(V * 4), o_dw = c.take(V * k * 4), o_x = in_place ? o_dw : c.take(V * k * 4),
                  o_ws = c.take(std::max(ce_bytes, or_bytes));
    plan_sync_last(pl);
    char* ws = workspace(pl, c.at);
    hipStream_t s = pl->ctx->stream;
    auto f = [&](int64_t o) { return reinterpret_cast<float*>(ws + o); };
    auto i32 = [&](int64_t o) { return reinterpret_cast<int32_t*>(ws + o); };
    auto up = [&](int64_t o, const void* h, int64_t bytes) { RS_HIP(hipMemcpyAsync(ws + o, h, static_cast<size_t>(bytes), hipMemcpyHostToDevice, s)); };
    up(o_users, users, n * 4);
    up(o_tgt, target.data(), n * 4);
    up(o_w, weight.data(), n * 4);
    up(o_rows, rows.data(), m * 4);
    up(o_seg, seg.data(), (n_seg + 1) * 4);
    up(o_su, seg_user.data(), n_seg * 4);
    rank_gather_kernel<<<wide_grid(ceil_div(n, 4)), 256, 0, s>>>(pl->P.p, ld, k, pl->n_users, n, i32(o_users), f(o_h));
    RS_HIP(hipGetLastError());
    rank_bias_kernel<<<wide_grid(ceil_div(V, 256)), 256, 0, s>>>(pl->Q.p, ld, k, V, f(o_bias));
    RS_HIP(hipGetLastError());
    check(pl, rs_softmax_ce(pl->ctx, RS_TYPE_F32, n, V, k, f(o_h), k, pl->Q.p, ld, f(o_bias), i32(o_tgt), f(o_w), f(o_loss), f(o_lse), f(o_dh), k,
                            f(o_dw), k, f(o_db), ws + o_ws, ce_bytes, nullptr));
    check(pl, rs_orthogonalize(pl->ctx, RS_TYPE_F32, V, k, f(o_dw), k, 5, 3.4445, -4.7750, 2.0315, f(o_x), k, ws + o_ws, or_bytes, nullptr));
    // both tables' steps are looked through before either is written: a step that a logit or the rates throw out of fp32
    // leaves the plan as it was
    RS_HIP(hipMemsetAsync(ws + o_bad, 0, 4, s));
    auto step = [&](auto apply) {
        constexpr bool APPLY = decltype(apply)::value;
        rank_users_kernel<APPLY><<<wide_grid(ceil_div(n_seg, 4)), 256, 0, s>>>(pl->P.p, ld, k, i32(o_seg), i32(o_su), i32(o_rows), n_seg, f(o_dh), lr,
                                                                               reg / static_cast<float>(m), i32(o_bad));
        RS_HIP(hipGetLastError());
        rank_items_kernel<APPLY><<<wide_grid(ceil_div(V, 4)), 256, 0, s>>>(pl->Q.p, ld, k, V, f(o_x), f(o_db), lr, q_lr, reg, i32(o_bad));
        RS_HIP(hipGetLastError());
    };
    step(std::false_type{});
    step(std::true_type{});
    std::vector<float> h(static_cast<size_t>(n));
    int32_t bad = 0;
    RS_HIP(hipMemcpyAsync(h.data(), f(o_loss), static_cast<size_t>(n) * 4, hipMemcpyDeviceToHost, s));
    RS_HIP(hipMemcpyAsync(&bad, ws + o_bad, 4, hipMemcpyDeviceToHost, s));
    RS_HIP(hipStreamSynchronize(s));
    if (bad) throw NumericError{"the ranking step would leave fp32 (a logit, a gradient or a stepped value that is not finite); the plan is unchanged"};
    plan_factors_changed(pl, s);
    RS_HIP(hipStreamSynchronize(s));
    double sum = 0.0;
    for (int64_t r = 0; r < n; ++r)
        if (target[static_cast<size_t>(r)] >= 0) sum += h[static_cast<size_t>(r)];
    if (loss) *loss = sum / static_cast<double>(m);
}

void score_items(rs_svd_plan* pl, int64_t n, const int32_t* users, float* out) {
    const int32_t k = pl->k, ld = pl->ld;
    const int64_t V = pl->n_items, ldq = round_up(k, 16);
    const int64_t batch = std::max<int64_t>(1, std::min<int64_t>(n, (int64_t{1} << 26) / V));  // scores of 256 MiB at a time
    Carver c;
    const int64_t o_users = c.take(n * 4), o_h = c.take(batch * k * 4), o_hq = c.take(batch * ldq), o_hs = c.take(batch * 4), o_rb = c.take(batch * 4),
                  o_q = c.take(V * ldq), o_qs = c.take(V * 4), o_cb = c.take(V * 4), o_out = c.take(batch * V * 4);
    plan_sync_last(pl);
    char* ws = workspace(pl, c.at);
    hipStream_t s = pl->ctx->stream;
    auto f = [&](int64_t o) { return reinterpret_cast<float*>(ws + o); };
    auto i8 = [&](int64_t o) { return reinterpret_cast<int8_t*>(ws + o); };
    RS_HIP(hipMemcpyAsync(ws + o_users, users, static_cast<size_t>(n) * 4, hipMemcpyHostToDevice, s));
    check(pl, rs_quantize_rows(pl->ctx, RS_TYPE_F32, V, k, pl->Q.p, ld, i8(o_q), ldq, f(o_qs), nullptr));
    rank_bias_kernel<<<wide_grid(ceil_div(V, 256)), 256, 0, s>>>(pl->Q.p, ld, k, V, f(o_cb));
    RS_HIP(hipGetLastError());
    for (int64_t r = 0; r < n; r += batch) {
        const int64_t b = std::min(batch, n - r);
        const int32_t* du = reinterpret_cast<int32_t*>(ws + o_users) + r;
        rank_gather_kernel<<<wide_grid(ceil_div(b, 4)), 256, 0, s>>>(pl->P.p, ld, k, pl->n_users, b, du, f(o_h));
        RS_HIP(hipGetLastError());
        rank_row_bias_kernel<<<wide_grid(ceil_div(b, 256)), 256, 0, s>>>(pl->P.p, ld, k, pl->n_users, b, du, pl->gb.p, f(o_rb));
        RS_HIP(hipGetLastError());
        check(pl, rs_quantize_rows(pl->ctx, RS_TYPE_F32, b, k, f(o_h), k, i8(o_hq), ldq, f(o_hs), nullptr));
        check(pl, rs_i8_matmul(pl->ctx, b, V, k, i8(o_hq), ldq, f(o_hs), i8(o_q), ldq, f(o_qs), f(o_rb), f(o_cb), RS_TYPE_F32, f(o_out), V, nullptr));
        RS_HIP(hipMemcpyAsync(out + r * V, f(o_out), static_cast<size_t>(b * V) * 4, hipMemcpyDeviceToHost, s));
    }
    RS_HIP(hipStreamSynchronize(s));
}

}  // namespace
}  // namespace rs

extern "C" int rs_svd_plan_rank_step(rs_svd_plan* pl, int64_t n, const int32_t* users, const int32_t* items, double lr, double q_lr, double reg,
                                     double* loss) {
    if (!pl) return rs::set_error(nullptr, RS_ERR_INVALID, "plan is NULL");
    return rs_guard(pl->ctx, [&]() -> int {
        if (n < 0 || (n > 0 && (!users || !items))) return rs::set_error(pl->ctx, RS_ERR_INVALID, "bad rank step arguments");
        if (n > (int64_t{1} << 20)) return rs::set_error(pl->ctx, RS_ERR_UNSUPPORTED, "a rank step takes at most 2^20 interactions");
        if (!std::isfinite(static_cast<float>(lr)) || !std::isfinite(static_cast<float>(q_lr)) || !std::isfinite(static_cast<float>(reg)))
            return rs::set_error(pl->ctx, RS_ERR_INVALID, "lr, q_lr and reg must be finite floats");
        if (pl->shard) return rs::set_error(pl->ctx, RS_ERR_UNSUPPORTED, "the plan is joined to a group: its factors are replicas");
        rs::rank_step(pl, n, users, items, static_cast<float>(lr), static_cast<float>(q_lr), static_cast<float>(reg), loss);
        return RS_OK;
    });
}

extern "C" int rs_svd_plan_score_items(rs_svd_plan* pl, int64_t n, const int32_t* users, float* out) {
    if (!pl) return rs::set_error(nullptr, RS_ERR_INVALID, "plan is NULL");
    return rs_guard(pl->ctx, [&]() -> int {
        if (n < 0 || (n > 0 && (!users || !out))) return rs::set_error(pl->ctx, RS_ERR_INVALID, "bad score arguments");
        if (n == 0 || pl->n_items == 0) return RS_OK;
        rs::score_items(pl, n, users, out);
        return RS_OK;
    });
}
