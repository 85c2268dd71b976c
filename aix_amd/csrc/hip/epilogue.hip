// epilogue.hip -- matrix products with bias, activation and residual, and their backward pass: the checks, and the pass that
// forms dz = grad act'(pre) together with its column sums.  The forward kernels are those of matmul_mfma.hip.
#pragma clang fp contract(fast)

#include "attention_host.hpp"
#include "epilogue.hpp"

using namespace aixd;
using namespace aixk;

namespace aixk {
int matmul_mfma_epilogue(aixk_ctx* ctx, const aixhip_tensor* a, const aixhip_tensor* b, const aixhip_tensor* out, const EpiArgs& epi);      // matmul_mfma.hip
int matmul_plain(aixk_ctx* ctx, const aixhip_tensor* a, const aixhip_tensor* b, const aixhip_tensor* out);
}

namespace {

struct SlopeArgs {
    const void *grad, *pre; u64 g0, g1, p0, p1;
    void* dz;                                  // or null
    float* sums;                               // [row chunk][N] or null
    u64 M, N, rows;                            // rows per chunk
    i32 act;
};

// One pass over grad and pre.  WIDE: a lane owns eight columns, 32 lanes side by side, eight rows at a time; otherwise a lane
// owns one column, 64 side by side, four rows at a time.  The rows' sums of a chunk meet in LDS and leave as one partial
// sum per column and chunk; sum_chunks_k adds those in their order.
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void slope_k(SlopeArgs a)
{
    constexpr int C = WIDE ? 8 : 1, LANES = WIDE ? 32 : 64, ROWS = 256 / LANES;
    __shared__ float sums[ROWS][LANES * C];
    const int lane = threadIdx.x % LANES, r = threadIdx.x / LANES;
    const u64 col = ((u64)blockIdx.x * LANES + lane) * C;
    const u64 from = (u64)blockIdx.y * a.rows, to = from + a.rows < a.M ? from + a.rows : a.M;
    const T* G = (const T*)a.grad;
    const T* P = (const T*)a.pre;
    T* Z = (T*)a.dz;
    float sum[C] = {};
    if (col < a.N) {
        for (u64 row = from + r; row < to; row += ROWS) {
            if constexpr (WIDE) {
                float g[8], z[8];
                get8(G + row * a.g0 + col, g);
                if (a.act) {
                    get8(P + row * a.p0 + col, z);
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[j] *= slope(z[j], a.act);
                }
                if (Z) put8(Z + row * a.N + col, g);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j] += g[j];
            } else {
                float g = up<T>(G[row * a.g0 + col * a.g1]);
                if (a.act) g *= slope(up<T>(P[row * a.p0 + col * a.p1]), a.act);
                if (Z) Z[row * a.N + col] = down<T>(g);
                sum[0] += g;
            }
        }
    }
    if (!a.sums) return;
#pragma unroll
    for (int j = 0; j < C; ++j) sums[r][lane * C + j] = sum[j];
    __syncthreads();
    for (int c = threadIdx.x; c < LANES * C; c += 256) {
        const u64 at = (u64)blockIdx.x * LANES * C + c;
        if (at >= a.N) continue;
        float total = 0.0f;
#pragma unroll
        for (int k = 0; k < ROWS; ++k) total += sums[k][c];
        a.sums[(u64)blockIdx.y * a.N + at] = total;
    }
}

// 16 columns per workgroup, 16 lanes on each (eight lanes that wait for a load per chunk: 11 us for 256 chunks of 768 columns)
template <class T>
__global__ __launch_bounds__(256) void sum_chunks_k(const float* sums, T* out, u64 N, u32 chunks)
{
    __shared__ float part[16][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
    const u64 col = (u64)blockIdx.x * 16 + c;
    float total = 0.0f;
    if (col < N) {
#pragma unroll 8
        for (u32 k = r; k < chunks; k += 16) total += sums[(u64)k * N + col];
    }
    part[r][c] = total;
    __syncthreads();
    if (r == 0 && col < N) {
#pragma unroll
        for (int k = 1; k < 16; ++k) total += part[k][c];
        out[col] = down<T>(total);
    }
}

bool float_type(int dtype) { return dtype == AIXK_F32 || dtype == AIXK_F16 || dtype == AIXK_BF16; }
bool matrix(const aixhip_tensor* t, int dtype, uint64_t rows, uint64_t cols)
{
    return valid_tensor(t) && t->rank == 2 && t->dtype == dtype && t->shape[0] == rows && t->shape[1] == cols && t->size == rows * cols;
}
bool dense(const aixhip_tensor* t)
{
    uint64_t run = 1;
    for (int d = t->rank - 1; d >= 0; --d) {
        if (t->shape[d] > 1 && t->strides[d] != run) return false;
        run *= t->shape[d];
    }
    return true;
}
// [n] or [1, n]
bool row_vector(const aixhip_tensor* t, int dtype, uint64_t n)
{
    return valid_tensor(t) && t->dtype == dtype && t->size == n && ((t->rank == 1 && t->shape[0] == n) || (t->rank == 2 && t->shape[0] == 1 && t->shape[1] == n));
}
char* start(const aixhip_tensor* t) { return (char*)t->data + t->offset * aixk_dtype_size(t->dtype); }
// the kernels write from `data` on
aixhip_tensor from_start(const aixhip_tensor* t)
{
    aixhip_tensor d = *t;
    d.data = start(t);
    d.offset = 0;
    for (int k = t->rank - 1; k >= 0; --k) d.strides[k] = k == t->rank - 1 ? 1 : d.strides[k + 1] * t->shape[k + 1];
    return d;
}
aixhip_tensor transposed(const aixhip_tensor* t)
{
    aixhip_tensor d = *t;
    d.shape[0] = t->shape[1]; d.shape[1] = t->shape[0];
    d.strides[0] = t->strides[1]; d.strides[1] = t->strides[0];
    return d;
}

} // namespace

extern "C" int32_t aixk_matmul_epilogue(aixk_ctx* ctx, const aixhip_tensor* a, const aixhip_tensor* b, const aixk_epilogue* e, const aixhip_tensor* out)
{
    const char* what = "matmul_epilogue";
    AIXK_REQUIRE(e != nullptr, "%s: null epilogue", what);
    AIXK_REQUIRE(valid_tensor(a) && valid_tensor(b) && a->rank == 2 && b->rank == 2 && a->size == numel(a) && b->size == numel(b), "%s: operands must be 2-D", what);
    AIXK_REQUIRE(a->shape[1] == b->shape[0], "%s: inner dimensions differ", what);
    AIXK_REQUIRE(float_type(a->dtype) && b->dtype == a->dtype, "%s: operands must have one element type, f32, f16 or bf16", what);
    const uint64_t M = a->shape[0], N = b->shape[1];
    const int dt = a->dtype;
    AIXK_REQUIRE(matrix(out, dt, M, N) && dense(out), "%s: the result must be a dense [M, N] of the operands' type", what);
    AIXK_REQUIRE(!e->bias || row_vector(e->bias, dt, N), "%s: the bias must be [N] of the operands' type", what);
    AIXK_REQUIRE(!e->residual || matrix(e->residual, dt, M, N), "%s: the residual must be [M, N] of the operands' type", what);
    AIXK_REQUIRE(!e->pre || (matrix(e->pre, dt, M, N) && dense(e->pre)), "%s: pre must be a dense [M, N] of the operands' type", what);
    AIXK_REQUIRE(e->activation >= AIXK_ACT_NONE && e->activation <= AIXK_ACT_SILU, "%s: unknown activation %d", what, e->activation);
    AIXK_REQUIRE(!overlap(out, a) && !overlap(out, b) && !overlap(out, e->bias), "%s: the result overlaps an operand", what);
    AIXK_REQUIRE(!overlap(out, e->residual) || (start(out) == start(e->residual) && dense(e->residual)), "%s: the result overlaps the residual (in place means the same dense view)", what);
    AIXK_REQUIRE(!overlap(e->pre, a) && !overlap(e->pre, b) && !overlap(e->pre, e->bias) && !overlap(e->pre, e->residual) && !overlap(e->pre, out), "%s: pre overlaps an operand or the result", what);
    AIXK_TRY(set_device(ctx));
    if (M == 0 || N == 0) return AIXK_OK;
    EpiArgs epi{};
    const size_t es = aixk_dtype_size(dt);
    epi.act = e->activation;
    bool whole = N % 8 == 0 && aligned16(start(out));
    if (e->bias) {
        epi.bias = start(e->bias);
        epi.bias_step = e->bias->strides[e->bias->rank - 1];
        whole = whole && epi.bias_step == 1 && aligned16(epi.bias);
    }
    if (e->residual) {
        epi.res = start(e->residual);
        epi.rs0 = e->residual->strides[0]; epi.rs1 = e->residual->strides[1];
        whole = whole && epi.rs1 == 1 && (M == 1 || epi.rs0 % (16 / es) == 0) && aligned16(epi.res);
    }
    if (e->pre) { epi.pre = start(e->pre); whole = whole && aligned16(epi.pre); }
    epi.whole = whole;
    const aixhip_tensor o = from_start(out);
    return matmul_mfma_epilogue(ctx, a, b, &o, epi);
}

extern "C" int32_t aixk_matmul_epilogue_backward(aixk_ctx* ctx, const aixhip_tensor* grad, const aixhip_tensor* a, const aixhip_tensor* b, const aixhip_tensor* pre,
                                                 int32_t activation, const aixhip_tensor* dz, const aixhip_tensor* da, const aixhip_tensor* db, const aixhip_tensor* dbias)
{
    const char* what = "matmul_epilogue_backward";
    AIXK_REQUIRE(valid_tensor(a) && valid_tensor(b) && a->rank == 2 && b->rank == 2 && a->size == numel(a) && b->size == numel(b), "%s: operands must be 2-D", what);
    AIXK_REQUIRE(a->shape[1] == b->shape[0], "%s: inner dimensions differ", what);
    AIXK_REQUIRE(float_type(a->dtype) && b->dtype == a->dtype, "%s: operands must have one element type, f32, f16 or bf16", what);
    const uint64_t M = a->shape[0], K = a->shape[1], N = b->shape[1];
    const int dt = a->dtype;
    AIXK_REQUIRE(activation >= AIXK_ACT_NONE && activation <= AIXK_ACT_SILU, "%s: unknown activation %d", what, activation);
    AIXK_REQUIRE(matrix(grad, dt, M, N), "%s: grad must be [M, N] of the operands' type", what);
    AIXK_REQUIRE(!pre || matrix(pre, dt, M, N), "%s: pre must be [M, N] of the operands' type", what);
    AIXK_REQUIRE(!dz || (matrix(dz, dt, M, N) && dense(dz)), "%s: dz must be a dense [M, N] of the operands' type", what);
    AIXK_REQUIRE(activation == AIXK_ACT_NONE || (pre && dz), "%s: an activation needs pre and dz", what);
    AIXK_REQUIRE(!da || (matrix(da, dt, M, K) && dense(da)), "%s: da must be a dense [M, K] of the operands' type", what);
    AIXK_REQUIRE(!db || (matrix(db, dt, K, N) && dense(db)), "%s: db must be a dense [K, N] of the operands' type", what);
    AIXK_REQUIRE(!dbias || (row_vector(dbias, dt, N) && dense(dbias)), "%s: dbias must be a dense [N] of the operands' type", what);
    const aixhip_tensor* results[] = {dz, da, db, dbias};
    const aixhip_tensor* operands[] = {grad, a, b, pre};
    for (int r = 0; r < 4; ++r) {
        for (const aixhip_tensor* o : operands) AIXK_REQUIRE(!overlap(results[r], o), "%s: a result overlaps an operand", what);
        for (int s = r + 1; s < 4; ++s) AIXK_REQUIRE(!overlap(results[r], results[s]), "%s: results overlap", what);
    }
    AIXK_TRY(set_device(ctx));

    if ((dz || dbias) && N > 0) {
        const size_t es = aixk_dtype_size(dt);
        SlopeArgs s{};
        s.grad = start(grad); s.g0 = grad->strides[0]; s.g1 = grad->strides[1];
        s.act = activation; s.M = M; s.N = N;
        bool wide = N % 8 == 0 && s.g1 == 1 && (M <= 1 || s.g0 % (16 / es) == 0) && aligned16(s.grad);
        if (activation != AIXK_ACT_NONE) {
            s.pre = start(pre); s.p0 = pre->strides[0]; s.p1 = pre->strides[1];
            wide = wide && s.p1 == 1 && (M <= 1 || s.p0 % (16 / es) == 0) && aligned16(s.pre);
        }
        if (dz) { s.dz = start(dz); wide = wide && aligned16(s.dz); }
        // chunks of rows until every compute unit has four workgroups, none below 32 rows
        const u64 across = (N + (wide ? 255 : 63)) / (wide ? 256 : 64);
        u64 chunks = ((u64)ctx->cus * 4 + across - 1) / across;
        if (chunks > (M + 31) / 32) chunks = (M + 31) / 32;
        if (chunks > 65535) chunks = 65535;
        if (chunks < 1) chunks = 1;
        s.rows = (M + chunks - 1) / chunks;
        if (s.rows == 0) s.rows = 1;
        chunks = M ? (M + s.rows - 1) / s.rows : 1;
        AIXK_REQUIRE(across < (1ull << 31), "%s: too many columns", what);
        if (dbias) {
            void* ws;
            AIXK_TRY(block_scratch(ctx, attn::kScratchColumns, (size_t)(chunks * N) * sizeof(float), &ws));
            s.sums = (float*)ws;
        }
        auto run = [&](auto type) -> int {
            typedef decltype(type) T;
            const dim3 grid((unsigned)across, (unsigned)chunks);
            if (wide) hipLaunchKernelGGL((slope_k<T, true>), grid, dim3(256), 0, ctx->stream, s);
            else hipLaunchKernelGGL((slope_k<T, false>), grid, dim3(256), 0, ctx->stream, s);
            AIXK_HIP(hipGetLastError());
            if (dbias) {
                hipLaunchKernelGGL((sum_chunks_k<T>), dim3((unsigned)((N + 15) / 16)), dim3(256), 0, ctx->stream, (const float*)s.sums, (T*)start(dbias), (u64)N, (u32)chunks);
                AIXK_HIP(hipGetLastError());
            }
            return AIXK_OK;
        };
        AIXK_TRY(dt == AIXK_F32 ? run(float{}) : dt == AIXK_F16 ? run(f16{}) : run(bf16{}));
    }
    const aixhip_tensor* z = dz ? dz : grad;
    if (da && M && K) {
        const aixhip_tensor bt = transposed(b), o = from_start(da);
        AIXK_TRY(matmul_plain(ctx, z, &bt, &o));
    }
    if (db && K && N) {
        const aixhip_tensor at = transposed(a), o = from_start(db);
        AIXK_TRY(matmul_plain(ctx, &at, z, &o));
    }
    return AIXK_OK;
}
