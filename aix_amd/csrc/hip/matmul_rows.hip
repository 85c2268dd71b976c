// matmul_rows.hip -- products of a few rows with an epilogue, 16-bit: out = act(a . b + bias) + residual for at most 16 rows
// of a.  Reading b once is all there is to do, so b goes from memory to the matrix unit on the shortest way and everything
// else serves to have enough of it in flight: a workgroup owns COLS columns, its eight waves share K between them, each fetches
// the words of four K steps at a time, and the eight partial results meet in LDS, where the epilogue finishes them.
//
// C^T = B^T A^T with v_mfma 16x16x32: a lane of the result holds four columns of one row.  b as rows of K (unit stride along
// N): the words of 32 K rows pass through a slab of LDS that belongs to the wave alone and are read back transposed, as the
// values of attention_split_k; b as rows of N (unit stride along K): they are the operand as they lie.
#pragma clang fp contract(fast)

#include "attention.hpp"
#include "attention_host.hpp"
#include "epilogue.hpp"

using namespace aixd;
using namespace aixk;
using namespace aixk::attn;

namespace {

struct RowsArgs {
    const void *a, *b; void* c;
    u64 lda, ldb;                             // elements between rows of a, between K rows (BT) or N rows of b
    u32 M, N, K;
    u32 per;                                  // K steps of 32 per share
    float* partial;                           // [share][M][N], or null
    EpiArgs epi;
};

constexpr int kWaves = 8, kAhead = 4;

// Workgroups go round the 8 XCDs one by one; number them so that each XCD works on a contiguous run of columns.  A bijection for any n.
__device__ __forceinline__ u32 xcd_order(u32 id, u32 n)
{
    const u32 q = n / 8u, r = n % 8u, x = id % 8u;
    return x * q + (x < r ? x : r) + id / 8u;
}

// slot of 16-byte word c of K row k in a slab: the transposed reads take 32 bytes from each of eight K rows at a time
template <int WORDS> __device__ __forceinline__ int turn(int k)
{
    if constexpr (WORDS >= 8) return ((k >> 1) & 3) << 1;
    else return ((k >> 2) & 1) << 1;
}
// where the partial result of column c of a row is kept: the rows of a wave start on the same banks
template <int COLS> __device__ __forceinline__ int beside(int row, int c) { return c ^ (4 * (row & (COLS / 4 - 1) & 15)); }

template <bool BT, int COLS> constexpr size_t rows_lds()
{
    constexpr size_t slab = BT ? (size_t)kWaves * 32 * COLS * 2 : 0, join = (size_t)kWaves * 16 * COLS * 4;
    return slab > join ? slab : join;
}

template <class T, bool BT, int COLS>
__global__ __launch_bounds__(kWaves * 64) void matmul_rows_k(RowsArgs g)
{
    typedef Mma<T> M;
    typedef typename M::Frag Frag;
    constexpr int NB = COLS / 16, WORDS = COLS / 8, NW = 32 * WORDS / 64, PITCH = COLS * 2;      // BT: words per K row, per lane and step
    constexpr int SLAB = BT ? 32 * PITCH : 0;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, c15 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const u32 n0 = xcd_order(blockIdx.x, gridDim.x) * COLS;             // neighbours, who share lines of b, on one XCD
    const u32 steps = (g.K + 31) / 32, first = blockIdx.y * g.per, last = first + g.per < steps ? first + g.per : steps;
    const T* A = (const T*)g.a;
    const T* B = (const T*)g.b;
    char* slab = lds + wave * SLAB;

    f32x4 acc[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[n] = f32x4{};

    // K index of element j of a lane: transposed reads number it 16 (j / 4) + 4 q + j % 4, rows of N 8 q + j
    u32x4 bw[kAhead][BT ? NW : NB];
    u32x2 aw[kAhead][2];
    const T* row = A + (u64)(c15 < (int)g.M ? c15 : 0) * g.lda;
    auto load = [&](int slot, u32 step) {
        const u32 k0 = step * 32;
#pragma unroll
        for (int w = 0; w < (BT ? NW : NB); ++w) {
            if constexpr (BT) {
                const int e = lane + 64 * w;
                const u32 k = k0 + e / WORDS, n = n0 + e % WORDS * 8;
                bw[slot][w] = *(const u32x4*)(B + (u64)(k < g.K ? k : g.K - 1) * g.ldb + (n < g.N ? n : 0));
            } else {
                const u32 n = n0 + w * 16 + c15, k = k0 + 8 * q;
                bw[slot][w] = *(const u32x4*)(B + (u64)(n < g.N ? n : 0) * g.ldb + (k < g.K ? k : 0));
            }
        }
        const u32 ka = BT ? k0 + 4 * q : k0 + 8 * q, kb = BT ? ka + 16 : ka + 4;
        aw[slot][0] = *(const u32x2*)(row + (ka < g.K ? ka : 0));
        aw[slot][1] = *(const u32x2*)(row + (kb < g.K ? kb : 0));
    };
    auto multiply = [&](int slot, u32 step) {
        const u32 k0 = step * 32;
        if constexpr (BT) {
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const int e = lane + 64 * w, k = e / WORDS, word = e % WORDS;
                *(u32x4*)(slab + k * PITCH + ((word ^ turn<WORDS>(k)) << 4)) = k0 + k < g.K ? bw[slot][w] : u32x4{0, 0, 0, 0};
            }
        }
        Frag f[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            if constexpr (BT) {
                const int k = 4 * q + (c15 >> 2), word = 2 * n + ((c15 & 3) >> 1);
                const char* lo = slab + k * PITCH + ((word ^ turn<WORDS>(k)) << 4) + 8 * (c15 & 1);
                const char* hi = slab + (k + 16) * PITCH + ((word ^ turn<WORDS>(k + 16)) << 4) + 8 * (c15 & 1);
                const u32x2 lw = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)lo));
                const u32x2 hw = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)hi));
                f[n] = u32x4{lw.x, lw.y, hw.x, hw.y};
            } else f[n] = k0 + 8 * q < g.K ? bw[slot][n] : M::zero();
        }
        const u32 ka = BT ? k0 + 4 * q : k0 + 8 * q, kb = BT ? ka + 16 : ka + 4;
        const u32x2 lo = ka < g.K ? aw[slot][0] : u32x2{0, 0}, hi = kb < g.K ? aw[slot][1] : u32x2{0, 0};
        const Frag x = u32x4{lo.x, lo.y, hi.x, hi.y};
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[n] = M::run16(f[n], x, acc[n]);
    };
    // steps first + wave, + 8, ...: kAhead of them in flight; loads behind the last step repeat it
    if (first + wave < last) {
        const u32 mine = (last - first - wave + kWaves - 1) / kWaves, at = first + wave;
        auto step_of = [&](u32 n) { return at + (n < mine ? n : mine - 1) * kWaves; };
#pragma unroll
        for (int d = 0; d < kAhead; ++d) load(d, step_of(d));
        u32 n = 0;
        for (; n + kAhead <= mine; n += kAhead) {
#pragma unroll
            for (int d = 0; d < kAhead; ++d) { multiply(d, step_of(n + d)); load(d, step_of(n + d + kAhead)); }
        }
#pragma unroll
        for (int d = 0; d < kAhead; ++d) if (n + d < mine) multiply(d, step_of(n + d));
    }

    // [wave][row][COLS] partial results; a lane's four columns stand together
    __syncthreads();
    float* all = (float*)lds;
#pragma unroll
    for (int n = 0; n < NB; ++n) *(f32x4*)(all + (wave * 16 + c15) * COLS + beside<COLS>(c15, n * 16 + 4 * q)) = acc[n];
    __syncthreads();
    const bool whole = g.epi.whole && !g.partial;
    for (u32 e = tid; e < 16 * COLS / 8; e += kWaves * 64) {
        const u32 row = e / (COLS / 8), c = e % (COLS / 8) * 8, m = row, n = n0 + c;
        if (m >= g.M || n >= g.N) continue;
        float x[8] = {};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float* p = all + (w * 16 + row) * COLS;
            const f32x4 lo = *(const f32x4*)(p + beside<COLS>(row, c)), hi = *(const f32x4*)(p + beside<COLS>(row, c + 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) { x[j] += lo[j]; x[4 + j] += hi[j]; }
        }
        T* C = (T*)g.c;
        if (whole) {
            epilogue8<T>(x, g.epi, m, n, g.N);
            put8(C + (u64)m * g.N + n, x);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (n + j >= g.N) break;
                if (g.partial) g.partial[((u64)blockIdx.y * g.M + m) * g.N + n + j] = x[j];
                else C[(u64)m * g.N + n + j] = down<T>(epilogue1<T>(x[j], g.epi, m, n + j, g.N));
            }
        }
    }
}

} // namespace

namespace aixk {

// a: rows of unit stride, lda elements apart; b: rows of N (bt = false) or of K (bt = true), ldb elements apart; both with whole
// 16-byte words.  *shares > 1: K was shared out over workgroups and *partial holds [share][M][N] to be finished.
int matmul_rows(aixk_ctx* ctx, int dtype, const void* a, u64 lda, const void* b, u64 ldb, bool bt, void* out, u64 M, u64 N, u64 K, const EpiArgs& epi, u32* shares, float** partial)
{
    RowsArgs g{a, b, out, lda, ldb, (u32)M, (u32)N, (u32)K, 0, nullptr, epi};
    // 64 columns where they still give every second compute unit a workgroup (whole 128-byte lines of b), else 32
    const bool wide = (N + 63) / 64 >= (u64)ctx->cus / 2;
    const u64 across = wide ? (N + 63) / 64 : (N + 31) / 32, steps = (K + 31) / 32;
    // shares of K where the columns leave compute units idle, and none below four steps per wave (a share costs the pass that adds them up)
    u64 n = (u64)ctx->cus / across;
    if (n > steps / (4 * kWaves)) n = steps / (4 * kWaves);
    if (n < 1) n = 1;
    g.per = (u32)((steps + n - 1) / n);
    n = (steps + g.per - 1) / g.per;
    *shares = (u32)n;
    if (n > 1) {
        void* ws;
        AIXK_TRY(block_scratch(ctx, kScratchParts, (size_t)(n * M * N) * sizeof(float), &ws));
        g.partial = *partial = (float*)ws;
    }
    auto launch = [&](auto type, auto form, auto cols_tag) -> int {
        typedef decltype(type) T;
        constexpr bool BT = decltype(form)::value;
        constexpr int COLS = decltype(cols_tag)::value;
        constexpr size_t lds = rows_lds<BT, COLS>();
        AIXK_TRY(allow_lds(matmul_rows_k<T, BT, COLS>, lds));
        hipLaunchKernelGGL((matmul_rows_k<T, BT, COLS>), dim3((unsigned)across, (unsigned)n), dim3(kWaves * 64), lds, ctx->stream, g);
        AIXK_HIP(hipGetLastError());
        return AIXK_OK;
    };
    auto by_size = [&](auto type, auto form) -> int {
        return wide ? launch(type, form, std::integral_constant<int, 64>{}) : launch(type, form, std::integral_constant<int, 32>{});
    };
    auto by_form = [&](auto type) -> int { return bt ? by_size(type, std::true_type{}) : by_size(type, std::false_type{}); };
    return dtype == AIXK_BF16 ? by_form(bf16{}) : by_form(f16{});
}

} // namespace aixk
