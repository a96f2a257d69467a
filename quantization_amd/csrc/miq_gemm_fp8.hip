// Products of block-scaled e4m3 operands on the CDNA4 matrix cores (gfx950).
//
//     out[m, n] = sum_b (xs[b, m] * ws[n / 128, b]) * (sum_{k in block b} x[m, k] * w[n, k])  (+ bias[n])
//
// A block of 128 columns is one K-tile of 128 bytes.  The matrix cores sum a block's products from zero, and the vector unit
// adds the four results a lane, times the block's scale, to the running fp32 sum.  Both operands are rows of K-contiguous
// bytes, staged and read as the int8 GEMM does (miq_gemm_core.h): 16-byte chunks, the same chunk -> lane map for both, so
// the order of k inside an instruction need not be known.
//
// Which instruction.  v_mfma_f32_16x16x128_f8f6f4 takes the codes as they are, a block in one instruction; but it (and the
// 16x16x32 fp8 form) aligns the products of eight neighbouring k to the largest of the eight and drops what lies below 2^-13
// of it (measured: 2^16 + 2^2 gives 2^16 where 2^16 + 2^3 is right; across groups of eight it keeps 24 bits).  On layers'
// operands that is 3e-5 of the result, a hundred times an fp32 sum's error.  v_mfma_f32_16x16x32_bf16 keeps 24 bits
// throughout (1e-8 on the same operands), and e4m3 widens to bf16 exactly (v_cvt_scalef32_pk_bf16_fp8, two codes an
// instruction), at half the rate.
#include "miq_fp8.h"
#include "miq_gemm_core.h"

namespace {

using namespace miq;

struct Fp8Args {
    const uint8_t* x;      // [M, K]
    const float* xs;       // [kblocks, M]
    const uint8_t* w[2];   // [N, K]; the second one of a gated product
    const float* ws[2];    // [ceil(N / 128), kblocks]
    const float* bias;     // [N] or null
    void* out;             // [M, N]; slabs [splits][M][N] (for each weight) of a split product
    int64_t M;
    int N, K, kblocks;
    int tiles_m, tiles_n;
    int kt_per_split;      // K-tiles each blockIdx.y slice sums; 0 = all, straight to `out`
};

// A fragment of 16 rows and one K-tile: the lane's 16-byte chunks (lane >> 4) and 4 + (lane >> 4) of row lane & 15.
struct Codes {
    v4i c[2];
};
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
struct Widened {
    v8bf h[4];
};
__device__ __forceinline__ Widened widen(const Codes& f) {
    Widened r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const int src = f.c[i >> 1][(i & 1) * 2 + d];
            const v2bf lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, 1.0f, false);
            const v2bf hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, 1.0f, true);
            r.h[i][4 * d] = lo[0];
            r.h[i][4 * d + 1] = lo[1];
            r.h[i][4 * d + 2] = hi[0];
            r.h[i][4 * d + 3] = hi[1];
        }
    return r;
}
// The products of one block, summed from zero.
__device__ __forceinline__ v4f block_sum(const Widened& w, const Widened& x) {
    v4f c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.h[i], x.h[i], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ void add_scaled(v4f& acc, v4f c, float s) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(c[e], s, acc[e]);
}

template <int OUT>
__device__ __forceinline__ void store_value(void* out, int64_t i, float v) {
    if constexpr (OUT == MIQ_F32) static_cast<float*>(out)[i] = v;
    else if constexpr (OUT == MIQ_F16) static_cast<_Float16*>(out)[i] = static_cast<_Float16>(v);
    else static_cast<uint16_t*>(out)[i] = f32_to_bf16_bits(v);
}

// Four consecutive outputs of one row, `n` of them inside it.  `vec`: their address is aligned to four elements.
template <int OUT>
__device__ __forceinline__ void store4(void* out, int64_t i, int n, bool vec, v4f v) {
    if (vec && n >= 4) {
        if constexpr (OUT == MIQ_F32) {
            *reinterpret_cast<v4f*>(static_cast<float*>(out) + i) = v;
        } else if constexpr (OUT == MIQ_F16) {
            typedef _Float16 h4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<h4*>(static_cast<_Float16*>(out) + i) =
                h4{static_cast<_Float16>(v[0]), static_cast<_Float16>(v[1]), static_cast<_Float16>(v[2]), static_cast<_Float16>(v[3])};
        } else {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i) = pack4_bf16(v[0], v[1], v[2], v[3]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) store_value<OUT>(out, i + e, v[e]);
    }
}

// Fills one LDS tile: K-tile kt of the ROWS rows at `rows`, `nrows` of which exist.  VEC: 16-byte LDS-DMA through a
// descriptor that ends with the last row (K a multiple of 16); otherwise through registers, for any K and any alignment.
template <int ROWS, int NWAVES, bool VEC>
__device__ __forceinline__ void stage_rows(const uint8_t* rows, int nrows, int K, int kt, char* tile, int wave, int lane) {
    constexpr int kPieces = ROWS / 8, kIters = (kPieces + NWAVES - 1) / NWAVES;
    const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(rows, static_cast<uint32_t>(nrows) * static_cast<uint32_t>(K));
    const int slot = lane & 7;
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
        const int piece = wave + i * NWAVES;   // wave-uniform
        if (kPieces % NWAVES != 0 && piece >= kPieces) break;
        const int r = piece * 8 + (lane >> 3);
        const int k = kt * kTileK + (slot ^ ((r >> 1) & 7)) * kChunk;
        if constexpr (VEC) {
            dma16(rsrc, tile + piece * (8 * kTileK), r < nrows && k < K ? static_cast<uint32_t>(r) * static_cast<uint32_t>(K) + k : kOob);
        } else {
            v4i v = {0, 0, 0, 0};
            if (r < nrows && k < K) {
                const uint8_t* p = rows + static_cast<int64_t>(r) * K + k;
                if (K - k >= kChunk) {
                    __builtin_memcpy(&v, p, kChunk);
                } else {
                    for (int b = 0; b < K - k; ++b) v[b >> 2] |= static_cast<int>(p[b]) << (8 * (b & 3));
                }
            }
            *reinterpret_cast<v4i*>(tile + piece * (8 * kTileK) + lane * kChunk) = v;
        }
    }
}

// BM x BN outputs a workgroup, two K-tile buffers, one barrier a K-tile.
template <int BM, int BN, int WAVES_M, int WAVES_N, int OUT, bool VEC>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N) void gemm_fp8_tile_kernel(Fp8Args g) {
    constexpr int NWAVES = WAVES_M * WAVES_N;
    constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, FM = WM / 16, FN = WN / 16;
    constexpr int STAGE = (BM + BN) * kTileK;
    static_assert(128 % BN == 0, "a tile's columns lie in one 128-row block of the weight");
    extern __shared__ __attribute__((aligned(16))) char smem[];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;
    const int which = blockIdx.z;
    int tm, tn;
    tile_coords(blockIdx.x, gridDim.x, g.tiles_m, g.tiles_n, 8, tm, tn);
    const int64_t m0 = static_cast<int64_t>(tm) * BM;
    const int n0 = tn * BN;
    const int mrows = static_cast<int>(g.M - m0 < BM ? g.M - m0 : BM), nrows = g.N - n0 < BN ? g.N - n0 : BN;
    const uint8_t* xrows = g.x + m0 * g.K;
    const uint8_t* wrows = g.w[which] + static_cast<int64_t>(n0) * g.K;
    const float* wscale = g.ws[which] + static_cast<int64_t>(n0 / 128) * g.kblocks;

    const int kt0 = g.kt_per_split ? static_cast<int>(blockIdx.y) * g.kt_per_split : 0;
    const int kt1 = g.kt_per_split && kt0 + g.kt_per_split < g.kblocks ? kt0 + g.kt_per_split : g.kblocks;
    void* out = g.out;
    if constexpr (OUT == MIQ_F32) {
        if (g.kt_per_split) out = static_cast<float*>(out) + (static_cast<int64_t>(which) * gridDim.y + blockIdx.y) * g.M * g.N;
    }

    v4f acc[FM][FN] = {};
    const int lo0 = frag_lane_offset(lane, 0), lo1 = frag_lane_offset(lane, 1);
    int64_t row[FM];   // this lane's rows, held inside the matrix for the scales' loads
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int64_t m = m0 + wm * WM + i * 16 + (lane & 15);
        row[i] = m < g.M ? m : g.M - 1;
    }
    auto stage = [&](int kt) {
        char* buf = smem + (kt & 1) * STAGE;
        stage_rows<BM, NWAVES, VEC>(xrows, mrows, g.K, kt, buf, wave, lane);
        stage_rows<BN, NWAVES, VEC>(wrows, nrows, g.K, kt, buf + BM * kTileK, wave, lane);
    };
    if (kt0 < kt1) stage(kt0);
    __syncthreads();
    for (int kt = kt0; kt < kt1; ++kt) {
        if (kt + 1 < kt1) stage(kt + 1);
        const char* xt = smem + (kt & 1) * STAGE + wm * WM * kTileK;
        const char* wt = smem + (kt & 1) * STAGE + (BM + wn * WN) * kTileK;
        float s[FM];
        Widened xf[FM], wf[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) s[i] = g.xs[static_cast<int64_t>(kt) * g.M + row[i]] * wscale[kt];
#pragma unroll
        for (int i = 0; i < FM; ++i) xf[i] = widen({{lds_read16(xt + i * 16 * kTileK + lo0), lds_read16(xt + i * 16 * kTileK + lo1)}});
#pragma unroll
        for (int j = 0; j < FN; ++j) wf[j] = widen({{lds_read16(wt + j * 16 * kTileK + lo0), lds_read16(wt + j * 16 * kTileK + lo1)}});
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) add_scaled(acc[i][j], block_sum(wf[j], xf[i]), s[i]);
        __syncthreads();   // the next K-tile has landed and this one has been read
    }

    // A fragment's results: 4 * (lane >> 4) + register -> column n, lane & 15 -> row m.
    const bool vec = (g.N & 3) == 0;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int n = n0 + wn * WN + j * 16 + (lane >> 4) * 4;
        if (n >= g.N) continue;
        v4f b = {0.f, 0.f, 0.f, 0.f};
        if (g.bias && !g.kt_per_split)
            for (int e = 0; e < 4; ++e)
                if (n + e < g.N) b[e] = g.bias[n + e];
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int64_t m = m0 + wm * WM + i * 16 + (lane & 15);
            if (m < g.M) store4<OUT>(out, m * g.N + n, g.N - n, vec, acc[i][j] + b);
        }
    }
}

// ---- the gated product's second half -------------------------------------------------------------------------------
// h = act(sum of the gate's slabs) * (sum of the up projection's), in blocks: sixteen lanes a block of one row.
__device__ __forceinline__ float gate_value(float g, int act) {
    if (act == MIQ_ACT_SILU) return __fdiv_rn(g, 1.0f + expf(-g));
    return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
}

__global__ __launch_bounds__(256) void gated_join_kernel(const float* __restrict__ slabs, int splits, int64_t M, int N, int nblocks,
                                                         int act, uint8_t* __restrict__ q, float* __restrict__ scale) {
    const int lane = threadIdx.x & 15;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
    const int64_t m = id / nblocks;
    const int b = static_cast<int>(id % nblocks), n = b * 128 + lane * 8;
    const int inside = m < M && n < N ? (N - n < 8 ? N - n : 8) : 0;
    const int64_t size = M * N;
    float h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        h[i] = 0.0f;
        if (i < inside) {
            const int64_t o = m * N + n + i;
            float gate = 0.0f, up = 0.0f;
            for (int s = 0; s < splits; ++s) gate += slabs[s * size + o];
            for (int s = 0; s < splits; ++s) up += slabs[(splits + s) * size + o];
            h[i] = gate_value(gate, act) * up;
        }
    }
    uint32_t c[2];
    const float s = quantize8_in_row(h, c);
    store8_codes<false>(q, m * N + n, inside, c);
    if (lane == 0 && m < M) scale[static_cast<int64_t>(b) * M + m] = s;
}

// Every size that the kernels index with 32 bits, bounded before any arithmetic.
int check_sizes(const char* who, int64_t M, int64_t N, int64_t K) {
    MIQ_REQUIRE(M >= 0 && N >= 0 && K >= 0, MIQ_EINVAL, "%s: negative size (M=%lld N=%lld K=%lld)", who, (long long)M, (long long)N,
                (long long)K);
    MIQ_REQUIRE(M < (1ll << 31) && N < (1ll << 31) - 256 && K < (1ll << 22), MIQ_ERANGE,
                "%s: M and N must be below 2^31, K below 2^22 (M=%lld N=%lld K=%lld)", who, (long long)M, (long long)N, (long long)K);
    const int64_t tiles = ceil_div(M, 64) * ceil_div(N, 64);
    MIQ_REQUIRE(tiles <= (1ll << 22), MIQ_ERANGE, "%s: more than 2^22 tiles of 64 x 64 outputs", who);
    return MIQ_OK;
}

Fp8Args make_args(const uint8_t* x, const float* xs, const uint8_t* w, const float* ws, int64_t M, int64_t N, int64_t K) {
    Fp8Args g{};
    g.x = x;
    g.xs = xs;
    g.w[0] = w;
    g.ws[0] = ws;
    g.M = M;
    g.N = static_cast<int>(N);
    g.K = static_cast<int>(K);
    g.kblocks = static_cast<int>(ceil_div(K, kTileK));
    return g;
}

template <int OUT>
int launch_tiles(Fp8Args g, int products, bool vec, hipStream_t st) {
    constexpr int BM = 64, BN = 64, kLds = 2 * (BM + BN) * kTileK;
    g.tiles_m = static_cast<int>(ceil_div(g.M, BM));
    g.tiles_n = static_cast<int>(ceil_div(g.N, BN));
    const dim3 grid(static_cast<unsigned>(g.tiles_m) * g.tiles_n, 1, products);
    if (vec) gemm_fp8_tile_kernel<BM, BN, 2, 2, OUT, true><<<grid, 256, kLds, st>>>(g);
    else gemm_fp8_tile_kernel<BM, BN, 2, 2, OUT, false><<<grid, 256, kLds, st>>>(g);
    return check_launch("gemm_fp8_tile_kernel");
}

}  // namespace

extern "C" size_t miq_gemm_fp8_workspace(int64_t M, int64_t N, int64_t K) {
    if (check_sizes("miq_gemm_fp8_workspace", M, N, K) != MIQ_OK) return 0;
    return 0;
}

extern "C" int miq_gemm_fp8(const uint8_t* x, const float* x_scale, const uint8_t* w, const float* w_scale, int64_t M, int64_t N,
                            int64_t K, const float* bias, void* out, int out_dtype, void* workspace, size_t workspace_bytes,
                            void* stream) {
    if (int rc = check_sizes("miq_gemm_fp8", M, N, K)) return rc;
    MIQ_REQUIRE(out_dtype == MIQ_F32 || out_dtype == MIQ_F16 || out_dtype == MIQ_BF16, MIQ_EINVAL, "miq_gemm_fp8: unknown out_dtype %d",
                out_dtype);
    if (M == 0 || N == 0) return MIQ_OK;
    MIQ_REQUIRE(out && (K == 0 || (x && x_scale && w && w_scale)), MIQ_EINVAL, "miq_gemm_fp8: null pointer");
    MIQ_REQUIRE(aligned(x_scale, 4) && aligned(w_scale, 4) && aligned(bias, 4) && aligned(out, 16), MIQ_EALIGN,
                "miq_gemm_fp8: scales and bias must be 4-byte, out 16-byte aligned");
    Fp8Args g = make_args(x, x_scale, w, w_scale, M, N, K);
    g.bias = bias;
    g.out = out;
    const bool vec = K % 16 == 0 && aligned(x, 16) && aligned(w, 16);
    if (out_dtype == MIQ_F32) return launch_tiles<MIQ_F32>(g, 1, vec, as_stream(stream));
    if (out_dtype == MIQ_F16) return launch_tiles<MIQ_F16>(g, 1, vec, as_stream(stream));
    return launch_tiles<MIQ_BF16>(g, 1, vec, as_stream(stream));
}

extern "C" size_t miq_gated_fp8_workspace(int64_t M, int64_t N, int64_t K) {
    if (check_sizes("miq_gated_fp8_workspace", M, N, K) != MIQ_OK) return 0;
    return static_cast<size_t>(2 * 4 * M * N);
}

extern "C" int miq_gated_fp8(const uint8_t* x, const float* x_scale, const uint8_t* w_gate, const float* gate_scale,
                             const uint8_t* w_up, const float* up_scale, int64_t M, int64_t N, int64_t K, int act, uint8_t* q,
                             float* scale, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_sizes("miq_gated_fp8", M, N, K)) return rc;
    MIQ_REQUIRE(act == MIQ_ACT_SILU || act == MIQ_ACT_GELU, MIQ_EINVAL, "miq_gated_fp8: unknown activation %d", act);
    if (M == 0 || N == 0) return MIQ_OK;
    MIQ_REQUIRE(q && scale && (K == 0 || (x && x_scale && w_gate && gate_scale && w_up && up_scale)), MIQ_EINVAL,
                "miq_gated_fp8: null pointer");
    MIQ_REQUIRE(aligned(x_scale, 4) && aligned(gate_scale, 4) && aligned(up_scale, 4) && aligned(scale, 4), MIQ_EALIGN,
                "miq_gated_fp8: scales must be 4-byte aligned");
    const size_t need = miq_gated_fp8_workspace(M, N, K);
    MIQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), MIQ_EWORKSPACE, "miq_gated_fp8: %zu bytes of workspace needed, %zu given",
                need, workspace_bytes);
    MIQ_REQUIRE(aligned(workspace, 256), MIQ_EALIGN, "miq_gated_fp8: workspace must be 256-byte aligned");
    Fp8Args g = make_args(x, x_scale, w_gate, gate_scale, M, N, K);
    g.w[1] = w_up;
    g.ws[1] = up_scale;
    g.out = workspace;
    g.kt_per_split = g.kblocks > 0 ? g.kblocks : 1;
    const bool vec = K % 16 == 0 && aligned(x, 16) && aligned(w_gate, 16) && aligned(w_up, 16);
    if (int rc = launch_tiles<MIQ_F32>(g, 2, vec, as_stream(stream))) return rc;
    const int nblocks = static_cast<int>(ceil_div(N, 128));
    MIQ_REQUIRE(ceil_div(M * nblocks, 16) < (1ll << 24), MIQ_ERANGE, "miq_gated_fp8: too many blocks");
    gated_join_kernel<<<static_cast<unsigned>(ceil_div(M * nblocks, 16)), 256, 0, as_stream(stream)>>>(
        static_cast<const float*>(workspace), 1, M, g.N, nblocks, act, q, scale);
    return check_launch("gated_join_kernel");
}
