// Quantizers to block-scaled e4m3 and the root-mean-square norm that ends in one (gfx950; all three HBM-bound).
//
// Sixteen lanes (a DPP row) own a block of 128 columns, eight consecutive columns a lane: the block's maximum is four DPP
// steps away, a 16-bit element row is read with one 16-byte load a lane and its codes leave as 8 bytes a lane, 128 bytes a
// block.  Scales are block-major, [blocks, M]: the product reads one block of many rows at a time.
#include "miq_fp8.h"

namespace {

using namespace miq;

// ---- activations: 1 x 128 ------------------------------------------------------------------------------------------
// A workgroup of 16 sixteen-lane groups takes ROWS rows x (16 / ROWS) * kQuantPasses blocks.  Bound by HBM: 2048x14336 bf16
// 16.0-16.5 us (5.4 TB/s read and written; a copy 4.9), fp32 28.0-28.7 (5.2); few rows by the launch, 2.5 us up to 64x14336.
template <int DT, bool VEC, int ROWS, int kQuantPasses>
__global__ __launch_bounds__(256) void quantize_blocks_kernel(const void* __restrict__ x, int64_t M, int64_t K, int64_t kblocks,
                                                              int64_t col_groups, uint8_t* __restrict__ q,
                                                              float* __restrict__ scale) {
    constexpr int kAcross = 16 / ROWS;   // blocks of one row that a pass covers
    const int grp = threadIdx.x >> 4, lane = threadIdx.x & 15;
    const int64_t m = (blockIdx.x / col_groups) * ROWS + grp / kAcross;
    const int64_t kb0 = (blockIdx.x % col_groups) * (kAcross * kQuantPasses) + grp % kAcross;
    float f[kQuantPasses][8];
    int n[kQuantPasses];
#pragma unroll
    for (int p = 0; p < kQuantPasses; ++p) {
        const int64_t k = (kb0 + p * kAcross) * kBlockK + lane * 8;
        n[p] = m < M && k < K ? static_cast<int>(K - k < 8 ? K - k : 8) : 0;
        load8<DT, VEC>(x, m * K + k, n[p], f[p]);
    }
#pragma unroll
    for (int p = 0; p < kQuantPasses; ++p) {
        const int64_t kb = kb0 + p * kAcross;
        uint32_t c[2];
        const float s = quantize8_in_row(f[p], c);
        store8_codes<VEC>(q, m * K + kb * kBlockK + lane * 8, n[p], c);
        if (lane == 0 && m < M && kb < kblocks) scale[kb * M + m] = s;
    }
}

// ---- weights: 128 x 128 --------------------------------------------------------------------------------------------
// One workgroup a block: a thread holds eight columns of eight rows (64 values) in registers, so that the weight is read once.
// Bound by HBM: 14336x4096 fp32 50 us (5.9 TB/s), bf16 31.3 (5.6).  Rows that start anywhere (14336x4095 fp32) take 86: a block's rows
// begin and end inside cache lines, which the neighbouring block's workgroup, as a rule on another XCD, fetches and writes, too:
// 292 MB read for 235, 73 written for 59, a third of the writes partial lines; 365 MB at 4.2 TB/s.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void quantize_weight_kernel(const void* __restrict__ w, int64_t N, int64_t K, int64_t kblocks,
                                                              uint8_t* __restrict__ q, float* __restrict__ scale) {
    __shared__ uint32_t tops[2][4];
    const int grp = threadIdx.x >> 4, lane = threadIdx.x & 15, wave = threadIdx.x >> 6;
    const int64_t nb = blockIdx.x / kblocks, kb = blockIdx.x % kblocks;
    const int64_t k = kb * kBlockK + lane * 8;
    float f[8][8];
    int n[8];
    uint32_t top = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const int64_t row = nb * 128 + r * 16 + grp;
        n[r] = row < N && k < K ? static_cast<int>(K - k < 8 ? K - k : 8) : 0;
        load8<DT, VEC>(w, row * K + k, n[r], f[r]);
    }
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t b = magnitude_bits(f[r][i]);
            top = b > top ? b : top;
        }
    auto over_workgroup = [&](uint32_t v, int slot) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint32_t other = __shfl_xor(v, o, 64);
            v = other > v ? other : v;
        }
        if ((threadIdx.x & 63) == 0) tops[slot][wave] = v;
        __syncthreads();
        uint32_t t = tops[slot][0];
#pragma unroll
        for (int i = 1; i < 4; ++i) t = tops[slot][i] > t ? tops[slot][i] : t;
        return t;
    };
    top = over_workgroup(top, 0);
    const bool spoiled = top >= kInfBits;   // the same in every thread of the workgroup
    if (spoiled) {
        top = 0;
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = finite_magnitude_bits(f[r][i]);
                top = b > top ? b : top;
            }
        top = over_workgroup(top, 1);
    }
    const BlockScale s = block_scale(top);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        uint32_t c[2];
        codes8(f[r], s.inv, spoiled, c);
        store8_codes<VEC>(q, (nb * 128 + r * 16 + grp) * K + k, n[r], c);
    }
    if (threadIdx.x == 0) scale[nb * kblocks + kb] = s.scale;
}

// ---- root-mean-square norm -----------------------------------------------------------------------------------------
// h = x + residual (rounded to the type it is stored in, so that the norm is the norm of the stored row), y = (h / rms) * g,
// then y in blocks as above.  TPR threads a row; a row of at most TPR * 8 * VPT columns stays in registers between the sum
// of squares and the codes (VPT > 0); a longer one is read twice (VPT = 0).  Bound by HBM: 8192x8192 bf16 with a residual 83.1 us
// (5.7 TB/s), 8192x4096 44.7 (5.3), 1024x40000, read twice, 82.4 (3.5 TB/s of 7 bytes an element); one row 3.7 us, a launch.  Some
// hundred rows are all resident at once: beside the launch their bytes, 777x5000 fp16 6.9 us, 3.6 TB/s of the 3.2 us past one row's.
template <int DT>
__device__ __forceinline__ float round_to(float v) {
    if constexpr (DT == MIQ_BF16) return static_cast<float>(static_cast<__bf16>(v));
    if constexpr (DT == MIQ_F16) return static_cast<float>(static_cast<_Float16>(v));
    return v;
}

template <int DT, bool VEC>
__device__ __forceinline__ void store8(void* base, int64_t index, int n, const float (&f)[8]) {
    if constexpr (DT == MIQ_F32) {
        float* p = static_cast<float*>(base) + index;
        if (n == 8) {
            auto bits = [&](int i) { return __float_as_uint(f[i]); };
            *reinterpret_cast<u32x4_any*>(p) = u32x4{bits(0), bits(1), bits(2), bits(3)};
            *reinterpret_cast<u32x4_any*>(p + 4) = u32x4{bits(4), bits(5), bits(6), bits(7)};
        } else if (!VEC) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) p[i] = f[i];
        }
    } else {
        uint16_t* p = static_cast<uint16_t*>(base) + index;
        uint16_t h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (DT == MIQ_BF16) h[i] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(f[i]));
            else h[i] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(f[i]));
        }
        if (n == 8) {
            u32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = h[2 * i] | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
            // (with a residual 8192x8192 83.1 us, cached 88.4; 2048x28672 89.6 and 92.3, 8192x2048 23.3 and 24.6; but 8192x4096 44.7 and
            // 42.9, 1024x40000 82.4 and 79.4)
            __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(p));
        } else if (!VEC) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) p[i] = h[i];
        }
    }
}

struct NormArgs {
    const void* x;
    const void* residual;   // or null
    const void* g;
    int g_f32;              // g is fp32, else of x's type
    int64_t M, K, kblocks;
    float eps;
    void* sum;              // x + residual, written when there is a residual
    uint8_t* q;
    float* scale;
};

template <int DT, bool VEC, int TPR, int VPT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_norm_kernel(NormArgs a) {
    constexpr int kThreads = TPR < 256 ? 256 : TPR, kRows = kThreads / TPR, kWaves = TPR / 64;
    constexpr int kKeep = VPT > 0 ? VPT : 1;
    __shared__ float part[kWaves];
    __shared__ uint32_t tops[kWaves];
    const int t = threadIdx.x % TPR;
    const int64_t m = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR;
    const bool live = m < a.M;
    const int64_t row = m * a.K;
    const int64_t vecs = (a.kblocks * kBlockK) / 8;            // whole blocks: all 16 lanes of a block take part
    const int64_t rounds = (vecs + TPR - 1) / TPR;
    auto count = [&](int64_t k) { return live && k < a.K ? static_cast<int>(a.K - k < 8 ? a.K - k : 8) : 0; };
    auto load_h = [&](int64_t k, int n, float (&h)[8], bool write) {
        load8<DT, VEC>(a.x, row + k, n, h);
        if (a.residual) {
            float r[8];
            load8<DT, VEC>(a.residual, row + k, n, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = round_to<DT>(__fadd_rn(h[i], r[i]));
            if (write) store8<DT, VEC>(a.sum, row + k, n, h);
        }
    };
    float ss = 0.0f;
    auto add_squares = [&](const float (&v)[8]) {
        float s8 = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s8 = __fadd_rn(s8, __fmul_rn(v[i], v[i]));
        ss += s8;
    };
    auto over_row = [&](auto v, auto* of_wave, auto join) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v = join(v, __shfl_xor(v, o, 64));
        if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = v;
        __syncthreads();
        v = of_wave[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) v = join(v, of_wave[i]);
        return v;
    };
    auto plus = [](float a, float b) { return a + b; };
    auto inverse_rms = [&](float eps) {
        return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(a.K)), eps)));
    };
    auto finish = [&](int64_t k, int n, float (&hv)[8], float inv_rms) {
        float g[8];
        if (DT == MIQ_F32 || a.g_f32) load8<MIQ_F32, VEC, false>(a.g, k, k < a.K ? (a.K - k < 8 ? a.K - k : 8) : 0, g);
        else load8<DT, VEC, false>(a.g, k, k < a.K ? (a.K - k < 8 ? a.K - k : 8) : 0, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) hv[i] = __fmul_rn(__fmul_rn(hv[i], inv_rms), g[i]);
        uint32_t c[2];
        const float s = quantize8_in_row(hv, c);
        store8_codes<VEC>(a.q, row + k, n, c);
        if ((threadIdx.x & 15) == 0 && n > 0) a.scale[(k / kBlockK) * a.M + m] = s;
    };
    // The vectors of the row times 2^-shift, read one by one.
    auto each_vector = [&](int shift, bool write, auto use) {
        for (int64_t v = 0; v < rounds; ++v) {
            const int64_t k = (v * TPR + t) * 8;
            float h[8];
            load_h(k, count(k), h, write);
            if (shift) {
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] = ldexpf(h[i], -shift);
            }
            use(k, h);
        }
    };
    float h[kKeep][8];
    if constexpr (VPT > 0) {
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int64_t k = (static_cast<int64_t>(v) * TPR + t) * 8;
            load_h(k, count(k), h[v], true);
        }
#pragma unroll
        for (int v = 0; v < VPT; ++v) add_squares(h[v]);
    } else {
        each_vector(0, true, [&](int64_t, float (&hv)[8]) { add_squares(hv); });
    }
    ss = over_row(ss, part, plus);
    // The sum of squares of a finite row can pass fp32's range (bf16 and fp32 rows from some 1e18 on), or lie where squares lose
    // bits and eps does not cover them.  Such a row (the same finding in every thread) is read again and taken times the power of
    // two that puts its largest value between 1 and 2, which is exact; 2^120 at most, so that eps times its square is finite.
    if (!(ss < __builtin_inff()) || (ss < 0x1p-90f && a.eps < 0x1p-120f)) {
        uint32_t top = 0;
        each_vector(0, false, [&](int64_t, float (&hv)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = magnitude_bits(hv[i]);
                top = b > top ? b : top;
            }
        });
        top = over_row(top, tops, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
        const int exponent = static_cast<int>(top >> 23) - 127;
        // (an infinity or a NaN: as they are)
        const int shift = top == 0 || top >= kInfBits ? 0 : exponent > -120 ? exponent : -120;
        if (shift) {
            ss = 0.0f;
            each_vector(shift, false, [&](int64_t, float (&hv)[8]) { add_squares(hv); });
            ss = over_row(ss, part, plus);
        }
        // (a row of zeros without eps has no norm: its codes are 0)
        const float inv_rms = top == 0 && a.eps == 0.0f ? 1.0f : inverse_rms(ldexpf(a.eps, -2 * shift));
        each_vector(shift, false, [&](int64_t k, float (&hv)[8]) { finish(k, count(k), hv, inv_rms); });
        return;
    }
    const float inv_rms = inverse_rms(a.eps);
    if constexpr (VPT > 0) {
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int64_t k = (static_cast<int64_t>(v) * TPR + t) * 8;
            finish(k, count(k), h[v], inv_rms);
        }
    } else {
        each_vector(0, false, [&](int64_t k, float (&hv)[8]) { finish(k, count(k), hv, inv_rms); });
    }
}

bool float_code(int dt) { return dt == MIQ_F32 || dt == MIQ_F16 || dt == MIQ_BF16; }
int elem_size(int dt) { return dt == MIQ_F32 ? 4 : 2; }

template <typename F>
int for_dtype(int dt, F&& f) {
    if (dt == MIQ_F32) return f(std::integral_constant<int, MIQ_F32>{});
    if (dt == MIQ_F16) return f(std::integral_constant<int, MIQ_F16>{});
    return f(std::integral_constant<int, MIQ_BF16>{});
}

constexpr int64_t kMaxGrid = (1ll << 24) - 1;   // 256 threads each: a launch holds less than 2^32 threads

}  // namespace

extern "C" int miq_quantize_blocks_fp8(const void* x, int x_dtype, int64_t M, int64_t K, uint8_t* q, float* scale,
                                       void* stream) {
    MIQ_REQUIRE(M >= 0 && K >= 0, MIQ_EINVAL, "miq_quantize_blocks_fp8: negative size (M=%lld K=%lld)", (long long)M, (long long)K);
    MIQ_REQUIRE(float_code(x_dtype), MIQ_EINVAL, "miq_quantize_blocks_fp8: unknown x_dtype %d", x_dtype);
    if (M == 0 || K == 0) return MIQ_OK;
    MIQ_REQUIRE(all_below_2_31({M, K}), MIQ_ERANGE, "miq_quantize_blocks_fp8: a dimension at or beyond 2^31");
    MIQ_REQUIRE(x && q && scale, MIQ_EINVAL, "miq_quantize_blocks_fp8: null pointer");
    MIQ_REQUIRE(aligned(x, elem_size(x_dtype)) && aligned(scale, 4), MIQ_EALIGN, "miq_quantize_blocks_fp8: misaligned pointer");
    const bool vec = K % 8 == 0 && aligned(x, 16) && aligned(q, 8);
    const int64_t kblocks = ceil_div(K, kBlockK);
    // Sixteen rows of a block at a time where there are as many, so that their scales leave as one line (2048x14336 bf16 16.5 us,
    // rows one by one 18.2; fewer rows are a launch either way); four blocks a thread in flight (16.4 us; one: 17.3), or one
    // where four would leave CUs idle (64x4096 2.5 us, four 3.3; 256x4096 2.7 and 3.7; 512x14336 5.9 both).
    const bool tall = M >= 16, few = ceil_div(M, tall ? 16 : 1) * ceil_div(kblocks, tall ? 4 : 64) < 256;
    const int64_t col_groups = ceil_div(kblocks, (tall ? 1 : 16) * (few ? 1 : 4));
    const int64_t grid = (tall ? ceil_div(M, 16) : M) * col_groups;
    MIQ_REQUIRE(grid <= kMaxGrid, MIQ_ERANGE, "miq_quantize_blocks_fp8: too many blocks");
    return for_dtype(x_dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        auto go = [&](auto v, auto rows, auto passes) {
            quantize_blocks_kernel<DT, decltype(v)::value, decltype(rows)::value, decltype(passes)::value>
                <<<static_cast<unsigned>(grid), 256, 0, as_stream(stream)>>>(x, M, K, kblocks, col_groups, q, scale);
        };
        auto shape = [&](auto v) {
            std::integral_constant<int, 16> r16;
            std::integral_constant<int, 1> one;
            std::integral_constant<int, 4> four;
            if (tall) few ? go(v, r16, one) : go(v, r16, four);
            else few ? go(v, one, one) : go(v, one, four);
        };
        if (vec) shape(std::true_type{});
        else shape(std::false_type{});
        return check_launch("quantize_blocks_kernel");
    });
}

extern "C" int miq_quantize_weight_fp8(const void* w, int w_dtype, int64_t N, int64_t K, uint8_t* q, float* scale,
                                       void* stream) {
    MIQ_REQUIRE(N >= 0 && K >= 0, MIQ_EINVAL, "miq_quantize_weight_fp8: negative size (N=%lld K=%lld)", (long long)N, (long long)K);
    MIQ_REQUIRE(float_code(w_dtype), MIQ_EINVAL, "miq_quantize_weight_fp8: unknown w_dtype %d", w_dtype);
    if (N == 0 || K == 0) return MIQ_OK;
    MIQ_REQUIRE(all_below_2_31({N, K}), MIQ_ERANGE, "miq_quantize_weight_fp8: a dimension at or beyond 2^31");
    MIQ_REQUIRE(w && q && scale, MIQ_EINVAL, "miq_quantize_weight_fp8: null pointer");
    MIQ_REQUIRE(aligned(w, elem_size(w_dtype)) && aligned(scale, 4), MIQ_EALIGN, "miq_quantize_weight_fp8: misaligned pointer");
    const bool vec = K % 8 == 0 && aligned(w, 16) && aligned(q, 8);
    const int64_t kblocks = ceil_div(K, kBlockK), grid = ceil_div(N, 128) * kblocks;
    MIQ_REQUIRE(grid <= kMaxGrid, MIQ_ERANGE, "miq_quantize_weight_fp8: too many blocks");
    return for_dtype(w_dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (vec) quantize_weight_kernel<DT, true><<<static_cast<unsigned>(grid), 256, 0, as_stream(stream)>>>(w, N, K, kblocks, q, scale);
        else quantize_weight_kernel<DT, false><<<static_cast<unsigned>(grid), 256, 0, as_stream(stream)>>>(w, N, K, kblocks, q, scale);
        return check_launch("quantize_weight_kernel");
    });
}

extern "C" int miq_rms_norm_fp8(const void* x, const void* residual, const void* weight, int dtype, int weight_dtype, int64_t M,
                                int64_t K, float eps, void* sum, uint8_t* q, float* scale, void* stream) {
    MIQ_REQUIRE(M >= 0 && K >= 0, MIQ_EINVAL, "miq_rms_norm_fp8: negative size (M=%lld K=%lld)", (long long)M, (long long)K);
    MIQ_REQUIRE(float_code(dtype), MIQ_EINVAL, "miq_rms_norm_fp8: unknown dtype %d", dtype);
    MIQ_REQUIRE(weight_dtype == dtype || weight_dtype == MIQ_F32, MIQ_EINVAL,
                "miq_rms_norm_fp8: weight_dtype must be dtype or MIQ_F32 (got %d)", weight_dtype);
    MIQ_REQUIRE(eps >= 0.0f && eps < __builtin_inff(), MIQ_EINVAL, "miq_rms_norm_fp8: eps must be finite and not negative");
    if (M == 0 || K == 0) return MIQ_OK;
    MIQ_REQUIRE(all_below_2_31({M, K}), MIQ_ERANGE, "miq_rms_norm_fp8: a dimension at or beyond 2^31");
    MIQ_REQUIRE(x && weight && q && scale, MIQ_EINVAL, "miq_rms_norm_fp8: null pointer");
    MIQ_REQUIRE((residual == nullptr) == (sum == nullptr), MIQ_EINVAL, "miq_rms_norm_fp8: residual and sum come together");
    const int es = elem_size(dtype);
    MIQ_REQUIRE(aligned(x, es) && aligned(residual, es) && aligned(sum, es) && aligned(weight, elem_size(weight_dtype)) && aligned(scale, 4),
                MIQ_EALIGN, "miq_rms_norm_fp8: misaligned pointer");
    const bool vec = K % 8 == 0 && aligned(x, 16) && aligned(residual, 16) && aligned(sum, 16) && aligned(weight, 16) && aligned(q, 8);
    NormArgs a{x, residual, weight, weight_dtype == MIQ_F32, M, K, ceil_div(K, kBlockK), eps, sum, q, scale};
    const int64_t cols = a.kblocks * kBlockK;
    MIQ_REQUIRE(M * (cols <= 256 * 16 ? 256 : cols <= 512 * 16 ? 512 : 1024) < (1ll << 32), MIQ_ERANGE, "miq_rms_norm_fp8: too many rows");
    return for_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        auto go = [&](auto v) {
            constexpr bool V = decltype(v)::value;
            const unsigned grid = static_cast<unsigned>(M);
            // Two vectors a thread where a row has as many threads (8192 x 8192 bf16 with a residual: 83 us as 512 threads of
            // two, 90 as 256 of four, 109 as 1024 of one; 8192x4096 44 as 256 of two, 49 as 512; 8192x2048 23.6 as 256 of one,
            // 36 as 512); four keep rows of up to 32768 columns in registers (2048x28672 90 us, read twice 116).
            if (cols <= 256 * 8) rms_norm_kernel<DT, V, 256, 1><<<grid, 256, 0, as_stream(stream)>>>(a);
            else if (cols <= 256 * 16) rms_norm_kernel<DT, V, 256, 2><<<grid, 256, 0, as_stream(stream)>>>(a);
            else if (cols <= 512 * 16) rms_norm_kernel<DT, V, 512, 2><<<grid, 512, 0, as_stream(stream)>>>(a);
            else if (cols <= 1024 * 16) rms_norm_kernel<DT, V, 1024, 2><<<grid, 1024, 0, as_stream(stream)>>>(a);
            else if (cols <= 1024 * 32) rms_norm_kernel<DT, V, 1024, 4><<<grid, 1024, 0, as_stream(stream)>>>(a);
            else rms_norm_kernel<DT, V, 1024, 0><<<grid, 1024, 0, as_stream(stream)>>>(a);
        };
        if (vec) go(std::true_type{});
        else go(std::false_type{});
        return check_launch("rms_norm_kernel");
    });
}
