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
// of it (measured: 2^16 + 2^3 comes out right, 2^16 + 2^2 as 2^16; across groups of eight it keeps 24 bits).  On layers'
// operands that is 3e-5 of the outputs' root mean square, a hundred times an fp32 sum's error.  v_mfma_f32_16x16x32_bf16 keeps 24
// bits throughout (1e-8 on the same operands), and e4m3 widens to bf16 exactly (v_cvt_scalef32_pk_bf16_fp8, two codes an
// instruction), at half the rate.  So 16-bit outputs, whose own rounding is coarser (bf16 1.7e-3, 57 times as coarse; fp16 2.1e-4,
// seven times), take the 8-bit instruction; fp32 outputs, the gated product (its scales are fp32) and products of at most 16 rows
// (which the weight's stream bounds in either form) widen.
//
// What a block's scale costs: an accumulator is written by the vector unit once a K-tile, one fused multiply-add an output,
// beside the matrix instructions; a product with one scale for a whole tensor has none of that.  The 16 x 16 instructions
// leave it room: a SIMD issues two vector instructions in the time of one 16x16x32 bf16 instruction without slowing it.
#include <cmath>

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
    int N, K, kblocks;     // K: bytes between two rows of x and w, a multiple of 16
    int tiles_m, tiles_n;
    int kt_per_split;      // K-tiles each blockIdx.y slice sums; 0 = all, straight to `out`
    int pitch;             // floats between two rows of a slab: N rounded up to 8 (columns past N hold 0, or NaN in a row with a NaN code)
};

// A fragment of 16 rows and one K-tile: the lane's 16-byte chunks (lane >> 4) and 4 + (lane >> 4) of row lane & 15.
struct Codes {
    v4i c[2];
};
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
// The same fragment widened to bf16: h[i] is the operand of the i-th of a block's four matrix instructions.
struct Widened {
    v4i h[4];
};
// Dword `pos` (0 .. 15) of a widened fragment: two codes.
__device__ __forceinline__ void widen1(Widened& w, const Codes& f, int pos) {
    const int src = f.c[pos >> 3][(pos & 7) >> 1];
    w.h[pos >> 2][pos & 3] = (pos & 1) ? __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, 1.0f, true))
                                       : __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(src, 1.0f, false));
}
__device__ __forceinline__ Widened widen(const Codes& f) {
    Widened r;
#pragma unroll
    for (int i = 0; i < 16; ++i) widen1(r, f, i);
    return r;
}
__device__ __forceinline__ v4f mfma_bf16(v4i w, v4i x, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, x), c, 0, 0, 0);
}
// The products of one block, summed from zero.
__device__ __forceinline__ v4f block_sum(const Widened& w, const Widened& x) {
    v4f c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) c = mfma_bf16(w.h[i], x.h[i], c);
    return c;
}

// The operand of a fragment: the codes themselves for the 8-bit instruction (NATIVE), else widened.
template <bool NATIVE>
struct OperandOf;
template <>
struct OperandOf<true> {
    using Frag = Codes;
};
template <>
struct OperandOf<false> {
    using Frag = Widened;
};

constexpr int kNoAct = -1;   // (an epilogue without a gate)

typedef int v8i __attribute__((ext_vector_type(8)));
__device__ __forceinline__ v4f block_sum(const Codes& w, const Codes& x) {
    const v8i a = __builtin_shufflevector(w.c[0], w.c[1], 0, 1, 2, 3, 4, 5, 6, 7);
    const v8i b = __builtin_shufflevector(x.c[0], x.c[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
template <bool NATIVE>
__device__ __forceinline__ auto operand(const Codes& c) {
    if constexpr (NATIVE) return c;
    else return widen(c);
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

// Four outputs of a 16-bit type.
template <int OUT>
__device__ __forceinline__ uint2 pack4(v4f v) {
    if constexpr (OUT == MIQ_F16) {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(uint2, h4{static_cast<_Float16>(v[0]), static_cast<_Float16>(v[1]), static_cast<_Float16>(v[2]),
                                            static_cast<_Float16>(v[3])});
    } else {
        return pack4_bf16(v[0], v[1], v[2], v[3]);
    }
}

// Four consecutive outputs of one row, `n` of them inside it.  `vec`: their address is aligned to four elements.
template <int OUT>
__device__ __forceinline__ void store4(void* out, int64_t i, int n, bool vec, v4f v) {
    if (vec && n >= 4) {
        if constexpr (OUT == MIQ_F32) {
            *reinterpret_cast<v4f*>(static_cast<float*>(out) + i) = v;
        } else {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i) = pack4<OUT>(v);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) store_value<OUT>(out, i + e, v[e]);
    }
}

// Memory requests before this stay before it, those after it after: the counted waits below depend on the order of issue.
__device__ __forceinline__ void keep_order() { asm volatile("" ::: "memory"); }

// v without its first `drop` bytes, zeros behind them.
__device__ __forceinline__ v4i drop_front(v4i v, int drop) {
    typedef unsigned __int128 u128;
    return drop < 16 ? __builtin_bit_cast(v4i, __builtin_bit_cast(u128, v) >> (8 * drop)) : v4i{0, 0, 0, 0};
}

// Rows of K bytes -> rows of `pitch` bytes (K rounded up to 16), zeros past K, up to three matrices in one launch.  A wave takes a
// row, a lane a 16-byte piece: five whole dwords shifted together, where these lie inside the row; the pieces at its end are the
// row's last sixteen bytes, shifted down.  (2000 + 2000 rows of 1001 bytes 5.6 us, one thread a piece of any row, loaded at any
// address, 8.2; 14336 rows of 4095 19.7 and 26.4 us, 5.9 TB/s read and written.)
struct PadArgs {
    const uint8_t* src[3];   // 4-byte aligned
    uint8_t* dst[3];
    int64_t rows[3];   // 0: none
    int K, pitch;
};
__global__ __launch_bounds__(256) void pad_rows_kernel(PadArgs a) {
    const int lane = threadIdx.x & 63, o = blockIdx.y;
    for (int64_t r = blockIdx.x * 4ll + (threadIdx.x >> 6); r < a.rows[o]; r += gridDim.x * 4ll) {
        const uint8_t* const row = a.src[o] + r * a.K;
        const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row)) & 3;
        v4i* const to = reinterpret_cast<v4i*>(a.dst[o] + r * a.pitch);
#pragma unroll 4
        for (int k = lane * kChunk; k < a.K; k += 64 * kChunk) {
            v4i v = {0, 0, 0, 0};
            if (k + kChunk + 4 <= a.K) {
                const uint8_t* const p = row - shift + k;
                const u32x4 d = load16<false>(p);
                const uint32_t e = *reinterpret_cast<const uint32_t*>(p + kChunk);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[i] = static_cast<int>(__builtin_amdgcn_alignbyte(i < 3 ? d[i < 3 ? i + 1 : 3] : e, d[i], shift));
            } else if (a.K >= kChunk) {
                const int last = k < a.K - kChunk ? k : a.K - kChunk;
                v = drop_front(__builtin_bit_cast(v4i, load16<false>(row + last)), k - last);
            } else {
                for (int b = 0; b < a.K; ++b) v[b >> 2] |= static_cast<int>(static_cast<uint32_t>(row[b]) << (8 * (b & 3)));
            }
            to[k / kChunk] = v;
        }
    }
}

// The gate's activation.  The logistic function is the hardware's power of two and reciprocal (one unit each): the rounded
// argument costs an exponential of a large gate |g| / 2 units, so that the activation is within |g| / 2 + 5 units of its own size
// (40 at g = -70, under 1e-5 of it, beside an e4m3 code's half step of 6e-2).  (With the library's exponential and an IEEE
// division the epilogue of a 256 x 128 tile took 11 us of vector instructions, a tenth of a K of 4096.)
// GELU's 1 + erf(g / sqrt 2) is erfc(-g / sqrt 2): of a negative gate the sum would leave what rounding leaves of 1 - 1 (4% off at
// g = -5, nothing at -5.5), and a block of negative gates takes its scale and every code from it.  (4096x14336x4096 861 us, with the
// error function 840; one token 29.3 both.)
template <int ACT>
__device__ __forceinline__ float gate_value(float g) {
    if constexpr (ACT == MIQ_ACT_SILU) return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504f));
    return 0.5f * g * erfcf(g * -0.70710678118654752f);
}

// What a wave's lanes wrote to LDS before this they may read after it (a wave's LDS operations are done in order).
__device__ __forceinline__ void wave_lds_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

// ---- small tiles: products that do not fill the chip with 256 x 256 ones --------------------------------------------
// BM x BN outputs a workgroup.  STAGES == 2: two K-tile buffers and one barrier a K-tile, for tiles whose matrix work covers
// a fetch; STAGES > 2: a ring with STAGES - 1 K-tiles in flight and a counted wait, for the thin ones (a few rows against a
// weight that streams from HBM), whose K-tile of matrix work is far shorter than a fetch.  Split-K: slice blockIdx.y sums its
// K-tiles into an fp32 slab of its own; blockIdx.z picks the weight of a gated product.
//
// Bound by the weight's stream where there are few rows (77x14336x4096 bf16: 16.5 us, 3.7 TB/s of weight; 24x14336x4096 gated:
// 28 us with the join, 4.2 TB/s), by its LDS reads and vector work above: a 64 x 64 tile reads 3 bytes of LDS for each byte it
// fetches (1024x4096x4096 bf16 1.0 PFLOP/s with 64-row tiles, 1.2 with 128-row ones; fp32 427x5073x3712 30 us, 0.54).
constexpr int tile_stage_bytes(int bm, int bn, int waves) { return (bm + bn) * kTileK + waves * ((bm + 63) / 64) * 256; }

template <int BM, int BN, int WAVES_M, int WAVES_N, int STAGES, int OUT, bool NATIVE>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 2) void gemm_fp8_tile_kernel(Fp8Args g) {   // (2: at most 256 registers, and
    // no matrix results in accumulation registers, which the vector unit would have to fetch from there one by one)
    constexpr int NWAVES = WAVES_M * WAVES_N;
    constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, FM = WM / 16, FN = WN / 16;
    constexpr int kRowBytes = (BM + BN) * kTileK, kScaleLoads = (BM + 63) / 64;
    constexpr int STAGE = tile_stage_bytes(BM, BN, NWAVES);
    static_assert(128 % BN == 0, "a tile's columns lie in one 128-row block of the weight");
    static_assert((BM / 8) % NWAVES == 0 && (BN / 8) % NWAVES == 0, "every wave issues the same number of pieces");
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
    // Staging: a wave-instruction moves 8 rows x 128 B; wave v moves rows v * 8 + 8 NWAVES i.  Rows past the matrix lie past the
    // descriptor's end and read as zeros.
    const int srow = wave * 8 + (lane >> 3), cbyte = ((lane & 7) ^ ((srow >> 1) & 7)) * kChunk;
    const uint32_t off0 = static_cast<uint32_t>(srow) * static_cast<uint32_t>(g.K) + cbyte;
    const uint32_t piece_rows = 8u * NWAVES * static_cast<uint32_t>(g.K);
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(g.x + m0 * g.K, static_cast<uint32_t>(mrows) * static_cast<uint32_t>(g.K));
    const __amdgpu_buffer_rsrc_t rw =
        make_rsrc(g.w[which] + static_cast<int64_t>(n0) * g.K, static_cast<uint32_t>(nrows) * static_cast<uint32_t>(g.K));
    using scalar_floats = const __attribute__((address_space(4))) float*;   // (read through the scalar unit)
    const scalar_floats wscale = (scalar_floats)(g.ws[which] + static_cast<int64_t>(n0 / 128) * g.kblocks);

    const int kt0 = g.kt_per_split ? static_cast<int>(blockIdx.y) * g.kt_per_split : 0;
    const int kt1 = g.kt_per_split && kt0 + g.kt_per_split < g.kblocks ? kt0 + g.kt_per_split : g.kblocks;
    void* out = g.out;
    if constexpr (OUT == MIQ_F32) {
        if (g.kt_per_split) out = static_cast<float*>(out) + (static_cast<int64_t>(which) * gridDim.y + blockIdx.y) * g.M * g.pitch;
    }

    v4f acc[FM][FN] = {};
    const int lo0 = frag_lane_offset(lane, 0), lo1 = frag_lane_offset(lane, 1);
    // A stage of LDS: BM + BN rows of a K-tile, and for each wave a copy of the rows' scales (fetched by LDS-DMA like the rows:
    // a scale loaded into a register would be waited for together with the younger rows' requests).
    const float* xs_at = g.xs + static_cast<int64_t>(kt0) * g.M + m0;   // of the K-tile that stage() is called for next
    auto stage = [&](char* buf, int kt) {   // (a K-tile past the slice is requested out of range: zeros, no memory traffic)
        const int k = (kt < kt1 ? kt : g.kblocks) * kTileK;
        const uint32_t off = k + cbyte < g.K ? off0 + k : kOob;
        char* const to = buf + wave * (8 * kTileK);
#pragma unroll
        for (int i = 0; i < BM / 8 / NWAVES; ++i) dma16(rx, to + i * (8 * NWAVES * kTileK), off + i * piece_rows);
#pragma unroll
        for (int i = 0; i < BN / 8 / NWAVES; ++i) dma16(rw, to + BM * kTileK + i * (8 * NWAVES * kTileK), off + i * piece_rows);
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(xs_at, kt < kt1 ? static_cast<uint32_t>(mrows) * 4 : 0);
        xs_at += g.M;
#pragma unroll
        for (int i = 0; i < kScaleLoads; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(buf + kRowBytes + (wave * kScaleLoads + i) * 256), 4,
                                                     static_cast<uint32_t>(i * 64 + lane) * 4, 0, 0, 0);
    };
    auto multiply = [&](const char* buf, int kt) {
        const float* xs = reinterpret_cast<const float*>(buf + kRowBytes + wave * kScaleLoads * 256) + wm * WM + (lane & 15);
        const char* xt = buf + wm * WM * kTileK;
        const char* wt = buf + (BM + wn * WN) * kTileK;
        const float sw = wscale[kt];
        typename OperandOf<NATIVE>::Frag wf[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j)
            wf[j] = operand<NATIVE>({{lds_read16(wt + j * 16 * kTileK + lo0), lds_read16(wt + j * 16 * kTileK + lo1)}});
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const auto xf = operand<NATIVE>(Codes{{lds_read16(xt + i * 16 * kTileK + lo0), lds_read16(xt + i * 16 * kTileK + lo1)}});
            const float s = xs[i * 16] * sw;
#pragma unroll
            for (int j = 0; j < FN; ++j) add_scaled(acc[i][j], block_sum(wf[j], xf), s);
        }
    };

    if (kt0 < kt1) {
        if constexpr (STAGES == 2) {
            stage(smem, kt0);
            __syncthreads();
            for (int kt = kt0; kt < kt1; ++kt) {
                if (kt + 1 < kt1) stage(smem + ((kt + 1 - kt0) & 1) * STAGE, kt + 1);
                multiply(smem + ((kt - kt0) & 1) * STAGE, kt);
                __syncthreads();   // the next K-tile has landed and this one has been read
            }
        } else {
            // All but the youngest STAGES - 2 K-tiles have landed when at most that many K-tiles' requests are outstanding.
            constexpr int kKeep = ((BM / 8 + BN / 8) / NWAVES + kScaleLoads) * (STAGES - 2);
            static_assert(kKeep <= 63, "vmcnt is a 6-bit counter");
#pragma unroll
            for (int t = 0; t < STAGES - 1; ++t) {
                stage(smem + t * STAGE, kt0 + t);
                keep_order();
            }
            int slot = 0, fill = (STAGES - 1) * STAGE;
            for (int kt = kt0; kt < kt1; ++kt) {
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kKeep) : "memory");
                __builtin_amdgcn_s_barrier();   // K-tile kt is there for every wave; every wave has read kt - 1
                keep_order();
                stage(smem + fill, kt + STAGES - 1);
                multiply(smem + slot, kt);
                fill = slot;   // (the slot that was just read takes the K-tile STAGES - 1 on)
                slot = slot == (STAGES - 1) * STAGE ? 0 : slot + STAGE;
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
    }

    // A fragment's results: 4 * (lane >> 4) + register -> column n, lane & 15 -> row m.
    const int cols = g.kt_per_split ? g.pitch : g.N;   // of a row of `out`
    v4f b[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int n = n0 + wn * WN + j * 16 + (lane >> 4) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) b[j][e] = g.bias && !g.kt_per_split && n + e < g.N ? g.bias[n + e] : 0.f;
    }
    if ((cols & 3) == 0) {
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int n = n0 + wn * WN + j * 16 + (lane >> 4) * 4;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int64_t m = m0 + wm * WM + i * 16 + (lane & 15);
                if (n < cols && m < g.M) store4<OUT>(out, m * cols + n, cols - n, true, acc[i][j] + b[j]);
            }
        }
    } else {
        // Rows that start anywhere: a row fragment's 16 x WN through LDS, then 64 / WN rows an instruction, a column a lane (an
        // element at a time from where the results lie, 1 to 2 TB/s: 2312x2166x128 bf16 15.8 us, this way 9.1).
        constexpr int kPitch = WN + 4;
        static_assert(NWAVES * 16 * kPitch * 4 <= STAGES * STAGE, "fits the ring");
        __syncthreads();   // every wave has read its last K-tile
        float* const rows = reinterpret_cast<float*>(smem) + wave * (16 * kPitch);
        const int n = n0 + wn * WN + lane % WN;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int j = 0; j < FN; ++j) *reinterpret_cast<v4f*>(rows + (lane & 15) * kPitch + j * 16 + (lane >> 4) * 4) = acc[i][j] + b[j];
            wave_lds_order();
            const int64_t m = m0 + wm * WM + i * 16 + lane / WN;
            constexpr int kStep = 64 / WN;
            float v[16 / kStep];
#pragma unroll
            for (int r = 0; r < 16; r += kStep) v[r / kStep] = rows[(r + lane / WN) * kPitch + lane % WN];
            wave_lds_order();
#pragma unroll
            for (int r = 0; r < 16; r += kStep)
                if (n < cols && m + r < g.M) store_value<OUT>(out, (m + r) * cols + n, v[r / kStep]);
        }
    }
}

// ---- at most 16 rows: the weight streams once, HBM -> registers ------------------------------------------------------
// A row group of 16 weight rows is one operand fragment, and nothing is shared between waves, so nothing is staged: a lane
// loads the chunks that the instructions want from it.  A workgroup of kWaves waves owns GROUPS row groups; wave v sums
// the K-tiles v, v + kWaves, ... (eight consecutive K-tiles are 1 KiB of a row), DEPTH of them in flight, and the partial
// sums meet in LDS.  A gated product's groups are the gate's and the up projection's of the same columns: the workgroup
// finishes act(g) * u in fp32, and the quantizer follows (a workgroup that has a whole block's 128 columns could quantize it
// itself, but streams them alone: 1x4096x1024 12.6 us for 6.1, 1x14336x4096 44 for 30).  Bound by the weight's stream: 1x4096x14336 11.3 us (5.2 TB/s),
// 1x28672x8192 44 us (5.3), the two weights of 1x14336x4096 26 us (4.5); K that is no multiple of 128, so that a row's K-tile
// is two half lines, 3.3 (9x17784x10032 54 us).
//
// ANY: rows of any length from 16 bytes on, read where they lie: five whole dwords around a chunk, shifted together (sixteen
// bytes at any address are one load, too, but a slow one: 1x4096x14335 30 us).  A row's last chunk is the sixteen bytes that end
// it, shifted down, and what would lie behind them are zeros.  (1x4096x14335 16.6 us, through padded copies 33.5; rows of whole
// vectors, 1x4096x14336, 11.8.)
template <int GROUPS, int kWaves, int DEPTH, int OUT, int ACT, bool ANY>
__global__ __launch_bounds__(64 * kWaves) void gemm_fp8_rows16_kernel(Fp8Args g) {
    constexpr bool GATED = ACT != kNoAct;
    static_assert(!GATED || GROUPS % 2 == 0, "as many of the gate's groups as of the up projection's");
    constexpr int kEach = GATED ? GROUPS / 2 : GROUPS, kCols = kEach * 16;   // groups of one weight
    __shared__ float part[kWaves * GROUPS * 256];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * kCols;
    const int nrows = g.N - n0 < kCols ? g.N - n0 : kCols;
    const int kt0 = g.kt_per_split ? static_cast<int>(blockIdx.y) * g.kt_per_split : 0;
    const int kt1 = g.kt_per_split && kt0 + g.kt_per_split < g.kblocks ? kt0 + g.kt_per_split : g.kblocks;

    // Rows past the matrices lie past the descriptors' ends and read as zeros.
    const int cb = (lane >> 4) * kChunk;
    const uint32_t row = static_cast<uint32_t>(lane & 15) * static_cast<uint32_t>(g.K) + cb;
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(g.x, static_cast<uint32_t>(g.M) * static_cast<uint32_t>(g.K));
    __amdgpu_buffer_rsrc_t rw[GROUPS];
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
        const int first = j % kEach * 16, left = nrows - first;
        rw[j] = make_rsrc(g.w[j / kEach] + static_cast<int64_t>(n0 + first) * g.K,
                          left > 0 ? static_cast<uint32_t>(left) * static_cast<uint32_t>(g.K) : 0);
    }
    // ANY: the lane's rows themselves (past the matrices the last one; what they give is not stored)
    struct Row {
        const uint8_t* base;   // from a whole dword on
        uint32_t shift;        // bytes from there to the row
    };
    Row rows[ANY ? GROUPS + 1 : 1] = {};   // of the weights, and of x
    if constexpr (ANY) {
        const int mine = lane & 15;
        auto row_at = [](const uint8_t* p) {
            const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 3;
            return Row{p - shift, shift};
        };
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) {
            const int n = n0 + j % kEach * 16 + mine;
            rows[j] = row_at(g.w[j / kEach] + static_cast<int64_t>(n < g.N ? n : g.N - 1) * g.K);
        }
        rows[GROUPS] = row_at(g.x + static_cast<int64_t>(mine < g.M ? mine : g.M - 1) * g.K);
    }
    // The dwords of K-tile kt and the one behind them lie inside every row (the last row may end the tensor).
    auto inside = [&](int kt) { return (kt + 1) * kTileK + 4 <= g.K; };
    using scalar_floats = const __attribute__((address_space(4))) float*;
    scalar_floats wscale[GATED ? 2 : 1];
#pragma unroll
    for (int j = 0; j < (GATED ? 2 : 1); ++j) wscale[j] = (scalar_floats)(g.ws[j] + static_cast<int64_t>(n0 / 128) * g.kblocks);

    struct Slot {
        Codes w[GROUPS], x;
        float s;   // the scale of row lane & 15
        uint32_t more[ANY ? GROUPS + 1 : 1][2];   // the dword behind a chunk's four
    };
    auto fill = [&](Slot& s, int kt) {
        const bool in = kt < kt1;
        if constexpr (ANY) {
            const int at = in ? kt : kt0;   // (a K-tile past the slice is dropped as a whole)
            const bool whole = inside(at);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = at * kTileK + h * 64 + cb, last = k < g.K - kChunk ? k : g.K - kChunk;
#pragma unroll
                for (int j = 0; j <= GROUPS; ++j) {
                    const uint8_t* p = rows[j].base;
                    (j < GROUPS ? s.w[j < GROUPS ? j : 0] : s.x).c[h] =
                        __builtin_bit_cast(v4i, load16<false>(p + (whole ? k : last + static_cast<int>(rows[j].shift))));
                    s.more[j][h] = *reinterpret_cast<const uint32_t*>(p + (whole ? k + kChunk : 0));
                }
            }
        } else {
            const int kfirst = in ? kt * kTileK : 1 << 30;   // (past the slice: past K)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = kfirst + h * 64;
                const uint32_t off = k + cb < g.K ? row + k : kOob;
#pragma unroll
                for (int j = 0; j < GROUPS; ++j)
                    s.w[j].c[h] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rw[j], off, 0, 0));
                s.x.c[h] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rx, off, 0, 0));
            }
        }
        const __amdgpu_buffer_rsrc_t rs =
            make_rsrc(g.xs + static_cast<int64_t>(in ? kt : 0) * g.M, in ? static_cast<uint32_t>(g.M) * 4 : 0);
        s.s = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, (lane & 15) * 4, 0, 0));
    };

    v4f acc[GROUPS] = {};
    Slot ring[DEPTH];
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) fill(ring[u], kt0 + wave + u * kWaves);
    for (int kt = kt0 + wave; kt < kt1; kt += kWaves * DEPTH) {
#pragma unroll
        for (int u = 0; u < DEPTH; ++u) {
            const int t = kt + u * kWaves, ts = t < kt1 ? t : kt0;   // (a K-tile past the slice: zeros, times some scale)
            if constexpr (ANY) {
                if (t < kt1 && inside(t)) {   // (uniform)
#pragma unroll
                    for (int j = 0; j <= GROUPS; ++j)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            v4i& v = (j < GROUPS ? ring[u].w[j < GROUPS ? j : 0] : ring[u].x).c[h];
#pragma unroll
                            for (int d = 0; d < 4; ++d) {
                                const uint32_t next = d < 3 ? static_cast<uint32_t>(v[d < 3 ? d + 1 : 3]) : ring[u].more[j][h];
                                v[d] = static_cast<int>(__builtin_amdgcn_alignbyte(next, static_cast<uint32_t>(v[d]), rows[j].shift));
                            }
                        }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int k = t * kTileK + h * 64 + cb, past = t >= kt1 ? kChunk : k - (g.K - kChunk);
                        if (past <= 0) continue;
                        ring[u].x.c[h] = drop_front(ring[u].x.c[h], past);
#pragma unroll
                        for (int j = 0; j < GROUPS; ++j) ring[u].w[j].c[h] = drop_front(ring[u].w[j].c[h], past);
                    }
                }
            }
            const Widened x = widen(ring[u].x);
#pragma unroll
            for (int j = 0; j < GROUPS; ++j) add_scaled(acc[j], block_sum(widen(ring[u].w[j]), x), ring[u].s * wscale[j / kEach][ts]);
            fill(ring[u], t + DEPTH * kWaves);
        }
    }

    // A fragment's results: 4 * (lane >> 4) + register -> weight row, lane & 15 -> row m.
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) *reinterpret_cast<v4f*>(&part[((wave * GROUPS + j) * 64 + lane) * 4]) = acc[j];
    __syncthreads();
    auto sum_of = [&](int j, int m, int ch) {
        const int at = (j * 64 + (ch >> 2) * 16 + m) * 4 + (ch & 3);
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v += part[w * GROUPS * 256 + at];
        return v;
    };
    void* out = g.out;
    const int cols = g.kt_per_split ? g.pitch : g.N;   // of a row of `out`
    if (g.kt_per_split) out = static_cast<float*>(out) + static_cast<int64_t>(blockIdx.y) * g.M * cols;
    for (int e = threadIdx.x; e < 16 * kCols; e += 64 * kWaves) {
        const int m = e / kCols, ch = e % kCols, n = n0 + ch;
        if (m >= g.M || n >= cols) continue;
        float v;
        if constexpr (GATED) v = gate_value<ACT>(sum_of(ch >> 4, m, ch & 15)) * sum_of(kEach + (ch >> 4), m, ch & 15);
        else v = n < g.N ? sum_of(ch >> 4, m, ch & 15) + (g.bias && !g.kt_per_split ? g.bias[n] : 0.f) : 0.f;   // (0 behind a slab's row)
        store_value<OUT>(out, static_cast<int64_t>(m) * cols + n, v);
    }
}

struct GatedOut {
    uint8_t* q;      // [M, N]
    float* scale;    // [ceil(N / 128), M]
};

// ---- 256 x 256 outputs a workgroup: large products -----------------------------------------------------------------
// Eight waves, 2 (rows) x 4 (columns), a wave owns 128 x 64 outputs: eight row fragments by four column fragments (six, four
// or two row fragments where 256 rows would leave CUs idle).
//
// Within a K-tile a wave keeps the four column fragments and walks its row fragments; the sums of an earlier fragment are
// scaled into their accumulators behind the matrix instructions of a later one (two instructions later for the 8-bit form,
// four chains later for the bf16 form), so that vector and matrix work overlap without waiting for each other.
//
// A K-tile is two phases, A (read and widen the column fragments, the first half of the row fragments) and B (the others), a
// barrier before each.  Waves 4-7, the second wave of every SIMD, run one phase behind waves 0-3: while one wave reads and
// widens its column fragments the other keeps the matrix pipe busy.  With barrier 2t at the start of A(t) for waves 0-3:
//     after barrier 2t + 1 the rows x(t - 1) are read by nobody any more:  DMA of x(t + 2) into their slot (three slots)
//     after barrier 2t     the rows w(t - 2 + 1) likewise:                 DMA of w(t + 1) (two slots)
//     before barrier 2t    every wave has waited for its share of x(t) and w(t), issued three and two phases earlier; the
//                          four pieces of x(t + 1) may still be in flight
// which fills the CU's 160 KiB of LDS with 32 KiB slots.  K-tiles past the end are requested out of range (zeros, no memory
// traffic), so that every wave issues the same number of pieces.
//
// GATED: the tile is 128 columns of both weights, a wave's column fragments 0, 1 the gate's and 2, 3 the up projection's
// same 32 columns, so that a lane holds both factors of its outputs and the 128 columns are one block of the result.
//
// Measured: 8192x8192x8192 bf16 465-473 us (2.32-2.37 PFLOP/s; the library's product of the same size with one scale a tensor
// 383), gated 4096x14336x4096 740-755 us (1.27-1.30; the library's bf16 product does 1.52), fp32 1000x10001x4000 82.5 us (0.97;
// 240 tiles of 192 rows on 256 CUs).  Bound by the chip's power more than by any one pipe: the clock falls to 1.8 GHz (8-bit
// form) and 2.0 GHz (bf16 form) of 2.4 while the matrix pipes are 56% and 53% and vector issue 47% and 57% of the cycles busy.
// Without its LDS-DMA the 8-bit form took 385 us, without the scaling 445, without its reads of x 398; the bf16 form without
// widening 581.  32 x 32 instructions, which leave the vector unit more issue slots, were no faster: their accumulators, sixteen
// registers a piece, do not fit 256 rows beside the widened columns, and 192 rows took 825 us for 754.

// f(FIRST), ..., f(END - 1) with the index a constant.
template <int FIRST, int END, typename F>
__device__ __forceinline__ void static_for(F&& f) {
    if constexpr (FIRST < END) {
        f(std::integral_constant<int, FIRST>{});
        static_for<FIRST + 1, END>(f);
    }
}

template <int OUT, int ACT, bool NATIVE, int RF>
__global__ __launch_bounds__(512) void gemm_fp8_256_kernel(Fp8Args g, GatedOut go) {
    constexpr bool GATED = ACT != kNoAct;
    constexpr int kSlot = 256 * kTileK, kCols = GATED ? 128 : 256, kRows = RF * 32;   // (RF: row fragments of a wave)
    constexpr int AS = RF / 2;   // row fragments of phase A
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    int tm, tn;
    tile_coords(blockIdx.x, gridDim.x, g.tiles_m, g.tiles_n, 8, tm, tn);
    const int64_t m0 = static_cast<int64_t>(tm) * kRows;
    const int n0 = tn * kCols;
    const int mrows = static_cast<int>(g.M - m0 < kRows ? g.M - m0 : kRows), nrows = g.N - n0 < kCols ? g.N - n0 : kCols;

    // Staging: a wave-instruction moves 8 rows x 128 B; wave v moves rows v * 8 + 64 i, i = 0 .. 3, of each operand.  K-tile and
    // row group are in the lane's offset; rows past the matrix lie past the descriptor's end and read as zeros.  The operand is
    // picked by value, without a branch: a branch would leave the compiler unsure how many requests are younger than a scale's,
    // and it would wait for all of them before the scale's use.
    const int srow = wave * 8 + (lane >> 3);
    const int cbyte = ((lane & 7) ^ ((srow >> 1) & 7)) * kChunk;
    const uint32_t off0 = static_cast<uint32_t>(srow) * static_cast<uint32_t>(g.K) + cbyte, rows64 = 64u * static_cast<uint32_t>(g.K);
    const uint8_t* const x0 = g.x + m0 * g.K;
    const uint8_t* const w0 = g.w[0] + static_cast<int64_t>(n0) * g.K;
    const uint8_t* const w1 = g.w[GATED ? 1 : 0] + static_cast<int64_t>(n0) * g.K;
    const uint32_t xbytes = static_cast<uint32_t>(mrows) * static_cast<uint32_t>(g.K);
    const uint32_t wbytes = static_cast<uint32_t>(nrows) * static_cast<uint32_t>(g.K);
    // K-tile kt of the rows of w (else of x) to the 32 KiB at byte `slot` of LDS
    auto stage = [&](bool of_w, int kt, int slot) {
        const int k = kt * kTileK;
        const uint32_t off = k + cbyte < g.K ? off0 + k : kOob;
        const uint32_t bytes = of_w ? wbytes : xbytes;
        const uint8_t* const first = of_w ? w0 : x0;
        const uint8_t* const second = GATED && of_w ? w1 : first;   // of rows 128 .. 255: the other weight's, or 128 rows on
        const uint32_t on = GATED && of_w ? 0 : 2 * rows64;
        char* const to = smem + slot + wave * (8 * kTileK);
        dma16(make_rsrc(first, bytes), to, off);
        dma16(make_rsrc(first, bytes), to + 64 * kTileK, off + rows64);
        dma16(make_rsrc(second, bytes), to + 128 * kTileK, off + on);
        dma16(make_rsrc(second, bytes), to + 192 * kTileK, off + on + rows64);
    };
    auto x_slot = [](int slot) { return slot * kSlot; };
    auto w_slot = [](int kt) { return (3 + (kt & 1)) * kSlot; };

    // The scales of the wave's 128 rows for one K-tile, a lane one of each half: lane l has row l of the half.  spread() gives
    // every lane of a 16-lane row the scales of row fragment i, i.e. row 16 i + (lane & 15): three exchanges of 32- and
    // 16-lane rows between two copies.  Rows past the end read as 0.
    auto row_scales = [&](int kt, int half) {
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(g.xs + static_cast<int64_t>(kt) * g.M + m0, static_cast<uint32_t>(mrows) * 4);
        return __builtin_amdgcn_raw_buffer_load_b32(rs, static_cast<uint32_t>(wm * (RF * 16) + half * 64 + lane) * 4, 0, 0);
    };
    auto spread = [&](uint32_t v, float (&s)[4]) {
        const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const auto rows = __builtin_amdgcn_permlane16_swap(halves[h], halves[h], false, false);
            s[2 * h] = __uint_as_float(rows[0]);
            s[2 * h + 1] = __uint_as_float(rows[1]);
        }
    };
    const int nblock = GATED ? tn : tn * 2 + (wn >> 1);
    const int nblocks = (g.N + 127) / 128, nb = nblock < nblocks ? nblock : nblocks - 1;   // (columns past N: any scale)
    // (read through the scalar unit: a vector load here would be waited for behind the DMA issued before it)
    using scalar_floats = const __attribute__((address_space(4))) float*;
    const scalar_floats ws0 = (scalar_floats)(g.ws[0] + static_cast<int64_t>(nb) * g.kblocks);
    const scalar_floats ws1 = (scalar_floats)(g.ws[GATED ? 1 : 0] + static_cast<int64_t>(nb) * g.kblocks);

    // Column fragment j of this wave inside the staged 256 rows of w.
    const int lo0 = frag_lane_offset(lane, 0), lo1 = frag_lane_offset(lane, 1);
    auto w_row = [&](int j) { return GATED ? (j >> 1) * 128 + wn * 32 + (j & 1) * 16 : wn * 64 + j * 16; };
    auto read = [&](int tile, int row) {
        return Codes{{lds_read16(smem + tile + lo0 + row * kTileK), lds_read16(smem + tile + lo1 + row * kTileK)}};
    };

    using Frag = typename OperandOf<NATIVE>::Frag;
    v4f acc[RF][4] = {};
    v4f c[4] = {};   // sums of a block that are not scaled yet
    float s_cur[4], s[2] = {}, s_old[2] = {};   // scales of this row fragment (gate's or only, up's) and of the one before
    const int nt = g.kblocks;
    Frag wf[4], xf[2];        // column fragments; row fragment i (8-bit: in xf[i & 1], read one step ahead)
    Codes raw;                // the codes of row fragment i + 1
    auto scale_in = [&](v4f& a, const v4f& sum, float by, int e) { a[e] = __builtin_fmaf(sum[e], by, a[e]); };
    auto pin = [](v4f& a) { asm volatile("" : "+v"(a)); };   // scaled here, and not where the loop ends
    auto rows_step = [&](auto step, int xt, uint32_t sv, float sw0, float sw1) {
        constexpr int i = decltype(step)::value, p = i ? i - 1 : RF - 1;   // p: the row fragment before
        if constexpr (i % 4 == 0) spread(sv, s_cur);
        s_old[0] = s[0];
        s_old[1] = s[1];
        s[0] = s_cur[i % 4] * sw0;   // of column fragments 0, 1
        s[1] = GATED ? s_cur[i % 4] * sw1 : s[0];
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (NATIVE) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                __builtin_amdgcn_s_setprio(1);   // (over the other wave of the SIMD, which scales or reads meanwhile)
                c[j] = block_sum(wf[j], xf[i & 1]);
                __builtin_amdgcn_s_setprio(0);
                // column fragment j - 2 of this row fragment, or j + 2 of the one before
                v4f& a = j < 2 ? acc[p][j + 2] : acc[i][j - 2];
#pragma unroll
                for (int e = 0; e < 4; ++e) scale_in(a, c[j ^ 2], j < 2 ? s_old[0] : s[0], e);
                pin(a);
                if (i < RF - 1 && j == 0) xf[(i + 1) & 1] = read(xt, (i + 1) * 16);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            if (i > 0) {
                xf[0] = widen(raw);
                if (i < RF - 1) raw = read(xt, (i + 1) * 16);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) scale_in(acc[p][j], c[j], s_old[j >> 1], e);
                pin(acc[p][j]);
                c[j] = mfma_bf16(wf[j].h[0], xf[0].h[0], v4f{0.f, 0.f, 0.f, 0.f});
            }
#pragma unroll
            for (int h = 1; h < 4; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) c[j] = mfma_bf16(wf[j].h[h], xf[0].h[h], c[j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto barrier = [&] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // The youngest four pieces may be in flight (`with_scale`: and a row scale requested beside them), everything older has
    // landed; and this wave's LDS reads have returned (the slots that they read are written after the barrier).
    auto wait_all_but_one_slot = [](auto with_scale) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(with_scale.value ? 5 : 4) : "memory");
    };
    using One = std::integral_constant<bool, (RF > 4)>;   // row scales of a second half of the wave's rows
    auto wait_reads = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
    if (nt > 0) {
        uint32_t sv0 = row_scales(0, 0), sv1 = RF > 4 ? row_scales(0, 1) : 0;
        keep_order();
        stage(false, 0, x_slot(0));
        stage(true, 0, w_slot(0));
        keep_order();
        stage(false, 1, x_slot(1));
        wait_all_but_one_slot(std::false_type{});   // x(0), w(0)
        barrier();
        int group = wm;
        if (group == 1) {
            stage(true, 1, w_slot(1));
            barrier();
        }
        int slot = 0;   // of x(t)
        for (int t = 0; t < nt; ++t) {
            asm volatile("" : "+s"(group));   // (one loop for both groups: the body is not worth duplicating)
            const int xt = x_slot(slot) + wm * (RF * 16) * kTileK, wt = w_slot(t);
            const int ahead = slot == 0 ? 2 : slot - 1;   // of x(t + 2), and of x(t - 1)
            slot = slot == 2 ? 0 : slot + 1;
            const float sw0 = ws0[t], sw1 = GATED ? ws1[t] : sw0;
            // phase A
            Codes codes[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) codes[j] = read(wt, w_row(j));
            raw = read(xt, 0);
            keep_order();
            stage(group == 0, group ? t + 2 : t + 1, group ? x_slot(ahead) : w_slot(t + 1));   // (while the reads are on their way)
            keep_order();
#pragma unroll
            for (int j = 0; j < 4; ++j) wf[j] = operand<NATIVE>(codes[j]);
            xf[0] = operand<NATIVE>(raw);
            if constexpr (!NATIVE) raw = read(xt, 16);
            static_for<0, AS>([&](auto i) { rows_step(i, xt, sv0, sw0, sw1); });
            if (group) wait_all_but_one_slot(std::false_type{});   // x(t + 1), w(t + 1); x(t + 2) stays in flight
            else wait_reads();
            barrier();
            // phase B: the next scales, each into the register that it replaces: the first half's is free, the second half's
            // after row fragment 4 (a copy at the loop's end would wait for the request, and for all pieces before it)
            const int tn1 = t + 1 < nt ? t + 1 : t;
            sv0 = row_scales(tn1, 0);
            keep_order();
            stage(group != 0, t + 2, group ? w_slot(t + 2) : x_slot(ahead));
            keep_order();
            constexpr int kLast = RF > 4 ? 5 : RF;   // (the row fragments behind it have their scales already)
            static_for<AS, kLast>([&](auto i) { rows_step(i, xt, sv1, sw0, sw1); });
            if constexpr (RF > 4) sv1 = row_scales(tn1, 1);
            keep_order();
            static_for<kLast, RF>([&](auto i) { rows_step(i, xt, sv1, sw0, sw1); });
            if (group) wait_reads();
            else wait_all_but_one_slot(One{});
            barrier();
        }
        if (wm == 0) barrier();   // every wave executes the same number of barriers
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the pieces requested for K-tiles past the end
    }
    // the sums still waiting
#pragma unroll
    for (int j = NATIVE ? 2 : 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) scale_in(acc[RF - 1][j], c[j], s[j >> 1], e);

    // Results of a fragment: 4 * (lane >> 4) + register -> column, lane & 15 -> row.
    const int64_t mw = m0 + wm * (RF * 16) + (lane & 15);
    if constexpr (GATED) {
        // The tile's 128 columns are a block of the result.  Its maximum for each row: over the lane's eight values, the
        // four lanes of the row, and the four waves of the row through LDS.
        __syncthreads();   // every wave has read its last K-tile
        uint32_t* tops = reinterpret_cast<uint32_t*>(smem);   // [4][256]
        auto top_of = [&](int i, auto bits) {
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t b = bits(acc[i][j][e]);
                    top = b > top ? b : top;
                }
            uint32_t o = __shfl_xor(top, 16, 64);
            top = o > top ? o : top;
            o = __shfl_xor(top, 32, 64);
            top = o > top ? o : top;
            if (lane < 16) tops[wn * 256 + wm * (RF * 16) + i * 16 + lane] = top;
        };
#pragma unroll
        for (int i = 0; i < RF; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = gate_value<ACT>(acc[i][j][e]) * acc[i][j + 2][e];
            top_of(i, magnitude_bits);
        }
        __syncthreads();
        auto row_top = [&](int i) {
            const uint32_t* t = tops + wm * (RF * 16) + i * 16 + (lane & 15);
            uint32_t top = t[0];
#pragma unroll
            for (int w = 1; w < 4; ++w) top = t[w * 256] > top ? t[w * 256] : top;
            return top;
        };
        bool spoiled = false;   // some value of this wave's rows is not finite: the same in the four waves of these rows
#pragma unroll
        for (int i = 0; i < RF; ++i) spoiled |= row_top(i) >= kInfBits;
        spoiled = __any(spoiled);
        __syncthreads();
        if (spoiled) {
#pragma unroll
            for (int i = 0; i < RF; ++i) top_of(i, finite_magnitude_bits);
        }
        __syncthreads();
        const bool vec = (g.N & 3) == 0;
#pragma unroll
        for (int i = 0; i < RF; ++i) {
            const int64_t m = mw + i * 16;
            const BlockScale s = block_scale(row_top(i));
            if (m >= g.M) continue;
            if (wn == 0 && lane < 16) go.scale[static_cast<int64_t>(tn) * g.M + m] = s.scale;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int n = n0 + wn * 32 + j * 16 + (lane >> 4) * 4;
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = __fmul_rn(spoiled ? infinite_to_nan(acc[i][j][e]) : acc[i][j][e], s.inv);
                const uint32_t code = pack4_e4m3(f[0], f[1], f[2], f[3]);
                uint8_t* o = go.q + m * g.N + n;
                if (vec && n + 3 < g.N) *reinterpret_cast<uint32_t*>(o) = code;
                else
                    for (int e = 0; e < 4; ++e)
                        if (n + e < g.N) o[e] = static_cast<uint8_t>(code >> (8 * e));
            }
        }
    } else {
        __syncthreads();               // every wave has read its last K-tile (LDS is used again below)
        const int nw = n0 + wn * 64;   // the wave's 64 columns
        if (g.bias) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = nw + j * 16 + (lane >> 4) * 4;
                v4f b;
#pragma unroll
                for (int e = 0; e < 4; ++e) b[e] = n + e < g.N ? g.bias[n + e] : 0.f;
#pragma unroll
                for (int i = 0; i < RF; ++i) acc[i][j] += b;
            }
        }
        if ((g.N & 7) == 0 && nw + 64 <= g.N) {
            // Whole cache lines: as they lie, an instruction would write sixteen rows x 64 (fp32) or 32 bytes.  Lanes r and
            // r ^ 8 of a 16-lane row trade halves of a row's pieces, so that one writes eight rows x 128 bytes.
            const int r = lane & 15;
            const bool lo = r < 8;
            auto store_rows = [&](v4i first, v4i second, int64_t m1, int n, int size) {   // first: columns of the low half
                v4i a, b;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int recv = __builtin_amdgcn_update_dpp(0, lo ? second[e] : first[e], 0x128 /* row_ror:8 */, 0xf, 0xf, false);
                    a[e] = lo ? first[e] : recv;
                    b[e] = lo ? recv : second[e];
                }
                char* o = static_cast<char*>(g.out) + (m1 * g.N + n) * size;
                if (m1 < g.M) __builtin_nontemporal_store(a, reinterpret_cast<v4i*>(o));
                if (m1 + 8 < g.M) __builtin_nontemporal_store(b, reinterpret_cast<v4i*>(o + 8ll * g.N * size));
            };
#pragma unroll
            for (int i = 0; i < RF; ++i) {
                const int64_t m1 = m0 + wm * (RF * 16) + i * 16 + (r & 7);
                if constexpr (OUT == MIQ_F32) {
#pragma unroll
                    for (int j = 0; j < 4; j += 2)
                        store_rows(__builtin_bit_cast(v4i, acc[i][j]), __builtin_bit_cast(v4i, acc[i][j + 1]), m1,
                                   nw + j * 16 + (lo ? 0 : 16) + (lane >> 4) * 4, 4);
                } else {
                    uint2 p[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[j] = pack4<OUT>(acc[i][j]);
                    store_rows(pair_rows_bf16(p[0], p[1]), pair_rows_bf16(p[2], p[3]), m1, nw + (lo ? 0 : 32) + paired_offset(lane), 2);
                }
            }
        } else {
            // Rows that start anywhere: a row fragment's 16 x 64 through LDS (the wave's own 16 rows of 68 floats), then one row
            // an instruction, a column a lane.
            float* const rows = reinterpret_cast<float*>(smem) + wave * (16 * 68);
            const int n = nw + lane;
#pragma unroll
            for (int i = 0; i < RF; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) *reinterpret_cast<v4f*>(rows + (lane & 15) * 68 + j * 16 + (lane >> 4) * 4) = acc[i][j];
                wave_lds_order();
                const int64_t m = m0 + wm * (RF * 16) + i * 16;
                float v[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) v[r] = rows[r * 68 + lane];
                wave_lds_order();
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (n < g.N && m + r < g.M) store_value<OUT>(g.out, (m + r) * g.N + n, v[r]);
            }
        }
    }
}

// ---- split products: the slabs' sums ---------------------------------------------------------------------------------
// In the slices' order, whatever order they ended in.  Launch-bound: 2.8 to 3.7 us at these sizes, 0.15 us more a slice.
// Eight consecutive sums of a row at `at`, over `splits` slabs of `size` floats, in order.
__device__ __forceinline__ void sum_slabs(const float* __restrict__ slabs, int splits, int64_t size, int64_t at, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const v4f* p = reinterpret_cast<const v4f*>(slabs + s * size + at);
        const v4f a = p[0], b = p[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] += a[i];
            v[4 + i] += b[i];
        }
    }
}

// out = the slabs' sum + bias; eight columns a thread (slab rows are a multiple of 8 long)
template <int OUT>
__global__ __launch_bounds__(256) void splitk_sum_kernel(const float* __restrict__ slabs, int splits, Fp8Args g, void* __restrict__ out) {
    const int per_row = g.pitch / 8;
    const int64_t total = g.M * per_row;
    const bool vec = (g.N & 3) == 0;
    for (int64_t id = blockIdx.x * 256ll + threadIdx.x; id < total; id += gridDim.x * 256ll) {
        const int64_t m = id / per_row;
        const int n = static_cast<int>(id % per_row) * 8;
        float v[8];
        sum_slabs(slabs, splits, g.M * g.pitch, m * g.pitch + n, v);
        if (g.bias) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (n + i < g.N) v[i] += g.bias[n + i];
        }
        store4<OUT>(out, m * g.N + n, g.N - n, vec, v4f{v[0], v[1], v[2], v[3]});
        store4<OUT>(out, m * g.N + n + 4, g.N - n - 4, vec, v4f{v[4], v[5], v[6], v[7]});
    }
}

// h = act(sum of the gate's slabs) * (sum of the up projection's), in blocks: sixteen lanes a block of one row (48 rows of 14336:
// 4.1 us for the 5.5 MB of two slabs, which come from the L2s and the Infinity Cache).
template <int ACT>
__global__ __launch_bounds__(256) void gated_join_kernel(const float* __restrict__ slabs, int splits, Fp8Args g, int nblocks,
                                                         uint8_t* __restrict__ q, float* __restrict__ scale) {
    const int lane = threadIdx.x & 15;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
    const int64_t m = id / nblocks;
    const int b = static_cast<int>(id % nblocks), n = b * 128 + lane * 8;
    const int64_t size = g.M * g.pitch;
    float gate[8] = {}, h[8] = {};
    if (m < g.M && n < g.pitch) {
        sum_slabs(slabs, splits, size, m * g.pitch + n, gate);
        sum_slabs(slabs + splits * size, splits, size, m * g.pitch + n, h);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = gate_value<ACT>(gate[i]) * h[i];   // (0 past the row)
    uint32_t c[2];
    const float s = quantize8_in_row(h, c);
    const int inside = m < g.M && n < g.N ? (g.N - n < 8 ? g.N - n : 8) : 0;
    if ((g.N & 7) == 0) store8_codes<true>(q, m * g.N + n, inside, c);
    else store8_codes<false>(q, m * g.N + n, inside, c);
    if (lane == 0 && m < g.M) scale[static_cast<int64_t>(b) * g.M + m] = s;
}

// Every size that the kernels index with 32 bits, bounded before any arithmetic.
int check_sizes(const char* who, int64_t M, int64_t N, int64_t K) {
    MIQ_REQUIRE(M >= 0 && N >= 0 && K >= 0, MIQ_EINVAL, "%s: negative size (M=%lld N=%lld K=%lld)", who, (long long)M, (long long)N,
                (long long)K);
    MIQ_REQUIRE(M < (1ll << 31) && N < (1ll << 31) - 256 && K < (1ll << 22), MIQ_ERANGE,
                "%s: M and N must be below 2^31, K below 2^22 (M=%lld N=%lld K=%lld)", who, (long long)M, (long long)N, (long long)K);
    const int64_t tiles = ceil_div(M, 64) * ceil_div(N, 64);
    MIQ_REQUIRE(tiles <= (1ll << 22), MIQ_ERANGE, "%s: more than 2^22 tiles of 64 x 64 outputs", who);
    // (at most 16 rows: 512 threads for 16 columns, and a launch holds less than 2^32 threads)
    MIQ_REQUIRE(M > 16 || N <= (1ll << 26), MIQ_ERANGE, "%s: more than 2^26 columns of at most 16 rows", who);
    return MIQ_OK;
}

size_t align256(int64_t n) { return static_cast<size_t>(round_up(n, 256)); }

// A row length that is no multiple of 16 bytes cannot be staged in 16-byte pieces: both operands are first copied to rows of
// a multiple of 16, zero-filled (codes of 0 add nothing), at the front of the workspace.  (The kernel for at most 16 rows stages
// nothing; it reads rows of at least 16 bytes as they are.)
int64_t pitch_of(int64_t K) { return round_up(K, kChunk); }
bool is_padded(int64_t M, int64_t K) { return K % kChunk != 0 && (M > 16 || K < kChunk); }
size_t padded_bytes(int64_t M, int64_t N, int64_t weights, int64_t K) {
    return is_padded(M, K) ? align256(M * pitch_of(K)) + static_cast<size_t>(weights) * align256(N * pitch_of(K)) : 0;
}
// What a product is cut into: which kernel, how K is split, and how much workspace that needs behind the padded operands.
struct Fp8Plan {
    int big;         // rows of the large kernel's tile, 256, 192, 128 or 64; 0: not that kernel
    int bm;          // rows of the tile kernel's tile, 128, 64 or 32; 0: the kernel for at most 16 rows
    int splits;      // slices of K; 1: none
    int kt_per_split;
    size_t slabs;    // bytes of fp32 slabs
};

constexpr int64_t kCus = 256;

// Above 16 rows the large kernel and the tile kernel, the latter with tiles of three heights and K in any number of slices, can
// all run a product: the one with the smallest estimate does.  The estimates' constants are us, fitted to the times of every
// variant on 227 shapes, M 17 to 7701, N 65 to 28672, K 128 to 28672, 0.6 TFLOP at most: the estimates are within 12% of the
// times, the choice within 3% of the best variant's on average.  E.g. 512x2048x2048 bf16: 64-row tiles 9.0, in two slices 14.8,
// 128-row tiles 17.3, the large kernel 16.3 (64 rows); 254x354x2560 bf16: 32-row tiles in four slices 7.7, 64-row tiles whole 9.0,
// the large kernel 19.4; gated 2785x669x10032: 128-row tiles in four slices 112, in two 122, the large kernel 143 (128 rows);
// gated 2773x5456x224: the large kernel 34 (256 rows), 128-row tiles 57; fp32 1000x10001x4000: the large kernel 84 (192 rows), 101
// (256), 128-row tiles 97.
struct BigFit {
    double k_tile, round;
};
// `work` us of the workgroups' K-tiles while `weights` bytes stream at `rate` bytes a ps: the larger, somewhat more where they
// are near each other.
double overlapped_us(double work, double weights, double rate) {
    const double stream = weights / (rate * 1e6), w2 = work * work, s2 = stream * stream;
    return std::sqrt(std::sqrt(w2 * w2 + s2 * s2));
}
// One workgroup a CU: as many rounds as the tiles need, each a time a K-tile and a prologue and epilogue.
double big_us(int i, int64_t M, int64_t N, int64_t nt, double weights, bool gated, bool native) {
    static constexpr BigFit kFit[2][4] = {{{2.88, 12.9}, {2.25, 11.2}, {1.68, 8.9}, {1.22, 5.4}},   // bf16 form: 256 to 64 rows
                                          {{1.58, 10.0}, {1.16, 9.5}, {0.98, 6.2}, {0.91, 4.2}}};   // 8-bit form
    const BigFit& f = kFit[native][i];
    const int64_t tiles = ceil_div(M, 256 - 64 * i) * ceil_div(N, gated ? 128 : 256);
    return 3.0 + overlapped_us(static_cast<double>(ceil_div(tiles, kCus)) * (f.k_tile * static_cast<double>(nt) + f.round), weights, 2.8);
}
// `groups` workgroups of `kt` K-tiles each, `resident` on a CU.  A workgroup alone on its CU takes `alone` a K-tile (a fetch and
// its own matrix work), a full CU `full` for each workgroup's; `stream` is the rate of the weights' stream, bytes a ps.
struct TileFit {
    double fixed, alone, full, stream;
};
struct Tile {
    int rows, resident;
    TileFit fit[2];   // bf16 form, 8-bit form
};
constexpr Tile kTiles[3] = {{32, 4, {{4.1, 0.30, 0.228, 6.0}, {3.5, 0.223, 0.198, 5.9}}},
                            {64, 3, {{4.5, 0.414, 0.321, 6.0}, {3.7, 0.29, 0.285, 5.9}}},
                            {128, 2, {{5.9, 1.12, 0.916, 5.2}, {4.2, 1.06, 0.672, 4.25}}}};
double tile_us(const Tile& t, int64_t groups, int64_t kt, double weights, bool native) {
    const TileFit& f = t.fit[native];
    const int64_t deep = ceil_div(groups, kCus);   // workgroups of the busiest CU
    const double alone = f.alone * static_cast<double>(ceil_div(deep, t.resident)), full = f.full * static_cast<double>(deep);
    return f.fixed + overlapped_us(static_cast<double>(kt) * (alone > full ? alone : full), weights, f.stream);
}

Fp8Plan make_plan(int64_t M, int64_t N, int64_t K, bool gated, bool native) {
    Fp8Plan p{};
    p.splits = 1;
    const int64_t nt = ceil_div(K, kTileK);
    const int64_t slab = 4 * M * round_up(N, 8);
    if (M <= 16) {
        // K in slices of at least eight K-tiles where the columns give few workgroups and K is long enough to pay for the second
        // launch: 1x512x28672 18.3 us whole, 8.0 in eight slices, 1x512x14336 11.2 and 6.6 (and 4 us more of the host), 1x2048x8192
        // 7.4 and 8.3.  (In a captured graph, where a launch is no time of the host, 14336 columns of K would be worth slicing, too.)
        // A gated product is never sliced, whatever K is: tried was a launch for each weight's slabs and one that joins them, three
        // in all (8x2048x4096 12.9 us for 10.7).  Both weights' slabs from one launch, joined by the second, has not been built: the
        // narrow and long products run on N / 16 workgroups (1x512x14336 19.3 us, 4x1024x8192 14.4; the bytes of either are 3).
        const int64_t groups = ceil_div(N, 16);
        if (!gated && groups < 192 && nt >= 128) {
            int64_t splits = kCus / groups;
            if (splits > nt / 8) splits = nt / 8;
            if (splits > 32) splits = 32;
            p.kt_per_split = static_cast<int>(ceil_div(nt, splits));
            p.splits = static_cast<int>(ceil_div(nt, p.kt_per_split));
        }
        p.slabs = gated ? static_cast<size_t>(4 * M * N) : p.splits > 1 ? static_cast<size_t>(slab) * p.splits : 0;   // gated: act(g) * u
        return p;
    }
    const int products = gated ? 2 : 1;
    const double weights = static_cast<double>(products * N * K) * (K % kTileK ? 1.3 : 1.0);   // (rows that start inside a cache line)
    double best = 1e30;
    for (int i = 0; i < 4; ++i) {
        const double us = big_us(i, M, N, nt, weights, gated, native);
        if (us < best) {
            best = us;
            p.big = 256 - 64 * i;
        }
    }
    constexpr int64_t kMostSlabs = int64_t{1} << 28;
    static constexpr int kSlices[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
    for (const Tile& t : kTiles) {
        const int64_t tiles = ceil_div(M, t.rows) * ceil_div(N, t.rows == 128 ? 128 : 64) * products;
        for (const int s : kSlices) {
            if (s > 1 && (s > nt / 2 || tiles * s > 6 * kCus)) break;
            const int64_t kt = ceil_div(nt, s), slices = nt > 0 ? ceil_div(nt, kt) : 1;
            double us = tile_us(t, tiles * slices, kt, weights, native);
            if (slices > 1 || gated) {
                const int64_t bytes = products * slices * slab;
                if (bytes > kMostSlabs) break;
                us += 3.5 + 0.15 * static_cast<double>(slices) + static_cast<double>(bytes) / 3.3e6;   // second launch; slabs written, read
            }
            if (us >= best) continue;
            best = us;
            p.big = 0;
            p.bm = t.rows;
            p.splits = static_cast<int>(slices);
            p.kt_per_split = static_cast<int>(slices > 1 || gated ? (kt > 0 ? kt : 1) : 0);   // gated: one slab a weight at least
        }
    }
    if (!p.big && (gated || p.splits > 1)) p.slabs = static_cast<size_t>(products * p.splits * slab);
    return p;
}

template <int BM, int BN, int WAVES_M, int WAVES_N, int STAGES, int OUT, bool NATIVE>
int launch_tile(Fp8Args g, int splits, int products, hipStream_t st) {
    constexpr int kLds = STAGES * tile_stage_bytes(BM, BN, WAVES_M * WAVES_N);
    g.tiles_m = static_cast<int>(ceil_div(g.M, BM));
    g.tiles_n = static_cast<int>(ceil_div(g.N, BN));
    const dim3 grid(static_cast<unsigned>(g.tiles_m) * g.tiles_n, splits, products);
    const void* fn = reinterpret_cast<const void*>(&gemm_fp8_tile_kernel<BM, BN, WAVES_M, WAVES_N, STAGES, OUT, NATIVE>);
    if (int rc = allow_lds(fn, kLds)) return rc;
    gemm_fp8_tile_kernel<BM, BN, WAVES_M, WAVES_N, STAGES, OUT, NATIVE><<<grid, 64 * WAVES_M * WAVES_N, kLds, st>>>(g);
    return check_launch("gemm_fp8_tile_kernel");
}
// NATIVE16: the products of a 16-bit output (the slabs' sums included) may use the 8-bit instruction.  Stages and waves as
// measured: a ring of three K-tiles fits three workgroups a CU, one of four two (77x14336x4096 bf16 16.9 us against 17.2), one of
// two waits for each fetch (21.8); 64 x 64 tiles as four waves of 32 x 32 (as two of 32 x 64 21.0); 128 x 128 tiles as eight
// waves of 32 x 64 (256x4096x14336 bf16 31.9 us, as four of 64 x 64 32.7, with a ring of three 38.9).  A 64 x 64 tile that has
// its CU to itself goes to eight waves on the 8-bit instruction: nothing else covers a wave's wait (128x8192x8192 bf16 21.6 us,
// four waves 25.9; two workgroups a CU: 512x4096x4096 17.7 and 17.3; widening, eight waves lose: 427x5073x3712 36.2 and 30.0).
template <int OUT, bool NATIVE16>
int launch_tiles(const Fp8Plan& p, const Fp8Args& g, int products, hipStream_t st) {
    if (p.bm == 32) return launch_tile<32, 64, 2, 2, 3, OUT, NATIVE16>(g, p.splits, products, st);
    if (p.bm == 64) {
        const bool alone = ceil_div(g.M, 64) * ceil_div(g.N, 64) * p.splits * products <= kCus;
        if constexpr (NATIVE16)
            if (alone) return launch_tile<64, 64, 4, 2, 3, OUT, NATIVE16>(g, p.splits, products, st);
        return launch_tile<64, 64, 2, 2, 3, OUT, NATIVE16>(g, p.splits, products, st);
    }
    return launch_tile<128, 128, 4, 2, 2, OUT, NATIVE16>(g, p.splits, products, st);
}

template <int GROUPS, int OUT, int ACT>
int launch_rows16(const Fp8Plan& p, const Fp8Args& g, hipStream_t st) {
    // Two K-tiles in flight a wave: with four a wave holds 100 registers instead of 58 and fewer fit a SIMD (1 x 4096 x 14336:
    // 11.7 us against 12.6; 1 x 28672 x 8192 44.3 against 47.6).
    const dim3 grid(static_cast<unsigned>(ceil_div(g.N, ACT != kNoAct ? GROUPS * 8 : GROUPS * 16)), p.splits);
    if (g.K % kChunk) gemm_fp8_rows16_kernel<GROUPS, 8, 2, OUT, ACT, true><<<grid, 512, 0, st>>>(g);
    else gemm_fp8_rows16_kernel<GROUPS, 8, 2, OUT, ACT, false><<<grid, 512, 0, st>>>(g);
    return check_launch("gemm_fp8_rows16_kernel");
}
template <int OUT>
int launch_rows16_linear(const Fp8Plan& p, const Fp8Args& g, hipStream_t st) {
    // 32 columns a workgroup where a wave has few K-tiles to stream and that still gives every CU a workgroup (1 x 14336 x 4096:
    // 14.1 us against 15.8 with 16 columns), 16 elsewhere (1 x 4096 x 14336: 11.7 against 17.4, 1 x 28672 x 8192: 44 against 56).
    if (p.splits == 1 && g.kblocks <= 48 && ceil_div(g.N, 32) >= kCus) return launch_rows16<2, OUT, kNoAct>(p, g, st);
    return launch_rows16<1, OUT, kNoAct>(p, g, st);
}

template <int OUT, int ACT, bool NATIVE, int RF>
int launch_big_rows(Fp8Args g, GatedOut go, hipStream_t st) {
    constexpr int kLds = 5 * 256 * kTileK;
    g.tiles_m = static_cast<int>(ceil_div(g.M, RF * 32));
    g.tiles_n = static_cast<int>(ceil_div(g.N, ACT != kNoAct ? 128 : 256));
    const void* fn = reinterpret_cast<const void*>(&gemm_fp8_256_kernel<OUT, ACT, NATIVE, RF>);
    if (int rc = allow_lds(fn, kLds)) return rc;
    gemm_fp8_256_kernel<OUT, ACT, NATIVE, RF><<<static_cast<unsigned>(g.tiles_m) * g.tiles_n, 512, kLds, st>>>(g, go);
    return check_launch("gemm_fp8_256_kernel");
}
template <int OUT, int ACT, bool NATIVE>
int launch_big(const Fp8Plan& plan, const Fp8Args& g, GatedOut go, hipStream_t st) {
    if (plan.big == 256) return launch_big_rows<OUT, ACT, NATIVE, 8>(g, go, st);
    if (plan.big == 192) return launch_big_rows<OUT, ACT, NATIVE, 6>(g, go, st);
    if (plan.big == 128) return launch_big_rows<OUT, ACT, NATIVE, 4>(g, go, st);
    return launch_big_rows<OUT, ACT, NATIVE, 2>(g, go, st);
}

size_t workspace_of(const char* who, int64_t M, int64_t N, int64_t K, bool gated, bool native) {
    if (check_sizes(who, M, N, K) != MIQ_OK || M == 0 || N == 0) return 0;
    return padded_bytes(M, N, gated ? 2 : 1, K) + make_plan(M, N, K, gated, native).slabs;
}
int check_workspace(const char* who, size_t need, const void* workspace, size_t bytes) {
    MIQ_REQUIRE(need == 0 || (workspace && bytes >= need), MIQ_EWORKSPACE, "%s: %zu bytes of workspace needed, %zu given", who, need,
                workspace ? bytes : 0);
    MIQ_REQUIRE(aligned(workspace, 256), MIQ_EALIGN, "%s: workspace must be 256-byte aligned", who);
    return MIQ_OK;
}

// The arguments of a launch, operands padded where they need it; `at` is moved past what that took of the workspace.
Fp8Args make_args(const uint8_t* x, const float* xs, const uint8_t* w, const float* ws, const uint8_t* w2, const float* ws2, int64_t M,
                  int64_t N, int64_t K, char*& at, hipStream_t st) {
    Fp8Args g{};
    g.x = x;
    g.xs = xs;
    g.w[0] = w;
    g.w[1] = w2;
    g.ws[0] = ws;
    g.ws[1] = ws2;
    g.M = M;
    g.N = static_cast<int>(N);
    g.K = static_cast<int>(is_padded(M, K) ? pitch_of(K) : K);
    g.kblocks = static_cast<int>(ceil_div(K, kTileK));
    g.pitch = static_cast<int>(round_up(N, 8));
    if (is_padded(M, K)) {
        PadArgs a{{x, w, w2}, {}, {M, N, w2 ? N : 0}, static_cast<int>(K), g.K};
        for (int o = 0; o < 3; ++o) {
            a.dst[o] = reinterpret_cast<uint8_t*>(at);
            at += align256(a.rows[o] * g.K);
        }
        g.x = a.dst[0];
        g.w[0] = a.dst[1];
        if (w2) g.w[1] = a.dst[2];
        const int64_t groups = ceil_div(M > N ? M : N, 4);
        pad_rows_kernel<<<dim3(static_cast<unsigned>(groups < 16384 ? groups : 16384), w2 ? 3 : 2), 256, 0, st>>>(a);
    }
    return g;
}

template <int OUT>
int run_product(Fp8Args g, const Fp8Plan& p, void* slabs, hipStream_t st) {
    if (p.big) return launch_big<OUT, kNoAct, OUT != MIQ_F32>(p, g, {}, st);
    if (p.splits == 1) {
        if (p.bm == 0) return launch_rows16_linear<OUT>(p, g, st);
        return launch_tiles<OUT, OUT != MIQ_F32>(p, g, 1, st);
    }
    void* const out = g.out;
    g.out = slabs;
    g.kt_per_split = p.kt_per_split;
    const int rc = p.bm == 0 ? launch_rows16<1, MIQ_F32, kNoAct>(p, g, st) : launch_tiles<MIQ_F32, OUT != MIQ_F32>(p, g, 1, st);
    if (rc) return rc;
    const int64_t groups = ceil_div(g.M * (g.pitch / 8), 256);
    splitk_sum_kernel<OUT><<<static_cast<unsigned>(groups < 8192 ? groups : 8192), 256, 0, st>>>(static_cast<const float*>(slabs), p.splits,
                                                                                                g, out);
    return check_launch("splitk_sum_kernel");
}

template <int ACT>
int run_gated(Fp8Args g, const Fp8Plan& p, float* slabs, uint8_t* q, float* scale, hipStream_t st) {
    if (p.big) return launch_big<MIQ_F32, ACT, false>(p, g, {q, scale}, st);
    g.out = slabs;
    g.kt_per_split = p.kt_per_split;
    if (p.bm == 0) {
        if (int rc = launch_rows16<2, MIQ_F32, ACT>(p, g, st)) return rc;
        return miq_quantize_blocks_fp8(slabs, MIQ_F32, g.M, g.N, q, scale, st);
    }
    if (int rc = launch_tiles<MIQ_F32, false>(p, g, 2, st)) return rc;
    const int nblocks = static_cast<int>(ceil_div(g.N, 128));
    gated_join_kernel<ACT><<<static_cast<unsigned>(ceil_div(g.M * nblocks, 16)), 256, 0, st>>>(slabs, p.splits, g, nblocks, q, scale);
    return check_launch("gated_join_kernel");
}

}  // namespace

extern "C" size_t miq_gemm_fp8_workspace(int64_t M, int64_t N, int64_t K, int out_dtype) {
    return workspace_of("miq_gemm_fp8_workspace", M, N, K, false, out_dtype != MIQ_F32);
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
    MIQ_REQUIRE(aligned(x, 16) && aligned(w, 16), MIQ_EALIGN, "miq_gemm_fp8: x and w must be 16-byte aligned");
    const Fp8Plan plan = make_plan(M, N, K, false, out_dtype != MIQ_F32);
    if (int rc = check_workspace("miq_gemm_fp8", padded_bytes(M, N, 1, K) + plan.slabs, workspace, workspace_bytes)) return rc;
    const hipStream_t st = as_stream(stream);
    char* at = static_cast<char*>(workspace);
    Fp8Args g = make_args(x, x_scale, w, w_scale, nullptr, nullptr, M, N, K, at, st);
    g.bias = bias;
    g.out = out;
    if (out_dtype == MIQ_F32) return run_product<MIQ_F32>(g, plan, at, st);
    if (out_dtype == MIQ_F16) return run_product<MIQ_F16>(g, plan, at, st);
    return run_product<MIQ_BF16>(g, plan, at, st);
}

extern "C" size_t miq_gated_fp8_workspace(int64_t M, int64_t N, int64_t K) {
    return workspace_of("miq_gated_fp8_workspace", M, N, K, true, false);
}

extern "C" int miq_gated_fp8(const uint8_t* x, const float* x_scale, const uint8_t* w_gate, const float* gate_scale,
                             const uint8_t* w_up, const float* up_scale, int64_t M, int64_t N, int64_t K, int act, uint8_t* q,
                             float* scale, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_sizes("miq_gated_fp8", M, N, K)) return rc;
    MIQ_REQUIRE(act == MIQ_ACT_SILU || act == MIQ_ACT_GELU, MIQ_EINVAL, "miq_gated_fp8: unknown activation %d", act);
    if (M == 0 || N == 0) return MIQ_OK;
    MIQ_REQUIRE(q && scale && (K == 0 || (x && x_scale && w_gate && gate_scale && w_up && up_scale)), MIQ_EINVAL,
                "miq_gated_fp8: null pointer");
    MIQ_REQUIRE(aligned(x_scale, 4) && aligned(gate_scale, 4) && aligned(up_scale, 4) && aligned(scale, 4) && aligned(q, 16), MIQ_EALIGN,
                "miq_gated_fp8: scales must be 4-byte, q 16-byte aligned");
    MIQ_REQUIRE(aligned(x, 16) && aligned(w_gate, 16) && aligned(w_up, 16), MIQ_EALIGN,
                "miq_gated_fp8: x and the weights must be 16-byte aligned");
    const Fp8Plan plan = make_plan(M, N, K, true, false);
    if (int rc = check_workspace("miq_gated_fp8", padded_bytes(M, N, 2, K) + plan.slabs, workspace, workspace_bytes)) return rc;
    const hipStream_t st = as_stream(stream);
    char* at = static_cast<char*>(workspace);
    Fp8Args g = make_args(x, x_scale, w_gate, gate_scale, w_up, up_scale, M, N, K, at, st);
    float* slabs = reinterpret_cast<float*>(at);
    return act == MIQ_ACT_SILU ? run_gated<MIQ_ACT_SILU>(g, plan, slabs, q, scale, st)
                               : run_gated<MIQ_ACT_GELU>(g, plan, slabs, q, scale, st);
}
