// Products of e4m3 operands with a scale per block of 128, and their quantisation, on gfx950.
//
//   c[m, n] = sum over kb of sa[m, kb] sb[n / 128, kb] P_kb[m, n],   P_kb = sum over k in kb of a[m, k] b[n, k]
// P_kb comes from the matrix instructions, and one multiply-add per output and kb puts it into the f32 sum with its
// scale. The 8-bit instructions do not keep 32 bits of a sum: their results are 1.4e-5 of the norm off over 128 normal
// values (16x16x128 and 16x16x32 alike), as if the products were cut off 2^-17 below the largest. That is far below
// half a step of bf16 or f16, so 16-bit results use them; f32 results take the same codes as f16 values (exact)
// through the f16 instructions (9e-9 off), at half the rate. The weights are the instruction's A
// operand and the activations its B operand, so that a lane's results belong to one m: its scale is one register.
#include "kv8_device.hpp"

namespace tsfm {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int KB = 128;  // values per scale

__device__ __forceinline__ i32x8 pair(u32x4 lo, u32x4 hi) {
    return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
// 32 x 32 x 64 and 16 x 16 x 128: A and B hold 32 bytes of a row per lane, in the same order of k.
// EXACT: as four f16 instructions on 8 bytes each.
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
template <bool EXACT>
struct Operand {
    u32x4 h[4];  // f16
    __device__ __forceinline__ void set(i32x8 x) {
#pragma unroll
        for (int s = 0; s < 4; s++) h[s] = decode8<kCodeE4m3, false>((uint32_t)x[2 * s], (uint32_t)x[2 * s + 1]);
    }
};
template <>
struct Operand<false> {
    i32x8 x;
    __device__ __forceinline__ void set(i32x8 v) { x = v; }
};
__device__ __forceinline__ f32x16 mul(const Operand<false>& a, const Operand<false>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a.x, b.x, c, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mul(const Operand<false>& a, const Operand<false>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.x, b.x, c, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mul(const Operand<true>& a, const Operand<true>& b, f32x16 c) {
#pragma unroll
    for (int s = 0; s < 4; s++)
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a.h[s]), __builtin_bit_cast(f16x8, b.h[s]), c, 0,
                                                   0, 0);
    return c;
}
__device__ __forceinline__ f32x4 mul(const Operand<true>& a, const Operand<true>& b, f32x4 c) {
#pragma unroll
    for (int s = 0; s < 4; s++)
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.h[s]), __builtin_bit_cast(f16x8, b.h[s]), c, 0,
                                                   0, 0);
    return c;
}

// ---- quantisation ----

// Eight values at p as f32. DTYPE: TSFM_DTYPE_*.
template <int DTYPE>
__device__ __forceinline__ void load8(const void* x, int64_t at, float (&v)[8]) {
    if constexpr (DTYPE == 0) {
        const f32x4 a = ld4(static_cast<const float*>(x) + at), b = ld4(static_cast<const float*>(x) + at + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    } else {
        const u32x4 w = ld16(static_cast<const uint16_t*>(x) + at);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = half_to_f32<DTYPE == 1>((i & 1) ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu);
    }
}

// The largest finite magnitude of eight values.
__device__ __forceinline__ float amax8(const float (&v)[8]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float a = fabsf(v[i]);
        m = fmaxf(m, a <= kFltMax ? a : 0.f);
    }
    return m;
}
// Their codes. What is no finite number becomes a NaN (the sign kept): the conversion of a NaN.
__device__ __forceinline__ u32x2 codes8(const float (&v)[8], float mul) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = fabsf(v[i]) <= kFltMax ? v[i] * mul : __builtin_nanf("");
    return u32x2{encode4<kCodeE4m3>(y[0], y[1], y[2], y[3]), encode4<kCodeE4m3>(y[4], y[5], y[6], y[7])};
}

// Rows: 16 lanes per group of 128 values (8 each), four groups per wave. Bound by bytes.
template <int DTYPE>
__global__ __launch_bounds__(256) void quantize_rows(F8Quantize p) {
    const int groups = (p.cols - 1) / KB + 1;
    const int64_t id = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4, total = (int64_t)p.rows * groups;
    const int l = threadIdx.x & 15;
    const int64_t row = id / groups;
    const int grp = (int)(id % groups), col = grp * KB + 8 * l;
    const bool in = id < total && col < p.cols;  // cols is a multiple of 16: eight values or none
    float v[8] = {};
    if (in) load8<DTYPE>(p.x, row * p.x_ld + col, v);
    float m = amax8(v);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    float scale, mul;
    block_scale<kCodeE4m3>(m, scale, mul);
    if (in) *reinterpret_cast<u32x2*>(p.codes + row * p.codes_ld + col) = codes8(v, mul);
    if (id < total && l == 0) p.scales[row * p.scales_ld + grp] = scale;
}

// 128 x 128 tiles (weights, once): one workgroup per tile; 16 lanes per row, 16 rows at a time, read twice.
template <int DTYPE>
__global__ __launch_bounds__(256) void quantize_tiles(F8Quantize p) {
    __shared__ float s_max[4];
    const int groups = (p.cols - 1) / KB + 1;
    const int grp = blockIdx.x % groups;
    const int64_t row0 = (int64_t)(blockIdx.x / groups) * KB;
    const int l = threadIdx.x & 15, col = grp * KB + 8 * l;
    const int rows = (int)min((int64_t)KB, p.rows - row0);
    float m = 0.f, v[8];
    for (int i = threadIdx.x >> 4; i < rows; i += 16)
        if (col < p.cols) {
            load8<DTYPE>(p.x, (row0 + i) * p.x_ld + col, v);
            m = fmaxf(m, amax8(v));
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    float scale, mul;
    block_scale<kCodeE4m3>(m, scale, mul);
    for (int i = threadIdx.x >> 4; i < rows; i += 16)
        if (col < p.cols) {
            load8<DTYPE>(p.x, (row0 + i) * p.x_ld + col, v);
            *reinterpret_cast<u32x2*>(p.codes + (row0 + i) * p.codes_ld + col) = codes8(v, mul);
        }
    if (threadIdx.x == 0) p.scales[(int64_t)(blockIdx.x / groups) * p.scales_ld + grp] = scale;
}

// ---- products ----
// OUT: TSFM_DTYPE_*. One result at element `at`.
template <int OUT>
__device__ __forceinline__ void store1(void* c, int64_t at, float v) {
    if constexpr (OUT == 0) static_cast<float*>(c)[at] = v;
    else static_cast<uint16_t*>(c)[at] = (uint16_t)pack2<OUT == 1>(v, 0.f);
}

// Four consecutive results of a row at element `at`, the first `n` of them; ALIGNED: in one store.
template <int OUT>
__device__ __forceinline__ void store4(void* c, int64_t at, f32x4 v, int n, bool aligned) {
    if (n >= 4 && aligned) {
        if constexpr (OUT == 0) st4(static_cast<float*>(c) + at, v);
        else
            *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(c) + at) = u32x2{pack2<OUT == 1>(v[0], v[1]), pack2<OUT == 1>(v[2], v[3])};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < n) store1<OUT>(c, at + i, v[i]);
}

// 16 MT rows of a by 16 NT rows of b a workgroup, whose eight waves share the reduction by blocks of 128 and add up
// through LDS in order. Operands come straight from memory into registers, a block ahead: a load covers 16 rows of 64
// consecutive bytes. For few rows, bound by the bytes of b, and for products whose tiles would not fill the CUs, bound by
// latency: that of k / 1024 loads here.
constexpr int FW = 8;
template <int OUT, int MT, int NT>
__global__ __launch_bounds__(64 * FW) void gemm_few(F8Gemm p) {
    __shared__ __attribute__((aligned(16))) float part[FW][MT * NT][64][4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ql = lane & 15, g = lane >> 4;
    const int mt_n = (p.m - 1) / (16 * MT) + 1, kbs = (p.k + KB - 1) / KB;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int m0 = id % mt_n * 16 * MT, n0 = id / mt_n * 16 * NT;
    static_assert(KB % (16 * NT) == 0, "b's rows share their scales");
    const uint8_t *ra[MT], *rb[NT];
    const float* sa[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int64_t m = min(m0 + 16 * i + ql, p.m - 1);
        ra[i] = p.a + m * p.a_ld;
        sa[i] = p.a_scales + m * p.a_scales_ld;
    }
#pragma unroll
    for (int j = 0; j < NT; j++) rb[j] = p.b + (int64_t)min(n0 + 16 * j + ql, p.n - 1) * p.b_ld;
    const float* const sb = p.b_scales + (int64_t)(n0 / KB) * p.b_scales_ld;
    i32x8 a[MT], b[NT];
    float s[MT];
    auto load = [&](int kb) {  // pieces g and 4 + g of the block's 128 bytes; 0 past k
        const int k0 = kb * KB + 16 * g;
        const bool lo = k0 < p.k, hi = k0 + 64 < p.k;
        const u32x4 z = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < NT; j++) b[j] = pair(lo ? ld16(rb[j] + k0) : z, hi ? ld16(rb[j] + k0 + 64) : z);
#pragma unroll
        for (int i = 0; i < MT; i++) {
            a[i] = pair(lo ? ld16(ra[i] + k0) : z, hi ? ld16(ra[i] + k0 + 64) : z);
            s[i] = sa[i][kb] * sb[kb];
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = f32x4{0, 0, 0, 0};
    if (wave < kbs) load(wave);
    for (int kb = wave; kb < kbs; kb += FW) {
        Operand<OUT == 0> ob[NT], oa;
        i32x8 ac[MT];
        float sc[MT];
#pragma unroll
        for (int j = 0; j < NT; j++) ob[j].set(b[j]);
#pragma unroll
        for (int i = 0; i < MT; i++) {
            ac[i] = a[i];
            sc[i] = s[i];
        }
        if (kb + FW < kbs) load(kb + FW);
#pragma unroll
        for (int i = 0; i < MT; i++) {
            oa.set(ac[i]);
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const f32x4 x = mul(ob[j], oa, f32x4{0, 0, 0, 0});
#pragma unroll
                for (int r = 0; r < 4; r++) acc[i][j][r] = __builtin_fmaf(sc[i], x[r], acc[i][j][r]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) st4(part[wave][i * NT + j][lane], acc[i][j]);
    __syncthreads();
    constexpr int kElem = OUT == 0 ? 4 : 2;
    const bool aligned = p.c_ld % 4 == 0 && ((uintptr_t)p.c & (4 * kElem - 1)) == 0;
    for (int t = wave; t < MT * NT; t += FW) {
        f32x4 sum = ld4(part[0][t][lane]);
#pragma unroll
        for (int w = 1; w < FW; w++) sum += ld4(part[w][t][lane]);
        const int m = m0 + 16 * (t / NT) + ql, n = n0 + 16 * (t % NT) + 4 * g;  // the lane's results: n .. n + 3
        if (m < p.m) store4<OUT>(p.c, m * p.c_ld + n, sum, p.n - n, aligned);
    }
}

// Tiles of TM x TN, WM x WN waves, a step of 128 values at a time. Both operands go from memory into LDS by DMA
// (buffer loads whose descriptors end after the tile's rows: what is past m, n or k reads as 0), one step ahead,
// one barrier per step. LDS rows are the step's 128 bytes with their 16-byte pieces XOR-swizzled.
// A wave's tile decides what LDS has to deliver: 64 x 64 needs 128 bytes a cycle where the matrix unit is kept busy, all
// there is, 128 x 64 three quarters of it.
template <int OUT, int TM, int TN, int WM, int WN, int OCC>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(OCC, OCC))) void gemm_tiles(F8Gemm p) {
    constexpr int NWV = WM * WN, MT = TM / WM / 32, NT = TN / WN / 32;
    constexpr uint32_t kStage = (TM + TN) * KB;
    static_assert(KB % (TN / WN) == 0, "a wave's columns share their scales");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * kStage];
    __shared__ float scales[8][TN / KB][TM];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lr = lane & 31, lh = lane >> 5;
    const int mt_n = (p.m - 1) / TM + 1, nt_n = (p.n - 1) / TN + 1;
    // An XCD takes consecutive ids; they walk groups of 8 tiles of rows, so that the tiles in flight on it are about
    // as many rows as columns and share their panels in its L2.
    constexpr int GM = 8;
    int id = xcd_remap(blockIdx.x, gridDim.x);
    const int grp = id / (GM * nt_n), gm = min(GM, mt_n - grp * GM);
    id -= grp * GM * nt_n;
    const int m0 = (grp * GM + id % gm) * TM, n0 = id / gm * TN;
    const int wm = (wave % WM) * (TM / WM), wn = (wave / WM) * (TN / WN);
    const int kbs = (p.k + KB - 1) / KB;
    const int mrows = min(TM, p.m - m0), nrows = min(TN, p.n - n0);
    const u32x4 a_buf = buf_desc(p.a + (int64_t)m0 * p.a_ld, (uint32_t)((mrows - 1) * p.a_ld + p.k));
    const u32x4 b_buf = buf_desc(p.b + (int64_t)n0 * p.b_ld, (uint32_t)((nrows - 1) * p.b_ld + p.k));
    // One DMA instruction of a wave fills 1 KB: 8 rows, lane l piece l % 8 of row l / 8.
    constexpr int AI = TM / 8 / NWV, BI = TN / 8 / NWV;
    constexpr uint32_t kOutside = 0x80000000u;  // past every descriptor (the host keeps a tile's rows below 2 GiB)
    // Pieces are swizzled by half the row: 16 lanes, which LDS serves together, read two rows a bank half and eight
    // places in each. (By the row itself: every read two deep on its banks.)
    static_assert(AI % 2 == 0 && BI % 2 == 0, "the swizzle's upper bit goes by the instruction's parity");
    const int srow = lane >> 3, spiece0 = (lane & 7) ^ (srow >> 1);
    const uint32_t a_off0 = (uint32_t)(wave * AI * 8 + srow) * (uint32_t)p.a_ld;
    const uint32_t b_off0 = (uint32_t)(wave * BI * 8 + srow) * (uint32_t)p.b_ld;
    auto stage = [&](int kb, int buf) {
        const uint32_t st = lds0 + buf * kStage;
        uint32_t a_off = a_off0, b_off = b_off0, spiece = spiece0;
        asm volatile("" : "+v"(a_off), "+v"(b_off), "+v"(spiece));  // else every address is kept over the loop
#pragma unroll
        for (int i = 0; i < AI; i++) {
            const uint32_t at = 16u * (spiece ^ (4 * (i & 1)));
            dma16(a_buf, st + (wave * AI + i) * 1024,
                  kb * KB + (int)at < p.k ? a_off + (uint32_t)(8 * i) * (uint32_t)p.a_ld + at : kOutside, (uint32_t)kb * KB);
        }
#pragma unroll
        for (int i = 0; i < BI; i++) {
            const uint32_t at = 16u * (spiece ^ (4 * (i & 1)));
            dma16(b_buf, st + TM * KB + (wave * BI + i) * 1024,
                  kb * KB + (int)at < p.k ? b_off + (uint32_t)(8 * i) * (uint32_t)p.b_ld + at : kOutside, (uint32_t)kb * KB);
        }
    };
    typedef __attribute__((address_space(3))) u32x4* lds_ptr;
    // 32 bytes of a row: pieces 4 s + 2 lh and the next, at their swizzled places (the row's low bits are the lane's).
    const uint32_t sw0 = 16 * ((2 * lh) ^ ((lr >> 1) & 7)), sw1 = 16 * ((2 * lh + 1) ^ ((lr >> 1) & 7));
    auto operand = [&](uint32_t row0, int s) {
        const uint32_t r = row0 + lr * KB;
        return pair(*(lds_ptr)(uintptr_t)(r + (sw0 ^ (64 * s))), *(lds_ptr)(uintptr_t)(r + (sw1 ^ (64 * s))));
    };
    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = f32x16{};
    // The scales' products, by step, row and 128 columns, in LDS: a thread keeps one row and column group, four steps at a
    // time (16-byte loads; a load per step, wave and row asked for sixteen times as many cache lines). Steps k and k + 8
    // share a place. At step kb: fetched where kb % 4 is 0, written for the next four where it is 3; at the end some again.
    typedef f32x4 f32x4_any __attribute__((aligned(4)));
    f32x4 va = {0, 0, 0, 0}, vb = va;
    auto fetch_scales = [&](int kb) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));  // its addresses are not kept across the loop
        const int grp = tid / TM, ahead = min((kb & ~3) + 4, kbs - 4);
        if (grp >= TN / KB || (kb >= 0 && (kb | 3) + 1 >= kbs)) return;  // whole waves
        const float* const sa = p.a_scales + (int64_t)min(m0 + tid % TM, p.m - 1) * p.a_scales_ld;
        const float* const sb = p.b_scales + (int64_t)min(n0 / KB + grp, (p.n - 1) / KB) * p.b_scales_ld;
        if (kb < 0) {  // before the first step: the first four
            for (int k = 0; k < min(4, kbs); k++) scales[k][grp][tid % TM] = sa[k] * sb[k];
        } else if ((kb & 3) == 0) {
            va = *reinterpret_cast<const f32x4_any*>(sa + ahead);
            vb = *reinterpret_cast<const f32x4_any*>(sb + ahead);
        } else if ((kb & 3) == 3) {
#pragma unroll
            for (int i = 0; i < 4; i++) scales[(ahead + i) & 7][grp][tid % TM] = va[i] * vb[i];
        }
    };
    fetch_scales(-1);
    const uint32_t ra = lds0 + wm * KB, rb = lds0 + (TM + wn) * KB;
    stage(0, 0);
    if constexpr (OUT != 0) {
        // Tile by tile, the products of one issued before the multiply-adds of the one before: the vector unit works on
        // those while the matrix unit is at the next. a's operands are read a tile row ahead, the next step's first ones
        // beside the last row. The barrier stands before that row, when the wave has read all of this step's data: behind
        // it the next step's are there, and those of the step after it are sent for into this step's place (the barrier
        // between steps: 547 us where this takes 526, 16384 x 8192 x 4096). Bound by the matrix unit's share of the wave's
        // time: 64 of its cycles a product and wave, two waves a SIMD, are 43 % of it.
        static_assert(MT % 2 == 0, "a tile row's operands and the next one's alternate");
        Operand<false> a[2][2], b[NT][2];
        f32x16 x[2];
        auto read_a = [&](int i, int slot, int buf) {
#pragma unroll
            for (int h = 0; h < 2; h++) a[slot][h].set(operand(ra + buf * kStage + 32 * i * KB, h));
        };
        auto read_b = [&](int j, int buf) {
#pragma unroll
            for (int h = 0; h < 2; h++) b[j][h].set(operand(rb + buf * kStage + 32 * j * KB, h));
        };
        stage(1, 1);  // past k: zeros
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(AI + BI) : "memory");
        read_a(0, 0, 0);
#pragma unroll
        for (int j = 0; j < NT; j++) read_b(j, 0);
        for (int kb = 0; kb < kbs; kb++) {
            const int buf = kb & 1;
            fetch_scales(kb);
            float s[MT];
#pragma unroll
            for (int i = 0; i < MT; i++) s[i] = scales[kb & 7][wn / KB][wm + 32 * i + lr];
#pragma unroll
            for (int t = 0; t <= MT * NT; t++) {
                const int i = t / NT, j = t % NT;
                if (t == (MT - 1) * NT) {
                    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                    asm volatile("" : "+v"(va), "+v"(vb));  // the scales on their way, too, are there
                    stage(kb + 2, buf);
                }
                if (t < MT * NT) {
                    if (j == 0) i + 1 < MT ? read_a(i + 1, (i + 1) & 1, buf) : read_a(0, 0, buf ^ 1);
                    x[t & 1] = mul(b[j][1], a[i & 1][1], mul(b[j][0], a[i & 1][0], f32x16{}));
                    __builtin_amdgcn_sched_barrier(0);
                    if (i + 1 == MT) read_b(j, buf ^ 1);  // after the last step: nothing's
                }
                if (t > 0) {
                    const int u = t - 1;
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        acc[u / NT][u % NT][r] = __builtin_fmaf(s[u / NT], x[u & 1][r], acc[u / NT][u % NT][r]);
                }
                __builtin_amdgcn_sched_barrier(0x100);  // in this order but for the reads of LDS
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // of the zeros past k
    } else {
        for (int kb = 0; kb < kbs; kb++) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            fetch_scales(kb);  // before the copies: a wait for these would wait for those too
            if (kb + 1 < kbs) stage(kb + 1, (kb + 1) & 1);
            float s[MT];
#pragma unroll
            for (int i = 0; i < MT; i++) s[i] = scales[kb & 7][wn / KB][wm + 32 * i + lr];
            const uint32_t at = (kb & 1) * kStage;
#pragma unroll
            for (int h = 0; h < 2; h++) {  // half a step at a time: f16 operands are twice as large
                Operand<true> b[NT];
#pragma unroll
                for (int j = 0; j < NT; j++) b[j].set(operand(rb + at + 32 * j * KB, h));
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    Operand<true> a;
                    a.set(operand(ra + at + 32 * i * KB, h));
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        const f32x16 x = mul(b[j], a, f32x16{});
#pragma unroll
                        for (int r = 0; r < 16; r++) acc[i][j][r] = __builtin_fmaf(s[i], x[r], acc[i][j][r]);
                    }
                }
            }
        }
    }
    // Results: 32 rows of the wave's columns at a time through its part of LDS, so that a store writes whole lines (8 bytes
    // a row and lane straight from the registers: 80 us of 617 at 16384 x 8192 x 4096).
    constexpr int kElem = OUT == 0 ? 4 : 2, kRow = TN / WN * kElem, kPad = kRow + 16;  // bytes of a row, and in LDS
    constexpr int LR = kRow / 16, RL = 64 / LR;                                         // lanes per row, rows per store
    static_assert(32 * kPad * NWV <= (int)sizeof(smem), "a part of LDS for every wave");
    const bool whole = p.c_ld * kElem % 16 == 0 && ((uintptr_t)p.c & 15) == 0 && p.n - n0 - wn >= TN / WN;
    const bool aligned = p.c_ld % 4 == 0 && ((uintptr_t)p.c & (4 * kElem - 1)) == 0;
    asm volatile("s_barrier" ::: "memory");  // every wave has its last operands
    const uint32_t part = lds0 + wave * 32 * kPad;
    typedef __attribute__((address_space(3))) u32x2* lds8_ptr;
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int mrow = m0 + wm + 32 * i;
        if (whole) {
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const f32x16& x = acc[i][j];
                    const uint32_t at = part + lr * kPad + (32 * j + 8 * q + 4 * lh) * kElem;
                    if constexpr (OUT == 0)
                        *(lds_ptr)(uintptr_t)at = __builtin_bit_cast(u32x4, f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]});
                    else
                        *(lds8_ptr)(uintptr_t)at = u32x2{pack2<OUT == 1>(x[4 * q], x[4 * q + 1]), pack2<OUT == 1>(x[4 * q + 2], x[4 * q + 3])};
                }
#pragma unroll
            for (int t = 0; t < 32; t += RL) {
                const int row = t + lane / LR;
                const u32x4 v = *(lds_ptr)(uintptr_t)(part + row * kPad + 16 * (lane % LR));
                if (mrow + row < p.m)
                    *reinterpret_cast<u32x4*>(static_cast<char*>(p.c) + ((mrow + row) * p.c_ld + n0 + wn) * kElem + 16 * (lane % LR)) = v;
            }
            continue;
        }
        if (mrow + lr >= p.m) continue;
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int n = n0 + wn + 32 * j + 8 * q + 4 * lh;
                const f32x16& x = acc[i][j];
                store4<OUT>(p.c, (mrow + lr) * p.c_ld + n, f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]}, p.n - n, aligned);
            }
    }
}

template <int OUT, int TM, int TN, int WM, int WN, int OCC>
hipError_t tiles(const F8Gemm& p, hipStream_t s) {
    const int64_t grid = (((int64_t)p.m + TM - 1) / TM) * (((int64_t)p.n + TN - 1) / TN);
    if (grid > 0x7fffffff) return hipErrorInvalidValue;
    hipLaunchKernelGGL((gemm_tiles<OUT, TM, TN, WM, WN, OCC>), dim3((unsigned)grid), dim3(64 * WM * WN), 0, s, p);
    return hipGetLastError();
}

template <int OUT, int MT, int NT>
hipError_t few(const F8Gemm& p, hipStream_t s) {
    const int64_t grid = (((int64_t)p.m + 16 * MT - 1) / (16 * MT)) * (((int64_t)p.n + 16 * NT - 1) / (16 * NT));
    if (grid > 0x7fffffff) return hipErrorInvalidValue;
    hipLaunchKernelGGL((gemm_few<OUT, MT, NT>), dim3((unsigned)grid), dim3(64 * FW), 0, s, p);
    return hipGetLastError();
}

// gemm_few with the narrowest columns whose workgroups all run at once, one a CU; false if no width does.
template <int OUT, int MT>
bool few(const F8Gemm& p, int cus, hipStream_t s, hipError_t& err) {
    const int64_t mt = ((int64_t)p.m + 16 * MT - 1) / (16 * MT), n16 = ((int64_t)p.n + 15) / 16;
    if (mt * n16 <= cus) err = few<OUT, MT, 1>(p, s);
    else if (mt * ((n16 + 1) / 2) <= cus) err = few<OUT, MT, 2>(p, s);
    else if (MT == 1 || mt * ((n16 + 3) / 4) <= cus) err = few<OUT, MT, 4>(p, s);
    else return false;
    return true;
}

// Which kernel, measured on 256 CUs, us for m x n x k, bf16 results.
// gemm_few where its workgroups run at once: its waves split k, so that the chain of loads is an eighth as long as that
// of tiles: 64 x 2048 x 4096 14.7 against 25.0, 400 x 512 x 2048 8.5 against 14.3, 800 x 1024 x 4096 22.0 against 25.6.
// Its columns, 16 / 32 / 64: 16 x 4096 x 1024 3.3 / 3.8 / 4.7; 16 x 8192 x 2048 6.7 / 5.4 / 7.3;
// 16 x 16384 x 4096 20.2 / 15.6 / 13.2. Above that tiles read a's rows less often: 200 x 8192 x 2048 24.8 against 14.6,
// 32 x 32768 x 4096 32.0 against 26.3; 16 rows or less are so small that they do not count: 16 x 32768 x 4096 22.7
// against 25.9.
// Tiles of 256 x 256 cost 8/9 of the four of 128 x 128 that they replace (16384 x 8192 x 4096 547 against 619), but a
// last turn of few tiles costs more: the CUs' turns decide. 4096 x 4096 x 4096 71 against 81; the other way
// 2331 x 8192 x 4096 123 against 99, 6000 x 4096 x 4096 126 against 118.
template <int OUT>
hipError_t gemm(const F8Gemm& p, int cus, hipStream_t s) {
    hipError_t err = hipSuccess;
    if (p.m <= 16 && few<OUT, 1>(p, cus, s, err)) return err;
    if (p.m <= 32 && few<OUT, 2>(p, cus, s, err)) return err;
    if (few<OUT, 4>(p, cus, s, err)) return err;
    const int64_t big = (((int64_t)p.m + 255) / 256) * (((int64_t)p.n + 255) / 256);
    const int64_t mid = (((int64_t)p.m + 127) / 128) * (((int64_t)p.n + 127) / 128);
    if (32 * ((big + cus - 1) / cus) <= 9 * ((mid + cus - 1) / cus)) return tiles<OUT, 256, 256, 2, 4, 2>(p, s);
    return tiles<OUT, 128, 128, 2, 2, 2>(p, s);
}

template <int DTYPE>
hipError_t quantize(const F8Quantize& p, hipStream_t s) {
    const int64_t groups = (p.cols - 1) / KB + 1;
    if (p.group_rows == 1) {
        const int64_t grid = (p.rows * groups + 15) / 16;
        if (grid > 0x7fffffff) return hipErrorInvalidValue;
        hipLaunchKernelGGL(quantize_rows<DTYPE>, dim3((unsigned)grid), dim3(256), 0, s, p);
    } else {
        const int64_t grid = ((int64_t)p.rows + KB - 1) / KB * groups;
        if (grid > 0x7fffffff) return hipErrorInvalidValue;
        hipLaunchKernelGGL(quantize_tiles<DTYPE>, dim3((unsigned)grid), dim3(256), 0, s, p);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_f8_quantize(const F8Quantize& p, int dtype, hipStream_t s) {
    return dtype == 0 ? quantize<0>(p, s) : dtype == 1 ? quantize<1>(p, s) : quantize<2>(p, s);
}

hipError_t launch_f8_gemm(const F8Gemm& p, int out_dtype, int cus, hipStream_t s) {
    return out_dtype == 0 ? gemm<0>(p, cus, s) : out_dtype == 1 ? gemm<1>(p, cus, s) : gemm<2>(p, cus, s);
}

}  // namespace tsfm
