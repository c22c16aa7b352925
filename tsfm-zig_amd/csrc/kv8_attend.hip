// Causal attention over the paged 8-bit K/V cache on gfx950 (bf16 / f16 queries, f32 accumulation).
//
// Rows are (new token, query head of the group) pairs of one request and K/V head: all of them read the same
// keys, so a tile of rows shares each block's loads and decoding. With x = s_k scale log2(e) (q . code_k) for
// a key of a block with scales (s_k, s_v), the kernels carry
//     t = x + log2(s_v),  M = running max of t,  w = exp2(t - M) = s_v p,  O += w code_v,  l += w / s_v.
// s_k and log2(s_v) are one fused multiply-add on a score, the division one product per block and row; and since M
// follows p s_v, the weights that are rounded to 16 bits for the matrix instruction are at most 1 and lose nothing
// that counts beside the largest product of weight and value scale, whatever the blocks' scales are.
// Codes become bf16 / f16 in registers, exactly. The tail's values go in as they are (scales 1).
#include <algorithm>

#include "kv8_device.hpp"

namespace tsfm {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <bool BF16>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                       0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
}

// Keys that the rows up to token i of a request read.
__device__ __forceinline__ int keys_to(const Span& s, int i) { return max(0, s.before + i + 1); }

// Cache blocks per chunk of a row tile that reads nblk of them: the plan's, or more where that many chunks would not
// do (a context longer than the call's max_len).
__device__ __forceinline__ int chunk_blocks(const Kv8Attend& p, int nblk) {
    return max(p.chunk, (nblk + p.chunks - 1) / p.chunks);
}

// Eight dims of a row's result: to o where its keys were one chunk, else with the row's max and sum to the workspace.
template <bool BF16, int D>
__device__ __forceinline__ void store_row(const Kv8Attend& p, const Span& s, int h, int64_t row, int d0, int nchunk, int ck,
                                          float M, float L, f32x4 a0, f32x4 a1) {
    const int tok = (int)(row / p.group), hq = h * p.group + (int)(row % p.group);
    const int64_t at = s.t0 + (int64_t)tok;
    if (nchunk == 1) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
        a0 *= inv;
        a1 *= inv;
        *reinterpret_cast<u32x4*>(p.o + at * p.o_tok + hq * D + d0) = u32x4{
            pack2<BF16>(a0[0], a0[1]), pack2<BF16>(a0[2], a0[3]), pack2<BF16>(a1[0], a1[1]), pack2<BF16>(a1[2], a1[3])};
        return;
    }
    const int64_t slot = (at * p.heads + hq) * p.chunks + ck;
    float* dst = p.part + slot * D + d0;
    st4(dst, a0);
    st4(dst + 4, a1);
    if (d0 == 0)
        *reinterpret_cast<float2*>(p.part + (int64_t)p.max_tokens * p.heads * p.chunks * D + 2 * slot) = float2{M, L};
}

// ---- few rows: each wave streams whole blocks from HBM ----
// One workgroup = (request, K/V head, 16 QT rows, chunk of the keys); its four waves take blocks w, w + 4, ...
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32: a lane's 16-byte loads of K (one key, 16 dims) and V (one
// dim, 16 tokens in the operand's order) are the operands, so no block passes through LDS; only the tail's V does,
// to be transposed. A block's K is loaded again as soon as its scores are formed, its V after its products: what is
// in flight while a wave computes is the next block.
constexpr int NW = 4;

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4* lds_i16x4_ptr;
// Transposing read: each 16-lane group reads 16 dims of four rows (lane s: row s / 4, dims 4 (s % 4) .. + 3 at its
// address) and lane s gets dim s of the four.
__device__ __forceinline__ u32x2 lds_read_tr(uint32_t addr) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_ptr)(uintptr_t)addr));
}

// 16 bytes of a block; ONCE: past the caches, for a cache larger than they are.
template <bool ONCE>
__device__ __forceinline__ u32x4 ld_block(const uint8_t* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    else return ld16(p);
}

// Waves per SIMD that the few-row kernel is built for: registers of 128, 168 or 256 a wave. Measured either way: 64 dims
// at three waves 68 us where four take 63 (64 requests of up to 8192 tokens, 32 heads over 8, int8), 128 dims at three
// (two spills) 144 where two take 134 (two requests of 262144).
constexpr int few_waves(int d, int qt) { return d == 64 ? (qt == 1 ? 4 : 3) : 2; }

// The i-th request in the order in which workgroups take them; the i-th longest where the host asks for it.
__device__ __forceinline__ int nth_request(const Kv8Attend& p, int i) {
    if (!p.longest_first) return i;
    const int n = p.c.requests, lane = threadIdx.x & 63;
    const int len = lane < n ? p.c.len[lane] : INT32_MIN;
    int before = 0;
    for (int j = 0; j < n; j++) {
        const int other = __builtin_amdgcn_readlane(len, j);
        before += other > len || (other == len && j < lane);
    }
    asm volatile("" : "+v"(before));  // opaque: merged with what follows, the ranking costs the loops there registers
    return __builtin_ctzll(__ballot(lane < n && before == i));
}

template <int CODE, bool BF16, int D, int QT, bool ONCE>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(few_waves(D, QT), few_waves(D, QT)))) void attend_few(
    Kv8Attend p) {
    constexpr int R = 16 * QT;      // rows
    constexpr int KU = D / 64;      // 16-byte loads of a key's row per lane
    constexpr int DB = D / 16;      // 16-dim blocks of O
    struct Merge {
        float m[NW][R], l[NW][R];
        float o[NW][R][D + 4];
    };
    // The tail's K and V, rows of 2 D bytes whose 16-byte pieces are XOR-swizzled by row (operand reads of 16 rows and
    // transposing reads of four lie on different banks). The merge uses the same space.
    constexpr uint32_t kTail = kKvBlock * D * 2;
    __shared__ __attribute__((aligned(1024))) char lds[sizeof(Merge) > 2 * kTail ? sizeof(Merge) : 2 * kTail];
    Merge& mg = *reinterpret_cast<Merge*>(lds);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ql = lane & 15, g = lane >> 4;
    const Kv8& c = p.c;
    // Heads are dealt first, chunks last. Workgroups go to the 8 XCDs in turn: with chunks dealt first, a power of two of
    // them puts the late chunks, which only long contexts have, on the same XCDs (128 requests of up to 4096 tokens,
    // chunks of 16 blocks: 146 us, this way 120).
    int id = blockIdx.x;
    const int h = id % c.heads;
    id /= c.heads;
    const int tile0 = id % p.tiles;
    id /= p.tiles;
    const int r = nth_request(p, id % c.requests), ck = id / c.requests;
    const Span s = request_span(p.cu_tokens, c.len, r, p.max_tokens, c.width);
    const int G = p.group;
    const int64_t rows = (int64_t)s.n * G;
    const int nfull = s.total / kKvBlock;  // blocks held in 8 bits
    const int32_t* __restrict__ table = c.table + (int64_t)r * c.width;
    const int32_t early = table[min(ck * p.chunk + wave, c.width - 1)];  // the wave's first block, most likely

    for (int64_t row0 = (int64_t)tile0 * R; row0 < rows; row0 += (int64_t)p.tiles * R) {
        const int last = (int)((min(rows, row0 + R) - 1) / G);  // the tile's last token
        const int kend = keys_to(s, last), nblk = (kend + kKvBlock - 1) / kKvBlock;
        const int cb = chunk_blocks(p, nblk), nchunk = max(1, (nblk + cb - 1) / cb);
        if (ck >= nchunk) continue;
        const int b0 = ck * cb, b1 = min(nblk, b0 + cb);
        const int first_end = keys_to(s, (int)(row0 / G));  // keys every row of the tile reads
        const int bq = min(b1, nfull);  // end of the chunk's whole blocks

        u32x4 kc[4][KU], vc[DB];
        float2 sc;
        int64_t at;       // the loaded block, in (block, head) units
        int blk_next = 0;  // table entry of the block after it
        auto find = [&](int blk) {  // its place; a table entry that is no block: scales of NaN
            const bool ok = blk >= 0 && blk < c.blocks;
            at = (int64_t)(ok ? blk : 0) * c.heads + h;
            sc = reinterpret_cast<const float2*>(c.scales)[at];
            if (!ok) sc.x = __builtin_nanf("");
        };
        // A load instruction covers 1 KB of consecutive bytes: 16 rows of 64, or 8 rows of 128, for which lane bit 3 tells
        // the half of the row; take_k() then exchanges that bit with the pair of loads, so that as with 64 dims a lane
        // holds one row's pieces. (Sixteen half rows an instruction: every line asked for twice, 0.88 of the rate.)
        auto load_k = [&]() {
            const uint8_t* kb = c.k + at * kKvBlock * D + (KU == 1 ? ql * D : (ql & 7) * D + 8 * (ql & 8)) + 16 * g;
#pragma unroll
            for (int kg = 0; kg < 4; kg++)
#pragma unroll
                for (int u = 0; u < KU; u++) kc[kg][u] = ld_block<ONCE>(kb + (16 * kg + 8 * u) * D);
        };
        auto take_k = [&](int kg) {
            if constexpr (KU == 2)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    // rotations by 8 within 16 lanes: to lanes 8..15 the second load of lanes 0..7, and the other way round
                    const int a = (int)kc[kg][0][e], b = (int)kc[kg][1][e];
                    kc[kg][0][e] = (uint32_t)__builtin_amdgcn_update_dpp(a, b, 0x128, 0xf, 0xc, false);
                    kc[kg][1][e] = (uint32_t)__builtin_amdgcn_update_dpp(b, a, 0x128, 0xf, 0x3, false);
                }
        };
        auto load_v = [&]() {
            const uint8_t* vb = c.v + at * kKvBlock * D + ql * kKvBlock + 16 * g;
#pragma unroll
            for (int db = 0; db < DB; db++) vc[db] = ld_block<ONCE>(vb + 16 * db * kKvBlock);
        };
        int j = b0 + wave;
        // The tail follows the whole blocks in the deal. Its wave has it copied to LDS now, by DMA, without registers.
        constexpr int LR = D / 8, RL = 64 / LR;  // lanes per row, rows per 1 KB
        const bool has_tail = nfull >= b0 && nfull < b1 && (nfull - b0) % NW == wave;
        if (has_tail) {
            const uint32_t bytes = (uint32_t)(s.total - nfull * kKvBlock) * D * 2;  // rows past the last token read 0
            const int64_t at16 = ((int64_t)r * c.heads + h) * kKvBlock * D;
            const u32x4 kt = buf_desc(c.k_tail + at16, bytes), vt = buf_desc(c.v_tail + at16, bytes);
            const int row = lane / LR;
            const uint32_t off[2] = {(uint32_t)row * D * 2 + 16u * ((lane % LR) ^ (row & 7)),
                                     (uint32_t)row * D * 2 + 16u * ((lane % LR) ^ ((row + RL) & 7))};
#pragma unroll
            for (int i = 0; i < kKvBlock / RL; i++) {
                dma16(kt, lds0 + 1024 * i, off[i & 1], 1024 * i);
                dma16(vt, lds0 + kTail + 1024 * i, off[i & 1], 1024 * i);
            }
        }
        if (j < bq) {
            find(cb == p.chunk ? early : table[j]);
            load_k();
            load_v();
            if (j + NW < bq) blk_next = table[j + NW];
        }

        u32x4 qf[QT][2 * KU];
        int kv_end[QT];  // keys of this lane's row
#pragma unroll
        for (int qt = 0; qt < QT; qt++) {
            const int64_t row = row0 + 16 * qt + ql;
            const int tok = (int)(row / G), hq = h * G + (int)(row % G);
            kv_end[qt] = row < rows ? keys_to(s, tok) : 0;
#pragma unroll
            for (int u = 0; u < 2 * KU; u++)
                qf[qt][u] = row < rows ? ld16(p.q + (s.t0 + (int64_t)tok) * p.q_tok + hq * D + 64 * (u >> 1) + 16 * g + 8 * (u & 1))
                                       : u32x4{0, 0, 0, 0};
        }
        float m_run[QT], l_run[QT];
        f32x4 oacc[DB][QT];
#pragma unroll
        for (int qt = 0; qt < QT; qt++) {
            m_run[qt] = kNegInf;
            l_run[qt] = 0.f;
#pragma unroll
            for (int db = 0; db < DB; db++) oacc[db][qt] = f32x4{0, 0, 0, 0};
        }

        // One block's scores -> weights: t = s kx + lv, masked past the rows' keys; pf: the packed weights. bad: bits
        // 4 kg + i of the lane's keys whose V is no number.
        auto softmax = [&](f32x4 (&sa)[4][QT], float kx, float lv, int k0, bool plain, uint32_t bad, u32x4 (&pf)[2][QT]) {
            const float inv = __builtin_amdgcn_exp2f(-lv);
#pragma unroll
            for (int qt = 0; qt < QT; qt++) {
                float mloc = kNegInf;
#pragma unroll
                for (int kg = 0; kg < 4; kg++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float t = __builtin_fmaf(sa[kg][qt][i], kx, lv);
                        if (!plain) {
                            const int key = 16 * kg + 4 * g + i;
                            if (bad & (1u << (4 * kg + i))) t = __builtin_nanf("");
                            t = k0 + key < kv_end[qt] ? t : kNegInf;
                        }
                        sa[kg][qt][i] = t;
                        mloc = fmaxf(mloc, t);
                    }
                const float mn = fmaxf(max4(mloc), m_run[qt]);
                const float mu = mn == kNegInf ? 0.f : mn;
                const float alpha = __builtin_amdgcn_exp2f(m_run[qt] - mu);
                m_run[qt] = mn;
                float sum = 0.f;
#pragma unroll
                for (int kg = 0; kg < 4; kg++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float e = __builtin_amdgcn_exp2f(sa[kg][qt][i] - mu);
                        sa[kg][qt][i] = e;
                        sum += e;
                    }
                l_run[qt] = l_run[qt] * alpha + sum * inv;
#pragma unroll
                for (int db = 0; db < DB; db++) oacc[db][qt] *= alpha;
#pragma unroll
                for (int ch = 0; ch < 2; ch++) {
                    const f32x4 a = sa[2 * ch][qt], b = sa[2 * ch + 1][qt];
                    pf[ch][qt] = u32x4{pack2<BF16>(a[0], a[1]), pack2<BF16>(a[2], a[3]), pack2<BF16>(b[0], b[1]),
                                       pack2<BF16>(b[2], b[3])};
                }
            }
        };

        for (; j < bq; j += NW) {
            f32x4 sa[4][QT];
#pragma unroll
            for (int kg = 0; kg < 4; kg++) {
#pragma unroll
                for (int qt = 0; qt < QT; qt++) sa[kg][qt] = f32x4{0, 0, 0, 0};
                take_k(kg);
#pragma unroll
                for (int u = 0; u < KU; u++) {
                    const u32x4 lo = decode8<CODE, BF16>(kc[kg][u][0], kc[kg][u][1]);
                    const u32x4 hi = decode8<CODE, BF16>(kc[kg][u][2], kc[kg][u][3]);
#pragma unroll
                    for (int qt = 0; qt < QT; qt++) {
                        sa[kg][qt] = mfma16<BF16>(lo, qf[qt][2 * u], sa[kg][qt]);
                        sa[kg][qt] = mfma16<BF16>(hi, qf[qt][2 * u + 1], sa[kg][qt]);
                    }
                }
            }
            const float kx = sc.x * p.c2, lv = __builtin_amdgcn_logf(sc.y);
            const bool more = j + NW < bq;
            if (more) {
                find(blk_next);
                load_k();
                if (j + 2 * NW < bq) blk_next = table[j + 2 * NW];
            }
            u32x4 pf[2][QT];
            softmax(sa, kx, lv, j * kKvBlock, (j + 1) * kKvBlock <= first_end, 0, pf);
#pragma unroll
            for (int db = 0; db < DB; db++) {
                const u32x4 lo = decode8<CODE, BF16>(vc[db][0], vc[db][1]);
                const u32x4 hi = decode8<CODE, BF16>(vc[db][2], vc[db][3]);
#pragma unroll
                for (int qt = 0; qt < QT; qt++) {
                    oacc[db][qt] = mfma16<BF16>(lo, pf[0][qt], oacc[db][qt]);
                    oacc[db][qt] = mfma16<BF16>(hi, pf[1][qt], oacc[db][qt]);
                }
            }
            if (more) load_v();
        }
        if (has_tail) {
            // The lane's place, opaque: addresses formed from it are not kept in registers across the loop above.
            int lane_t = lane;
            asm volatile("" : "+v"(lane_t));
            const int ql = lane_t & 15, g = lane_t >> 4;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the copies; LDS that this wave alone reads: no barrier
            typedef __attribute__((address_space(3))) u32x4* lds_u32x4_ptr;
            // V's values that are no numbers become 0, and their tokens' weights NaN in the rows that see them: 0 * NaN
            // must not reach the rows that do not.
            uint64_t bad = 0;
#pragma unroll 2
            for (int i = 0; i < kKvBlock / RL; i++) {
                const uint32_t at = lds0 + kTail + 1024 * i + 16 * lane_t;
                u32x4 x = *(lds_u32x4_ptr)(uintptr_t)at;
                bool any = false;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    constexpr uint32_t ex = BF16 ? 0x7f80u : 0x7c00u;
                    const bool lo = (x[e] & ex) == ex, hi = ((x[e] >> 16) & ex) == ex;
                    any |= lo || hi;
                    if (lo) x[e] &= 0xffff0000u;
                    if (hi) x[e] &= 0xffffu;
                }
                const uint64_t m = __ballot(any);
                if (m) {
                    *(lds_u32x4_ptr)(uintptr_t)at = x;
                    for (int w = 0; w < RL; w++)
                        if ((m >> (w * LR)) & ((1ull << LR) - 1)) bad |= 1ull << (RL * i + w);
                }
            }
            f32x4 sa[4][QT];
#pragma unroll
            for (int kg = 0; kg < 4; kg++) {
                const uint32_t krow = lds0 + (16 * kg + ql) * D * 2;
#pragma unroll
                for (int qt = 0; qt < QT; qt++) sa[kg][qt] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < 2 * KU; u++) {
                    const int piece = (8 * (u >> 1) + 2 * g + (u & 1)) ^ (ql & 7);
                    const u32x4 a = *(lds_u32x4_ptr)(uintptr_t)(krow + 16 * piece);
#pragma unroll
                    for (int qt = 0; qt < QT; qt++) sa[kg][qt] = mfma16<BF16>(a, qf[qt][u], sa[kg][qt]);
                }
            }
            uint32_t mine = 0;
#pragma unroll
            for (int kg = 0; kg < 4; kg++) mine |= ((uint32_t)(bad >> (16 * kg + 4 * g)) & 15u) << (4 * kg);
            u32x4 pf[2][QT];
            softmax(sa, p.c2, 0.f, nfull * kKvBlock, false, mine, pf);
            const int vr = 4 * g + (ql >> 2);  // the lane's row of a transposing read (+ 16, 32, 48: the same swizzle)
            const uint32_t vrow = lds0 + kTail + vr * D * 2 + 8 * (ql & 1);
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int ch = 0; ch < 2; ch++) {
                    const uint32_t a = vrow + 32 * ch * D * 2 + 16 * ((2 * db + ((ql >> 1) & 1)) ^ (vr & 7));
                    const u32x2 lo = lds_read_tr(a), hi = lds_read_tr(a + 16 * D * 2);
                    const u32x4 v = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
                    for (int qt = 0; qt < QT; qt++) oacc[db][qt] = mfma16<BF16>(v, pf[ch][qt], oacc[db][qt]);
                }
        }

        // ---- merge the waves' results ----
        __syncthreads();  // the tail's rows, in the same LDS, have been read
        int tid_m = tid;  // opaque, as above
        asm volatile("" : "+v"(tid_m));
        const int ql_m = tid_m & 15, g_m = (tid_m & 63) >> 4;
#pragma unroll
        for (int qt = 0; qt < QT; qt++) {
            const float l = sum4(l_run[qt]);
            const int rr = 16 * qt + ql_m;
            if (g_m == 0) {
                mg.m[wave][rr] = m_run[qt];
                mg.l[wave][rr] = l;
            }
#pragma unroll
            for (int db = 0; db < DB; db++) st4(&mg.o[wave][rr][16 * db + 4 * g_m], oacc[db][qt]);
        }
        __syncthreads();
        constexpr int PR = D / 8;  // threads per row
        for (int i = tid_m; i < R * PR; i += 64 * NW) {
            const int rr = i / PR, d0 = 8 * (i % PR);
            const int64_t row = row0 + rr;
            if (row >= rows) continue;
            float M = kNegInf, L = 0.f;
#pragma unroll
            for (int w = 0; w < NW; w++) M = fmaxf(M, mg.m[w][rr]);
            f32x4 a0 = {0, 0, 0, 0}, a1 = a0;
#pragma unroll
            for (int w = 0; w < NW; w++) {
                // a wave without keys holds zeros at -inf; one that met a NaN holds NaN
                const float f = mg.m[w][rr] == kNegInf ? 1.f : __builtin_amdgcn_exp2f(mg.m[w][rr] - M);
                L += f * mg.l[w][rr];
                a0 += f * ld4(&mg.o[w][rr][d0]);
                a1 += f * ld4(&mg.o[w][rr][d0 + 4]);
            }
            store_row<BF16, D>(p, s, h, row, d0, nchunk, ck, M, L, a0, a1);
        }
        __syncthreads();  // the next tile's results go to the same LDS
    }
}

// ---- many rows: tiles through LDS ----
// One workgroup = (request, K/V head, 32 rows a wave, chunk of the keys), on v_mfma_f32_32x32x16. Each cache block is
// decoded once per workgroup, into LDS in the instructions' operand order; its codes are loaded a block earlier. Lane l of
// a score block holds one row (l % 32) and keys 8 (i / 4) + 4 (l / 32) + i % 4, i < 16: the order in which V's operand takes
// them, so the weights go from the scores' registers straight into the second product.
// A step computes the next block's scores beside this block's exponentials, and this block's second product beside the
// decoding, one product and a few vector instructions at a time, its operands read from LDS a product ahead (products and
// vector work one after the other, operands read where they were needed: 555 us where this took 473, four requests of up
// to 2048 new tokens over 8192, 32 heads of 128 dims, 8 in the cache; 494 GFLOP). Bound by the issue of two waves a SIMD:
// each unit is busy 40 to 45 % of the time; without the exponentials it takes 7 % less,
// without the decoding 14 %, without half of the products 18 %.
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <bool BF16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Waves: 8 at 128 dims, one workgroup a CU, decode a block for 256 rows (4: 505 us where these take 485). At 64 dims 4,
// with two workgroups a CU and 256 registers a lane (three and 168: 281 us where these take 214, 16 requests of 128
// tokens and 16 heads over up to 4096).
constexpr int many_waves(int d) { return d == 64 ? 4 : 8; }
// The running max follows a block's only when it is passed by this much (exp2 units): weights up to 2^8 cost nothing,
// and O is rescaled a few times per row instead of in every block.
constexpr float kSlack = 8.f;

template <int CODE, bool BF16, int D>
__global__ __launch_bounds__(64 * many_waves(D)) __attribute__((amdgpu_waves_per_eu(2, 2))) void attend_many(Kv8Attend p) {
    constexpr int MW = many_waves(D), MROWS = 32 * MW;
    constexpr int KS = D / 16;  // 16-dim steps of a score
    constexpr int DB = D / 32;  // 32-dim blocks of O
    constexpr int U = D / 16 / MW;        // 16-byte pieces of K, and of V, per thread and block
    static_assert(U * MW * 16 == D, "every thread stages as much");
    constexpr int PS = DB / U;            // a piece of the staging goes with every PS-th of the second products
    // Operand blocks of 1 KB (lane l's 16 bytes at 16 l). K: (32 keys, 16-dim step); V: (16 keys, 32 dims).
    constexpr uint32_t kOp = 1024 + 128;  // 128 bytes apart: a staging wave's pieces of two steps lie on different banks
    constexpr uint32_t kK = 2 * KS * kOp, kStage = kK + 4 * DB * kOp;
    __shared__ __attribute__((aligned(1024))) char lds[2 * kStage];
    __shared__ unsigned long long bad_keys;
    typedef __attribute__((address_space(3))) u32x4* lds_u32x4_ptr;
    typedef __attribute__((address_space(3))) u32x2* lds_u32x2_ptr;
    typedef __attribute__((address_space(3))) uint16_t* lds_u16_ptr;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lq = lane & 31, lh = lane >> 5;
    const Kv8& c = p.c;
    // Row tiles of one (request, head, chunk) read the same keys: on one XCD, whose L2 then holds them. Workgroups go to
    // the 8 XCDs in turn, and the triples are dealt to XCDs in turn too, heads first: every XCD has its share of each
    // request, however their lengths differ (requests dealt to XCDs whole: 999 us where this took 581). Late tiles,
    // which read the most keys, first.
    const int idx = blockIdx.x >> 3;
    const int tile0 = p.tiles - 1 - idx % p.tiles;
    int id = idx / p.tiles * 8 + (blockIdx.x & 7);
    const int h = id % c.heads;
    id /= c.heads;
    const int ck = id / c.requests;
    if (ck >= p.chunks) return;
    const int r = nth_request(p, id % c.requests);
    const Span s = request_span(p.cu_tokens, c.len, r, p.max_tokens, c.width);
    const int G = p.group;
    const int64_t rows = (int64_t)s.n * G;
    const int nfull = s.total / kKvBlock;
    const int32_t* __restrict__ table = c.table + (int64_t)r * c.width;

    for (int64_t row0 = (int64_t)tile0 * MROWS; row0 < rows; row0 += (int64_t)p.tiles * MROWS) {
        const int last = (int)((min(rows, row0 + MROWS) - 1) / G);
        const int kend = keys_to(s, last), nblk = (kend + kKvBlock - 1) / kKvBlock;
        const int cb = chunk_blocks(p, nblk), nchunk = max(1, (nblk + cb - 1) / cb);
        if (ck >= nchunk) continue;
        const int b0 = ck * cb, b1 = min(nblk, b0 + cb);
        const int bq = min(b1, nfull);  // end of the chunk's whole blocks

        // ---- this wave's rows ----
        const int64_t wrow = row0 + 32 * wave, row = wrow + lq;
        const int tok = (int)(min(row, rows - 1) / G), hq = h * G + (int)(min(row, rows - 1) % G);
        const int kv_end = row < rows ? keys_to(s, tok) : 0;                                        // keys of the lane's row
        const int plain_end = wrow < rows ? keys_to(s, (int)(wrow / G)) : 0;                        // of all the wave's rows
        u32x4 qf[KS];
#pragma unroll
        for (int t = 0; t < KS; t++)
            qf[t] = row < rows ? ld16(p.q + (s.t0 + (int64_t)tok) * p.q_tok + hq * D + 16 * t + 8 * lh) : u32x4{0, 0, 0, 0};
        f32x16 oacc[DB];
#pragma unroll
        for (int db = 0; db < DB; db++) oacc[db] = f32x16{};
        float m_run = kNegInf, l_run = 0.f;

        // ---- staging ----
        // K: a wave's load covers 1 KB: 16 keys of 64 dims (lane: key l % 16, step l / 16) or 8 keys of 128 (key l % 8,
        // step l / 8). V: the thread's dim and 16-byte piece g of its tokens.
        u32x4 kc[U], vc[U];
        auto base = [&](int blk) { return ((int64_t)blk * c.heads + h) * kKvBlock * D; };
        auto load_k = [&](int blk, int u) {
            const int key = D == 64 ? 16 * (U * wave + u) + (lane & 15) : 8 * (U * wave + u) + (lane & 7);
            kc[u] = ld16(c.k + base(blk) + key * D + 16 * (D == 64 ? lane >> 4 : lane >> 3));
        };
        auto load_v = [&](int blk, int u) {
            vc[u] = ld16(c.v + base(blk) + (16 * (U * wave + u) + (lane & 15)) * kKvBlock + 16 * (lane >> 4));
        };
        auto stage_k = [&](int buf, int u, int half) {
            const int key = D == 64 ? 16 * (U * wave + u) + (lane & 15) : 8 * (U * wave + u) + (lane & 7);
            const int step = D == 64 ? lane >> 4 : lane >> 3;
            const uint32_t a = lds0 + buf * kStage + ((key >> 5) * KS + step) * kOp + 16 * (key & 31);
            *(lds_u32x4_ptr)(uintptr_t)(a + 512 * half) = decode8<CODE, BF16>(kc[u][2 * half], kc[u][2 * half + 1]);
        };
        auto stage_v = [&](int buf, int u, int half) {
            // Words (c2, a2) of piece g are tokens 16 (2 c2 + a2) + 4 g .. + 3: four of the operand's eight slots.
            const int dim = 16 * (U * wave + u) + (lane & 15), g = lane >> 4;
            const uint32_t b = lds0 + buf * kStage + kK + (dim >> 5) * kOp + 16 * (32 * (g & 1) + (dim & 31)) + 8 * (g >> 1);
            const u32x4 x = decode8<CODE, BF16>(vc[u][2 * half], vc[u][2 * half + 1]);
            *(lds_u32x2_ptr)(uintptr_t)(b + 2 * half * DB * kOp) = u32x2{x[0], x[1]};
            *(lds_u32x2_ptr)(uintptr_t)(b + (2 * half + 1) * DB * kOp) = u32x2{x[2], x[3]};
        };
        // The tail's values as they are; rows past the last token 0. V's that are no numbers: 0, and their keys noted.
        auto tail_k = [&](int buf) {
            int tid_t = tid;  // opaque: its addresses are not kept across the loop
            asm volatile("" : "+v"(tid_t));
            const int live = s.total - nfull * kKvBlock;
            const int64_t at = ((int64_t)r * c.heads + h) * kKvBlock * D;
#pragma unroll 1
            for (int i = tid_t; i < kKvBlock * D / 8; i += 64 * MW) {
                const int key = i / (D / 8), d0 = 8 * (i % (D / 8));
                *(lds_u32x4_ptr)(uintptr_t)(lds0 + buf * kStage + ((key >> 5) * KS + (d0 >> 4)) * kOp +
                                            16 * (32 * ((d0 >> 3) & 1) + (key & 31))) =
                    key < live ? ld16(c.k_tail + at + key * D + d0) : u32x4{0, 0, 0, 0};
            }
        };
        auto tail_v = [&](int buf) {
            int tid_t = tid;
            asm volatile("" : "+v"(tid_t));
            const int live = s.total - nfull * kKvBlock;
            const int64_t at = ((int64_t)r * c.heads + h) * kKvBlock * D;
#pragma unroll 1
            for (int i = tid_t; i < kKvBlock * D / 8; i += 64 * MW) {
                const int key = i / (D / 8), d0 = 8 * (i % (D / 8));
                const u32x4 y = key < live ? ld16(c.v_tail + at + key * D + d0) : u32x4{0, 0, 0, 0};
                const int slot = key & 15;  // of its 16 keys: lane half (slot / 4) % 2, element 4 (slot / 8) + slot % 4
                const uint32_t b = lds0 + buf * kStage + kK + ((key >> 4) * DB + (d0 >> 5)) * kOp +
                                   16 * (32 * ((slot >> 2) & 1) + (d0 & 31)) + 2 * (4 * (slot >> 3) + (slot & 3));
                bool any = false;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    constexpr uint32_t ex = BF16 ? 0x7f80u : 0x7c00u;
                    uint32_t v = (e & 1) ? y[e >> 1] >> 16 : y[e >> 1] & 0xffffu;
                    if ((v & ex) == ex) {
                        any = true;
                        v = 0;
                    }
                    *(lds_u16_ptr)(uintptr_t)(b + 16 * e) = (uint16_t)v;
                }
                if (any) atomicOr(&bad_keys, 1ull << key);
            }
        };

        // ---- the blocks, one score product ahead ----
        // K of block j is in buffer j - b0, V too, both mod 2. At the start of step j: K up to block j + 1 and V up to j in
        // LDS, block j + 2's K codes and j + 1's V codes in registers. Past the last whole block old codes are staged again,
        // which nothing reads: the step stays free of branches.
        // Table entries and scales of 64 blocks at a time, a block per lane; a step takes its own from there.
        struct Block {
            int id;
            float sk, sv;
        };
        int lane_id = 0;
        f32x2 lane_s = {0, 0};
        auto block = [&](int x) {  // the chunk's x-th; the last whole one past the end
            if ((x & 63) == 0) {
                const int blk = table[max(0, min(b0 + x + lane, bq - 1))];
                const bool ok = blk >= 0 && blk < c.blocks;
                lane_id = ok ? blk : 0;
                lane_s = ld2(c.scales + 2 * ((int64_t)lane_id * c.heads + h));
                if (!ok) lane_s[0] = __builtin_nanf("");
                float sk = lane_s[0], sv = lane_s[1];
                asm volatile("" : "+v"(sk), "+v"(sv));  // waited for here, not with the codes' loads behind the branch
                lane_s = f32x2{sk, sv};
            }
            return Block{__builtin_amdgcn_readlane(lane_id, x & 63),
                         __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lane_s[0]), x & 63)),
                         __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lane_s[1]), x & 63))};
        };
        auto operand = [&](int buf, int i) { return *(lds_u32x4_ptr)(uintptr_t)(lds0 + buf * kStage + 16 * lane + i * kOp); };
        Block n0 = block(0), n1 = block(1), n2 = block(2), n3 = block(3);  // blocks j .. j + 3
#pragma unroll
        for (int u = 0; u < U; u++) {
            load_k(n0.id, u);
            load_v(n0.id, u);
        }
        if (tid == 0) bad_keys = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            stage_k(0, u, 0);
            stage_k(0, u, 1);
            load_k(n1.id, u);
            stage_v(0, u, 0);
            stage_v(0, u, 1);
            load_v(n1.id, u);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            stage_k(1, u, 0);
            stage_k(1, u, 1);
            load_k(n2.id, u);
        }
        __syncthreads();
        if (b0 >= nfull) {
            tail_k(0);
            __syncthreads();
        }
        f32x16 s_even[2], s_odd[2];
#pragma unroll
        for (int t = 0; t < KS; t++)
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
                s_even[kb] = mfma32<BF16>(operand(0, kb * KS + t), qf[t], t == 0 ? f32x16{} : s_even[kb]);
        __syncthreads();  // block b0's K is overwritten in the first step

        float mx[2];  // of the scores' products, as they are: half a row's keys each
        auto top = [&](f32x16 (&sb)[2], int first, int end) {
#pragma unroll
            for (int i = first; i < end; i++) {
                mx[0] = i ? fmaxf(mx[0], sb[0][i]) : sb[0][0];
                mx[1] = i ? fmaxf(mx[1], sb[1][i]) : sb[1][0];
            }
        };
        top(s_even, 0, 16);

        auto step = [&](int j, int buf, f32x16 (&sb)[2], f32x16 (&next)[2]) {
            const bool tail = j >= nfull;
            if (j + 1 == nfull || tail) {  // the tail is the last block there is
                if (tail) tail_v(buf);
                else if (j + 1 < b1) tail_k(buf ^ 1);
                __syncthreads();
            }
            u32x4 kop[2] = {operand(buf ^ 1, 0), operand(buf ^ 1, KS)}, vop[DB];  // read a group of products ahead
            float kx = tail ? p.c2 : n0.sk * p.c2, lv = tail ? 0.f : __builtin_amdgcn_logf(n0.sv);
            const float inv_v = __builtin_amdgcn_exp2f(-lv);
            if ((j + 1) * kKvBlock > plain_end) {
                const int rel = kv_end - j * kKvBlock - 4 * lh;  // register i's key is seen where its offset is below
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float t = __builtin_fmaf(sb[kb][i], kx, lv);
                        sb[kb][i] = 32 * kb + 8 * (i >> 2) + (i & 3) < rel ? t : kNegInf;
                    }
                kx = 1.f;  // already applied
                lv = 0.f;
                if (tail && bad_keys != 0) {  // rows that see a key whose V is no number
#pragma unroll
                    for (int kb = 0; kb < 2; kb++) {
                        const uint32_t w = (uint32_t)(bad_keys >> (32 * kb)) >> (4 * lh);
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if ((w & (1u << (8 * (i >> 2) + (i & 3)))) && sb[kb][i] != kNegInf) sb[kb][i] = __builtin_nanf("");
                    }
                }
                top(sb, 0, 16);
            }
            float mloc = __builtin_fmaf(fmaxf(mx[0], mx[1]), kx, lv);
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mloc), __float_as_uint(mloc), false, false);
            mloc = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
            // O follows the max rarely. The loop of at most one turn keeps its registers: around a branch the compiler holds O
            // twice and copies it in every block, which costs what scaling it every time does.
            int turns = __builtin_amdgcn_readfirstlane(__ballot(mloc > m_run + kSlack || (m_run == kNegInf && mloc > kNegInf)) != 0);
            asm volatile("" : "+s"(turns));
#pragma clang loop unroll(disable)
            for (; turns > 0; turns--) {
                const float mn = fmaxf(m_run, mloc);
                const float alpha = __builtin_amdgcn_exp2f(m_run - (mn == kNegInf ? 0.f : mn));
                m_run = mn;
                l_run *= alpha;
#pragma unroll
                for (int db = 0; db < DB; db++) oacc[db] *= alpha;
            }
            const float off = lv - (m_run == kNegInf ? 0.f : m_run);
            u32x4 pf[4];
            // Exponentials in a row, G pairs of them after every second product, and what they need and feed after the others
            // (alternating with multiply-adds an exponential takes 16 cycles, in a row 9; one at a time this kernel took the
            // same, 482 us).
            constexpr int G = 16 / KS;
            float sum[2] = {0.f, 0.f}, w[2][2 * G];
            auto add = [&](int g) {
#pragma unroll
                for (int e = 0; e < G; e++) {
                    const float e0 = w[g & 1][2 * e], e1 = w[g & 1][2 * e + 1];
                    sum[0] += e0;
                    sum[1] += e1;
                    pf[(g * G + e) >> 2][(g * G + e) & 3] = pack2<BF16>(e0, e1);
                }
            };
#pragma unroll
            for (int n = 0; n < 2 * KS; n++) {
                const int t = n >> 1, kb = n & 1;
                next[kb] = mfma32<BF16>(kop[kb], qf[t], t == 0 ? f32x16{} : next[kb]);
                if (t + 1 < KS) kop[kb] = operand(buf ^ 1, kb * KS + t + 1);
                if (n + 1 == 2 * KS)
#pragma unroll
                    for (int db = 0; db < DB; db++) vop[db] = operand(buf, 2 * KS + db);
                __builtin_amdgcn_sched_barrier(0);
                if (kb == 0 && t > 0) add(t - 1);
#pragma unroll
                for (int e = 0; e < 2 * G; e++) {
                    const int x = 2 * G * t + e;
                    w[t & 1][e] = kb == 0 ? __builtin_fmaf(sb[x >> 4][x & 15], kx, off) : __builtin_amdgcn_exp2f(w[t & 1][e]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            add(KS - 1);
            l_run = __builtin_fmaf(sum[0] + sum[1], inv_v, l_run);
#pragma unroll
            for (int n = 0; n < 4 * DB; n++) {
                const int q = n / DB, db = n % DB;
                oacc[db] = mfma32<BF16>(vop[db], pf[q], oacc[db]);
                if (q < 3) vop[db] = operand(buf, 2 * KS + (q + 1) * DB + db);
                __builtin_amdgcn_sched_barrier(0);
                if (n & 1) {
                    top(next, 8 / DB * (n >> 1), 8 / DB * (n >> 1) + 8 / DB);
                    asm volatile("" : "+v"(mx[0]), "+v"(mx[1]));  // here, not at its use
                } else if (n % PS == 0) {
                    const int i = n / PS, u = i >> 2, half = i & 1;
                    if (i & 2) stage_v(buf ^ 1, u, half);
                    else stage_k(buf, u, half);
                    if (half == 1) {
                        if (i & 2) load_v(n2.id, u);
                        else load_k(n3.id, u);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            n0 = n1;
            n1 = n2;
            n2 = n3;
            n3 = block(j + 4 - b0);
            __syncthreads();
        };
        for (int j = b0; j < b1; j += 2) {
            step(j, 0, s_even, s_odd);
            if (j + 1 == b1) break;
            step(j + 1, 1, s_odd, s_even);
        }

        // ---- results ----
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
        const float L = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
        if (row < rows) {
            const int64_t at = s.t0 + (int64_t)tok;
            if (nchunk == 1) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
                uint16_t* dst = p.o + at * p.o_tok + hq * D + 4 * lh;
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        *reinterpret_cast<u32x2*>(dst + 32 * db + 8 * q) =
                            u32x2{pack2<BF16>(oacc[db][4 * q] * inv, oacc[db][4 * q + 1] * inv),
                                  pack2<BF16>(oacc[db][4 * q + 2] * inv, oacc[db][4 * q + 3] * inv)};
            } else {
                const int64_t slot = (at * p.heads + hq) * p.chunks + ck;
                float* dst = p.part + slot * D + 4 * lh;
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        st4(dst + 32 * db + 8 * q,
                            f32x4{oacc[db][4 * q], oacc[db][4 * q + 1], oacc[db][4 * q + 2], oacc[db][4 * q + 3]});
                if (lh == 0)
                    *reinterpret_cast<float2*>(p.part + (int64_t)p.max_tokens * p.heads * p.chunks * D + 2 * slot) =
                        float2{m_run, L};
            }
        }
    }
}

// ---- joining the chunks ----
// WPR waves per row of o, each taking its share of the row's chunks, eight loads in flight, and adding up in order: four
// for the many chunks of few rows, one otherwise.
template <bool BF16, int D, int WPR>
__global__ __launch_bounds__(256) void attend_join(Kv8Attend p) {
    __shared__ float s_l[4], s_o[4][D];
    const int lane = threadIdx.x & 63, wave = WPR == 1 ? 0 : threadIdx.x >> 6;
    const int64_t id = WPR == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (id >= (int64_t)p.max_tokens * p.heads) return;
    const int t = (int)(id / p.heads), hq = (int)(id % p.heads);
    const Kv8& c = p.c;
    // The token's request: t itself where every request has one token, else the last r with cu[r] <= t.
    int r = min(t, c.requests - 1);
    if (!(p.cu_tokens[r] <= t && t < p.cu_tokens[r + 1])) {
        int lo = 0, hi = c.requests;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (p.cu_tokens[mid + 1] <= t) lo = mid + 1;
            else hi = mid;
        }
        r = lo;
        if (r >= c.requests) return;  // behind the last token
    }
    const Span s = request_span(p.cu_tokens, c.len, r, p.max_tokens, c.width);
    const int i = t - s.t0;
    if (i < 0 || i >= s.n) return;
    // The tile that held this row decided whether its result was split.
    const int64_t rows = (int64_t)s.n * p.group, row = (int64_t)i * p.group + hq % p.group;
    const int64_t tile_end = min(rows, (row / p.rows + 1) * p.rows);
    const int kend = keys_to(s, (int)((tile_end - 1) / p.group));
    const int nblk = (kend + kKvBlock - 1) / kKvBlock, cb = chunk_blocks(p, nblk);
    const int n = max(1, (nblk + cb - 1) / cb);
    if (n == 1) return;
    const int64_t slot = ((int64_t)t * p.heads + hq) * p.chunks;
    const float2* __restrict__ ml = reinterpret_cast<const float2*>(p.part + (int64_t)p.max_tokens * p.heads * p.chunks * D) + slot;
    const float* __restrict__ part = p.part + slot * D;
    float M = kNegInf;
    for (int k = lane; k < n; k += 64) M = fmaxf(M, ml[k].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    float L = 0.f;
    constexpr int E = D / 64;
    float acc[E] = {};
    const int k0 = n * wave / WPR, k1 = n * (wave + 1) / WPR;
#pragma unroll 8
    for (int k = k0; k < k1; k++) {
        const float2 x = ml[k];
        const float f = x.x == kNegInf ? 1.f : __builtin_amdgcn_exp2f(x.x - M);
        L += f * x.y;
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] += f * part[(int64_t)k * D + E * lane + e];
    }
    if constexpr (WPR > 1) {
#pragma unroll
        for (int e = 0; e < E; e++) s_o[wave][E * lane + e] = acc[e];
        if (lane == 0) s_l[wave] = L;
        __syncthreads();
        if (wave) return;
        L = ((s_l[0] + s_l[1]) + s_l[2]) + s_l[3];
#pragma unroll
        for (int e = 0; e < E; e++)
            acc[e] = ((s_o[0][E * lane + e] + s_o[1][E * lane + e]) + s_o[2][E * lane + e]) + s_o[3][E * lane + e];
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < E; e++) acc[e] *= inv;
    uint16_t* dst = p.o + (int64_t)t * p.o_tok + hq * D + E * lane;
    if constexpr (E == 1) *dst = (uint16_t)pack2<BF16>(acc[0], 0.f);
    else *reinterpret_cast<uint32_t*>(dst) = pack2<BF16>(acc[0], acc[1]);
}

template <int CODE, bool BF16, int D>
hipError_t attend(const Kv8Attend& p, hipStream_t s) {
    const int64_t grid = (int64_t)p.c.requests * p.c.heads * p.tiles * p.chunks;
    if (grid <= 0 || grid > 0x7fffffff) return hipErrorInvalidValue;
    const dim3 g((unsigned)grid), b(64 * NW);
    if (p.kernel == kAttendMany) {
        const int64_t eights = ((int64_t)p.c.requests * p.c.heads * p.chunks + 7) / 8;  // of (request, head, chunk)
        hipLaunchKernelGGL((attend_many<CODE, BF16, D>), dim3((unsigned)(eights * 8 * p.tiles)), dim3(64 * many_waves(D)), 0, s, p);
    }
    else if (p.rows == 16 && p.once) hipLaunchKernelGGL((attend_few<CODE, BF16, D, 1, true>), g, b, 0, s, p);
    else if (p.rows == 16) hipLaunchKernelGGL((attend_few<CODE, BF16, D, 1, false>), g, b, 0, s, p);
    else if (p.once) hipLaunchKernelGGL((attend_few<CODE, BF16, D, 2, true>), g, b, 0, s, p);
    else hipLaunchKernelGGL((attend_few<CODE, BF16, D, 2, false>), g, b, 0, s, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.chunks == 1) return e;
    const int64_t rows = (int64_t)p.max_tokens * p.heads;
    if (p.chunks <= 8)
        hipLaunchKernelGGL((attend_join<BF16, D, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((attend_join<BF16, D, 4>), dim3((unsigned)rows), dim3(256), 0, s, p);
    return hipGetLastError();
}

template <int CODE, bool BF16>
hipError_t attend_d(const Kv8Attend& p, int head_dim, hipStream_t s) {
    return head_dim == 64 ? attend<CODE, BF16, 64>(p, s) : attend<CODE, BF16, 128>(p, s);
}

}  // namespace

int64_t kv8_attend_plan(Kv8Attend& p, int head_dim, int max_new, int max_len, int cus) {
    const int64_t most = (int64_t)p.c.width * kKvBlock;
    const int64_t len = max_len > 0 && max_len < most ? max_len : most;
    const int64_t fresh = max_new > 0 && max_new < p.max_tokens ? max_new : p.max_tokens;
    const int64_t rows = fresh * p.group;
    // Whole tiles through LDS pay where there are many rows to share a block's decoding (us, tiles of 128 or 256 rows / of
    // 32; four requests of up to 4096 tokens, 64 dims: 512 rows 59 / 40, 1024 58 / 65, 2048 81 / 103; 128 dims 48 / 42,
    // 74 / 67, 107 / 122; one request 1024 rows 44 / 35 and 37 / 42, 16 173 / 162 and 190 / 171; 1200 rows over 20000 tokens
    // 123 / 219; four prompts of up to 8192 rows over 8192 tokens 473 / 749).
    p.kernel = rows <= 1024 ? kAttendFew : kAttendMany;
    p.rows = p.kernel == kAttendMany ? 32 * many_waves(head_dim) : rows <= 16 ? 16 : 32;
    // A cache too large to stay in the last-level cache is read past it: loads marked as used once (545 MB of K and V 106 ->
    // 96 us; the other way, 69 MB 20.0 -> 20.4 and 34 MB in blocks of 32 tokens 29.7 -> 33.8).
    p.once = (int64_t)p.c.requests * len * p.c.heads * head_dim >= (int64_t)256 << 20;
    const int64_t tiles = (rows + p.rows - 1) / p.rows;
    p.tiles = (int32_t)(tiles < 1024 ? tiles : 1024);
    const int64_t blocks = (len + kKvBlock - 1) / kKvBlock;
    const int64_t base = (int64_t)p.c.requests * p.c.heads * p.tiles;
    // Split the keys while the workgroups fit the CUs at once: a second round of shorter ones costs more than it fills
    // (two requests of 262144 tokens, 8 heads of 128: 384 workgroups 134 us, 768 147, 1536 163; 32 requests of up to
    // 2048 tokens, 16 heads of 64: unsplit 18.3 us, in two with the join 20.2). Chunks are 8 to 128 blocks: shorter ones
    // are all start and merge, and a longer one would keep a single workgroup busy after the others.
    const int64_t resident = (int64_t)cus * (p.kernel == kAttendMany ? head_dim == 64 ? 2 : 1 : few_waves(head_dim, p.rows / 16));
    const int64_t chunks_wanted = std::max<int64_t>(1, resident / base);
    const int64_t chunk = std::min<int64_t>(128, std::max<int64_t>(8, (blocks + chunks_wanted - 1) / chunks_wanted));
    const int64_t chunks = (blocks + chunk - 1) / chunk;
    p.chunk = (int32_t)chunk;
    p.chunks = (int32_t)chunks;
    // Where workgroups fill the CUs, the long requests first leave short ones for the end (16 requests of up to 4096
    // tokens, 128 dims: 128 rows 55 -> 46 us, 1024 171 -> 157, 2048 250 -> 200; four of up to 2048 new over 8192 486 ->
    // 471; the other way four, 512 rows 41.8 -> 44.1). With room left the ranking only costs (32 requests of one token 20.8
    // -> 21.4), and of more than 32 requests the last ones weigh little (64, 2048 rows: 727 -> 739).
    p.longest_first = p.c.requests > 1 && p.c.requests <= 32 && base * chunks >= resident;
    if ((base + 8 * p.tiles) * chunks > INT32_MAX || (int64_t)p.max_tokens * p.heads > INT32_MAX) return -1;
    return chunks == 1 ? 0 : (int64_t)p.max_tokens * p.heads * chunks * (head_dim + 2) * 4;
}

hipError_t launch_kv8_attend(const Kv8Attend& p, int code, bool bf16, int head_dim, hipStream_t s) {
    if (code == kCodeE4m3) return bf16 ? attend_d<kCodeE4m3, true>(p, head_dim, s) : attend_d<kCodeE4m3, false>(p, head_dim, s);
    return bf16 ? attend_d<kCodeI8, true>(p, head_dim, s) : attend_d<kCodeI8, false>(p, head_dim, s);
}

}  // namespace tsfm
