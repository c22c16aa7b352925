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

// ---- few rows: each wave streams whole blocks from HBM ----
// One workgroup = (request, K/V head, 16 QT rows, chunk of the keys); its four waves take blocks w, w + 4, ...
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32: a lane's 16-byte loads of K (one key, 16 dims) and V (one
// dim, 16 tokens in the operand's order) are the operands, so nothing passes through LDS until the waves' results
// are merged. Bound by HBM.
constexpr int NW = 4;

template <int CODE, bool BF16, int D, int QT>
__global__ __launch_bounds__(64 * NW) void attend_few(Kv8Attend p) {
    constexpr int R = 16 * QT;      // rows
    constexpr int KU = D / 64;      // 16-byte loads of a key's row per lane
    constexpr int DB = D / 16;      // 16-dim blocks of O
    struct Merge {
        float m[NW][R], l[NW][R];
        float o[NW][R][D + 4];
    };
    __shared__ Merge mg;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int ql = lane & 15, g = lane >> 4;
    const Kv8& c = p.c;
    int id = blockIdx.x;
    const int ck = id % p.chunks;
    id /= p.chunks;
    const int tile0 = id % p.tiles;
    id /= p.tiles;
    const int h = id % c.heads, r = id / c.heads;
    const Span s = request_span(p.cu_tokens, c.len, r, p.max_tokens, c.width);
    const int G = p.group;
    const int64_t rows = (int64_t)s.n * G;
    const int nfull = s.total / kKvBlock;  // blocks held in 8 bits

    for (int64_t row0 = (int64_t)tile0 * R; row0 < rows; row0 += (int64_t)p.tiles * R) {
        const int last = (int)((min(rows, row0 + R) - 1) / G);  // the tile's last token
        const int kend = keys_to(s, last), nblk = (kend + kKvBlock - 1) / kKvBlock;
        const int cb = chunk_blocks(p, nblk), nchunk = max(1, (nblk + cb - 1) / cb);
        if (ck >= nchunk) continue;
        const int b0 = ck * cb, b1 = min(nblk, b0 + cb);
        const int first_end = keys_to(s, (int)(row0 / G));  // keys every row of the tile reads

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

        u32x4 kc[4][KU], vc[DB];
        float2 sc;
        auto load = [&](int j) {  // block j of the request (a whole one)
            const int blk = c.table[(int64_t)r * c.width + j];
            const bool ok = blk >= 0 && blk < c.blocks;
            const int64_t at = (int64_t)(ok ? blk : 0) * c.heads + h;
            const uint8_t* kb = c.k + at * kKvBlock * D;
            const uint8_t* vb = c.v + at * kKvBlock * D;
            sc = reinterpret_cast<const float2*>(c.scales)[at];
            if (!ok) sc.x = __builtin_nanf("");
#pragma unroll
            for (int kg = 0; kg < 4; kg++)
#pragma unroll
                for (int u = 0; u < KU; u++) kc[kg][u] = ld16(kb + (16 * kg + ql) * D + 64 * u + 16 * g);
#pragma unroll
            for (int db = 0; db < DB; db++) vc[db] = ld16(vb + (16 * db + ql) * kKvBlock + 16 * g);
        };
        // One block's scores -> weights: t = s kx + lv, masked past the rows' keys; pf: the packed weights.
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
                        const int key = k0 + 16 * kg + 4 * g + i;
                        if (!plain) t = key < kv_end[qt] ? ((bad >> (4 * kg + i)) & 1 ? __builtin_nanf("") : t) : kNegInf;
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

        const int bq = min(b1, nfull);  // whole blocks of the chunk
        int j = b0 + wave;
        if (j < bq) load(j);
        for (; j < bq; j += NW) {
            f32x4 sa[4][QT];
#pragma unroll
            for (int kg = 0; kg < 4; kg++) {
#pragma unroll
                for (int qt = 0; qt < QT; qt++) sa[kg][qt] = f32x4{0, 0, 0, 0};
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
            u32x4 pf[2][QT], vd[DB];
            softmax(sa, sc.x * p.c2, __builtin_amdgcn_logf(sc.y), j * kKvBlock, (j + 1) * kKvBlock <= first_end, 0u, pf);
#pragma unroll
            for (int db = 0; db < DB; db++) vd[db] = vc[db];
            if (j + NW < bq) load(j + NW);
#pragma unroll
            for (int db = 0; db < DB; db++) {
                const u32x4 lo = decode8<CODE, BF16>(vd[db][0], vd[db][1]);
                const u32x4 hi = decode8<CODE, BF16>(vd[db][2], vd[db][3]);
#pragma unroll
                for (int qt = 0; qt < QT; qt++) {
                    oacc[db][qt] = mfma16<BF16>(lo, pf[0][qt], oacc[db][qt]);
                    oacc[db][qt] = mfma16<BF16>(hi, pf[1][qt], oacc[db][qt]);
                }
            }
        }
        if (j == nfull && j < b1) {  // the tail: this wave's next block
            const int live = s.total - nfull * kKvBlock;  // its tokens
            const uint16_t* kt = c.k_tail + ((int64_t)r * c.heads + h) * kKvBlock * D;
            const uint16_t* vt = c.v_tail + ((int64_t)r * c.heads + h) * kKvBlock * D;
            f32x4 sa[4][QT];
#pragma unroll
            for (int kg = 0; kg < 4; kg++) {
                const int t = 16 * kg + ql;
#pragma unroll
                for (int qt = 0; qt < QT; qt++) sa[kg][qt] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < 2 * KU; u++) {
                    const u32x4 a = t < live ? ld16(kt + t * D + 64 * (u >> 1) + 16 * g + 8 * (u & 1)) : u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int qt = 0; qt < QT; qt++) sa[kg][qt] = mfma16<BF16>(a, qf[qt][u], sa[kg][qt]);
                }
            }
            // V: the lane's 8 tokens of a chunk for one dim; values that are no numbers become 0 here, and their
            // tokens' weights NaN in the rows that see them: 0 * NaN must not reach the rows that do not.
            u32x4 va[2][DB];
            uint32_t bad = 0;
#pragma unroll
            for (int ch = 0; ch < 2; ch++)
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int t = 32 * ch + (e < 4 ? 4 * g + e : 12 + 4 * g + e);
                        uint32_t x = t < live ? vt[t * D + 16 * db + ql] : 0;
                        constexpr uint32_t ex = BF16 ? 0x7f80u : 0x7c00u;
                        if ((x & ex) == ex) {
                            bad |= 1u << (8 * ch + e);
                            x = 0;
                        }
                        va[ch][db][e >> 1] = (e & 1) ? va[ch][db][e >> 1] | (x << 16) : x;
                    }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) bad |= __shfl_xor((int)bad, o);  // over the 16 lanes of a group: its dims
            u32x4 pf[2][QT];
            softmax(sa, p.c2, 0.f, nfull * kKvBlock, false, bad, pf);
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int qt = 0; qt < QT; qt++) {
                    oacc[db][qt] = mfma16<BF16>(va[0][db], pf[0][qt], oacc[db][qt]);
                    oacc[db][qt] = mfma16<BF16>(va[1][db], pf[1][qt], oacc[db][qt]);
                }
        }

        // ---- merge the waves' results ----
#pragma unroll
        for (int qt = 0; qt < QT; qt++) {
            const float l = sum4(l_run[qt]);
            const int rr = 16 * qt + ql;
            if (g == 0) {
                mg.m[wave][rr] = m_run[qt];
                mg.l[wave][rr] = l;
            }
#pragma unroll
            for (int db = 0; db < DB; db++) st4(&mg.o[wave][rr][16 * db + 4 * g], oacc[db][qt]);
        }
        __syncthreads();
        constexpr int PR = D / 8;  // threads per row
        for (int i = tid; i < R * PR; i += 64 * NW) {
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
            const int tok = (int)(row / G), hq = h * G + (int)(row % G);
            const int64_t at = s.t0 + (int64_t)tok;
            if (nchunk == 1) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
                a0 *= inv;
                a1 *= inv;
                *reinterpret_cast<u32x4*>(p.o + at * p.o_tok + hq * D + d0) =
                    u32x4{pack2<BF16>(a0[0], a0[1]), pack2<BF16>(a0[2], a0[3]), pack2<BF16>(a1[0], a1[1]),
                          pack2<BF16>(a1[2], a1[3])};
            } else {
                const int64_t slot = (at * p.heads + hq) * p.chunks + ck;
                float* dst = p.part + slot * D + d0;
                st4(dst, a0);
                st4(dst + 4, a1);
                if (d0 == 0)
                    *reinterpret_cast<float2*>(p.part + (int64_t)p.max_tokens * p.heads * p.chunks * D + 2 * slot) =
                        float2{M, L};
            }
        }
        __syncthreads();  // the next tile's results go to the same LDS
    }
}

// ---- joining the chunks ----
// One wave per row of o: the partial results of its chunks, in order.
template <bool BF16, int D>
__global__ __launch_bounds__(256) void attend_join(Kv8Attend p) {
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
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
    const float2* ml = reinterpret_cast<const float2*>(p.part + (int64_t)p.max_tokens * p.heads * p.chunks * D) + slot;
    float M = kNegInf;
    for (int k = lane; k < n; k += 64) M = fmaxf(M, ml[k].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    float L = 0.f;
    constexpr int E = D / 64;
    float acc[E] = {};
    for (int k = 0; k < n; k++) {
        const float2 x = ml[k];
        const float f = x.x == kNegInf ? 1.f : __builtin_amdgcn_exp2f(x.x - M);
        L += f * x.y;
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] += f * p.part[(slot + k) * D + E * lane + e];
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    uint16_t* dst = p.o + (int64_t)t * p.o_tok + hq * D + E * lane;
    if constexpr (E == 1) *dst = (uint16_t)pack2<BF16>(acc[0] * inv, 0.f);
    else *reinterpret_cast<uint32_t*>(dst) = pack2<BF16>(acc[0] * inv, acc[1] * inv);
}

template <int CODE, bool BF16, int D>
hipError_t attend(const Kv8Attend& p, hipStream_t s) {
    const int64_t grid = (int64_t)p.c.requests * p.c.heads * p.tiles * p.chunks;
    if (grid <= 0 || grid > 0x7fffffff) return hipErrorInvalidValue;
    if (p.rows == 16) hipLaunchKernelGGL((attend_few<CODE, BF16, D, 1>), dim3((unsigned)grid), dim3(64 * NW), 0, s, p);
    else hipLaunchKernelGGL((attend_few<CODE, BF16, D, 2>), dim3((unsigned)grid), dim3(64 * NW), 0, s, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.chunks == 1) return e;
    const int64_t rows = ((int64_t)p.max_tokens * p.heads + 3) / 4;
    hipLaunchKernelGGL((attend_join<BF16, D>), dim3((unsigned)rows), dim3(256), 0, s, p);
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
    p.rows = rows <= 16 ? 16 : 32;
    p.kernel = kAttendFew;
    const int64_t tiles = (rows + p.rows - 1) / p.rows;
    p.tiles = (int32_t)(tiles < 1024 ? tiles : 1024);
    const int64_t blocks = (len + kKvBlock - 1) / kKvBlock;
    const int64_t base = (int64_t)p.c.requests * p.c.heads * p.tiles;
    int64_t chunks = 1;
    const int64_t want = 4 * cus;
    if (base < want) chunks = (want + base - 1) / base;
    int64_t chunk = (blocks + chunks - 1) / chunks;
    if (chunk < 8) chunk = 8;
    p.chunk = (int32_t)chunk;
    chunks = (blocks + chunk - 1) / chunk;
    p.chunks = (int32_t)chunks;
    if (base * chunks > INT32_MAX || (int64_t)p.max_tokens * p.heads > INT32_MAX) return -1;
    return chunks == 1 ? 0 : (int64_t)p.max_tokens * p.heads * chunks * (head_dim + 2) * 4;
}

hipError_t launch_kv8_attend(const Kv8Attend& p, int code, bool bf16, int head_dim, hipStream_t s) {
    if (code == kCodeE4m3) return bf16 ? attend_d<kCodeE4m3, true>(p, head_dim, s) : attend_d<kCodeE4m3, false>(p, head_dim, s);
    return bf16 ? attend_d<kCodeI8, true>(p, head_dim, s) : attend_d<kCodeI8, false>(p, head_dim, s);
}

}  // namespace tsfm
