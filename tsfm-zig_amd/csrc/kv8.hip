// The paged 8-bit K/V cache's bookkeeping and writes on gfx950: block tables and slot maps from request
// lengths (plan), blocks back to the pool (release), and the step's K/V into the cache (append).
#include "kv8_device.hpp"

namespace tsfm {
namespace {

// ---- plan ----
// Three exclusive prefix sums over the requests (new tokens, blocks taken, cache blocks touched), then one
// pass over the packed tokens. The sums are one workgroup's: 1024 requests a round, one per thread, wave scans
// on lane shifts and one LDS exchange. What it costs is latency, not bytes.
constexpr int PT = 1024, PW = PT / 64;
constexpr int kFillTokens = 1024;  // tokens (and items) per workgroup of plan_fill

__device__ __forceinline__ int blocks_of(int64_t tokens) { return (int)((tokens + kKvBlock - 1) / kKvBlock); }

// The request whose new tokens hold packed token t (t < cu[R]): the last r with cu[r] <= t.
__device__ __forceinline__ int find_request(const int32_t* cu, int lo, int hi, int t) {
    while (lo < hi) {  // cu[lo] <= t < cu[hi + 1]
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Slot, position, table entry and item of packed token t of request r.
__device__ __forceinline__ void fill_token(const Kv8Plan& p, int t, int r, int cu_r, int n, int total, int cb, int ci,
                                           int count_old) {
    const int before = total - n, pos = before + (t - cu_r), blk = pos / kKvBlock;
    const int first = blocks_of(before);  // the request's first new block
    int id;
    if (blk < first) {
        id = p.table[(int64_t)r * p.width + blk];
    } else {
        id = p.free_list[max(0, count_old - 1 - (cb + blk - first))];
        if (pos % kKvBlock == 0) p.table[(int64_t)r * p.width + blk] = id;
    }
    p.slots[t] = (int64_t)id * kKvBlock + pos % kKvBlock;
    p.pos[t] = pos;
    if (t == cu_r || pos % kKvBlock == 0) {
        const int w = ci + blk - before / kKvBlock;
        reinterpret_cast<int2*>(p.items)[w] = int2{r, blk};
    }
}

// FILL: the whole plan in one launch (up to PT requests and kFillTokens tokens); otherwise the sums, and
// plan_fill writes the maps.
template <bool FILL>
__global__ __launch_bounds__(PT) void plan_sums(Kv8Plan p) {
    __shared__ int64_t s_red[PW][2];
    __shared__ int s_bad;
    __shared__ int s_wave[PW][3];
    __shared__ int s_cu[FILL ? PT + 1 : 1], s_cb[FILL ? PT : 1], s_ci[FILL ? PT : 1], s_total[FILL ? PT : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    int64_t tokens = 0, taken = 0;
    bool bad = false;
    for (int r = tid; r < p.requests; r += PT) {
        const int64_t n = max(p.n_new[r], 0), len = p.len[r];
        bad |= len < 0 || len + n > (int64_t)p.width * kKvBlock;
        tokens += n;
        if (len >= 0) taken += blocks_of(len + n) - blocks_of(len);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        tokens += __shfl_xor(tokens, o);
        taken += __shfl_xor(taken, o);
    }
    if (bad) s_bad = 1;  // any writer writes the same
    if (lane == 0) {
        s_red[wave][0] = tokens;
        s_red[wave][1] = taken;
    }
    __syncthreads();
    tokens = taken = 0;
#pragma unroll
    for (int w = 0; w < PW; w++) {
        tokens += s_red[w][0];
        taken += s_red[w][1];
    }
    const int count_old = min(max(*p.free_count, 0), p.blocks);
    const int code = tokens > p.max_tokens ? 1 : s_bad ? 2 : taken > count_old ? 3 : 0;

    int base[3] = {0, 0, 0};
    for (int r0 = 0; r0 < p.requests; r0 += PT) {
        const int r = r0 + tid;
        const bool in = r < p.requests;
        const int len = in ? p.len[r] : 0, n = in && code == 0 ? max(p.n_new[r], 0) : 0;
        const int own[3] = {n, n ? blocks_of((int64_t)len + n) - blocks_of(len) : 0,
                            n ? (len + n - 1) / kKvBlock - len / kKvBlock + 1 : 0};
        int inc[3] = {own[0], own[1], own[2]};
#pragma unroll
        for (int o = 1; o < 64; o <<= 1)
#pragma unroll
            for (int i = 0; i < 3; i++) {
                const int up = __shfl_up(inc[i], o);
                if (lane >= o) inc[i] += up;
            }
        if (lane == 63)
#pragma unroll
            for (int i = 0; i < 3; i++) s_wave[wave][i] = inc[i];
        __syncthreads();
        int tot[3] = {0, 0, 0};
#pragma unroll
        for (int w = 0; w < PW; w++)
#pragma unroll
            for (int i = 0; i < 3; i++) {
                const int x = s_wave[w][i];
                if (w < wave) inc[i] += x;
                tot[i] += x;
            }
        if (in) {
            const int cu = base[0] + inc[0] - own[0], cb = base[1] + inc[1] - own[1], ci = base[2] + inc[2] - own[2];
            p.cu_tokens[r] = cu;
            p.cu_blocks[r] = cb;
            p.cu_items[r] = ci;
            p.len_out[r] = len + n;
            if (FILL) {
                s_cu[tid] = cu;
                s_cb[tid] = cb;
                s_ci[tid] = ci;
                s_total[tid] = len + n;
            }
        }
#pragma unroll
        for (int i = 0; i < 3; i++) base[i] += tot[i];
        __syncthreads();  // s_wave is written again in the next round
    }
    if (tid == 0) {
        p.cu_tokens[p.requests] = base[0];
        p.cu_blocks[p.requests] = base[1];
        p.cu_items[p.requests] = base[2];
        *p.free_count_out = code == 0 ? count_old - base[1] : *p.free_count;
        p.status[0] = code;
        p.status[1] = base[0];
        p.status[2] = base[2];
        p.status[3] = base[1];
        if (FILL) s_cu[p.requests] = base[0];
    }
    if (!FILL) return;
    __syncthreads();
    for (int t = tid; t < p.max_tokens; t += PT) {
        if (t < base[0]) {
            const int r = find_request(s_cu, 0, p.requests - 1, t);
            fill_token(p, t, r, s_cu[r], s_cu[r + 1] - s_cu[r], s_total[r], s_cb[r], s_ci[r], count_old);
        } else {
            p.slots[t] = -1;
            p.pos[t] = -1;
        }
    }
    for (int i = base[2] + tid; i < p.max_items; i += PT) reinterpret_cast<int2*>(p.items)[i] = int2{-1, -1};
}

// The maps of kFillTokens packed tokens per workgroup. The workgroup's first and last request come from a
// 64-way search (each lane tests one request: two loads deep for 4096 requests), its stretch of the prefix sums
// goes to LDS, and each token's request from a search there.
__global__ __launch_bounds__(256) void plan_fill(Kv8Plan p) {
    constexpr int kRange = 2048;
    __shared__ int s_cu[kRange + 1];
    const int tid = threadIdx.x, lane = tid & 63;
    const int t0 = blockIdx.x * kFillTokens, R = p.requests;
    const int tokens = p.cu_tokens[R], items = p.cu_items[R];
    for (int i = t0 + tid; i < min(p.max_items, t0 + kFillTokens); i += 256)
        if (i >= items) reinterpret_cast<int2*>(p.items)[i] = int2{-1, -1};
    for (int t = t0 + tid; t < min(p.max_tokens, t0 + kFillTokens); t += 256)
        if (t >= tokens) {
            p.slots[t] = -1;
            p.pos[t] = -1;
        }
    const int t1 = min(t0 + kFillTokens, tokens);
    if (t0 >= t1) return;
    auto search = [&](int t) {  // the last r with cu[r] <= t
        int lo = 0, n = R;      // r in [lo, lo + n)
        while (n > 1) {
            const int step = (n + 63) / 64, at = lo + lane * step;
            const uint64_t le = __ballot(at < lo + n && p.cu_tokens[min(at, R)] <= t);
            const int k = __popcll(le) - 1;  // lane 0 always holds: cu[lo] <= t
            const int next = lo + k * step;
            n = min(step, lo + n - next);
            lo = next;
        }
        return lo;
    };
    const int ra = search(t0), rb = search(t1 - 1);
    const bool staged = rb - ra < kRange;
    if (staged)
        for (int i = tid; i <= rb - ra + 1; i += 256) s_cu[i] = p.cu_tokens[ra + i];
    __syncthreads();
    const int count_old = *p.free_count_out + p.cu_blocks[R];
    for (int t = t0 + tid; t < t1; t += 256) {
        const int r = staged ? ra + find_request(s_cu, 0, rb - ra, t) : find_request(p.cu_tokens, ra, rb, t);
        const int cu = p.cu_tokens[r];
        fill_token(p, t, r, cu, p.cu_tokens[r + 1] - cu, p.len_out[r], p.cu_blocks[r], p.cu_items[r], count_old);
    }
}

// ---- release ----
// One workgroup: 1024 requests a round; their blocks are counted (a wave per dropped request), placed by a
// prefix sum, and copied.
__global__ __launch_bounds__(PT) void release(Kv8Release p) {
    __shared__ int s_n[PT];
    __shared__ long long s_off[PT], s_wave[PW];  // 64 bits: tables that name a block many times pass 32
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int count = min(max(*p.free_count, 0), p.blocks);
    auto valid = [&](int r, int j) {  // the pool block at entry j, or -1
        const int id = p.table[(int64_t)r * p.width + j];
        return id >= 0 && id < p.blocks ? id : -1;
    };
    auto entries = [&](int r) {
        const int64_t len = max(p.len[r], 0);
        return (int)min((len + kKvBlock - 1) / kKvBlock, (int64_t)p.width);
    };
    int64_t total = 0;
    for (int pass = 0; pass < 2; pass++) {
        int64_t base = count;
        for (int r0 = 0; r0 < p.requests; r0 += PT) {
            const int n = min(PT, p.requests - r0);
            s_n[tid] = 0;
            __syncthreads();
            for (int i = wave; i < n; i += PW) {
                if (!p.drop[r0 + i]) continue;
                const int e = entries(r0 + i);
                int have = 0;
                for (int j0 = 0; j0 < e; j0 += 64)
                    have += __popcll(__ballot(j0 + lane < e && valid(r0 + i, min(j0 + lane, e - 1)) >= 0));
                if (lane == 0) s_n[i] = have;
            }
            __syncthreads();
            long long inc = s_n[tid];
            const long long own = inc;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const long long up = __shfl_up(inc, o);
                if (lane >= o) inc += up;
            }
            if (lane == 63) s_wave[wave] = inc;
            __syncthreads();
            long long tot = 0;
            for (int w = 0; w < PW; w++) {
                if (w < wave) inc += s_wave[w];
                tot += s_wave[w];
            }
            s_off[tid] = inc - own;
            __syncthreads();
            if (pass == 1)
                for (int i = wave; i < n; i += PW) {
                    if (!p.drop[r0 + i]) continue;
                    const int r = r0 + i, e = entries(r);
                    int64_t at = base + s_off[i];
                    for (int j0 = 0; j0 < e; j0 += 64) {
                        const int j = j0 + lane, id = j < e ? valid(r, j) : -1;
                        const uint64_t m = __ballot(id >= 0);
                        if (id >= 0) p.free_list[at + __popcll(m & ((1ull << lane) - 1))] = id;
                        if (j < e) p.table[(int64_t)r * p.width + j] = -1;
                        at += __popcll(m);
                    }
                    if (lane == 0) p.len[r] = 0;
                }
            base += tot;
            __syncthreads();
        }
        if (pass == 0) {
            total = base - count;
            if (base > p.blocks) {  // the list would pass the pool: tables and list do not belong together
                if (tid == 0) {
                    p.status[0] = 1;
                    p.status[1] = 0;
                }
                return;
            }
        }
    }
    if (tid == 0) {
        *p.free_count = count + (int)total;
        p.status[0] = 0;
        p.status[1] = (int)total;
    }
}

// ---- append ----
// One wave per (touched block, head, K or V). A lane holds tokens 16 s + 4 g + i (g = lane / 16; s, i < 4) of
// E = D / 16 dims: a row's 16 lanes read its 2 D bytes together, a lane's four consecutive tokens of one dim pack
// into the word that V's byte order wants, and the four words of a dim are 16 contiguous bytes of the block: V is
// transposed in registers, without LDS.
// Bytes bound it where there are many blocks (2 read, 1 written per element), latency for single tokens.
template <int CODE, bool BF16, int D>
__global__ __launch_bounds__(256) void kv8_append(Kv8Append p) {
    constexpr int E = D / 16, W = E / 2;  // dims per lane, dwords of a lane's piece of a row
    typedef uint32_t piece __attribute__((ext_vector_type(W)));
    const int lane = threadIdx.x & 63, g = lane >> 4, cl = lane & 15;
    const Kv8& c = p.c;
    const int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (id >= (int64_t)p.max_items * c.heads * 2) return;
    const int which = (int)(id & 1), h = (int)((id >> 1) % c.heads), w = (int)((id >> 1) / c.heads);
    const int r = p.items[2 * (int64_t)w], j = p.items[2 * (int64_t)w + 1];
    if (r < 0 || r >= c.requests || j < 0 || j >= c.width) return;
    const Span s = request_span(p.cu_tokens, c.len, r, p.max_tokens, c.width);
    const int blk = c.table[(int64_t)r * c.width + j];
    const int first = s.before >= 0 ? s.before / kKvBlock : 0;
    const int64_t x_tok = which ? p.v_tok : p.k_tok;
    const uint16_t* const x = (which ? p.v : p.k) + h * D + E * cl;
    uint16_t* const tail = (which ? c.v_tail : c.k_tail) + ((int64_t)r * c.heads + h) * kKvBlock * D + E * cl;

    auto fresh = [&](int pos) {  // the new token at position pos
        return *reinterpret_cast<const piece*>(x + (s.t0 + (int64_t)(pos - s.before)) * x_tok);
    };
    auto to_tail = [&](int jb) {  // the new tokens of the partial block jb
        const int lo = max(s.before - jb * kKvBlock, 0), hi = s.total - jb * kKvBlock;
        for (int t = lo + g; t < hi; t += 4) *reinterpret_cast<piece*>(tail + t * D) = fresh(jb * kKvBlock + t);
    };
    // The tail holds the first block's old tokens until that block's wave has read them: where the step both
    // completes that block and leaves a new tail, that wave writes the tail, after its loads.
    const bool old_tail = s.before > first * kKvBlock;
    if ((j + 1) * kKvBlock > s.total) {
        if (j * kKvBlock < s.total && (j == first || !old_tail)) to_tail(j);
        return;
    }
    piece d[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int t = 16 * (i >> 2) + 4 * g + (i & 3), pos = j * kKvBlock + t;
        d[i] = pos >= s.before ? fresh(pos) : *reinterpret_cast<const piece*>(tail + t * D);
    }
    float amax = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 16; i++)
#pragma unroll
        for (int e = 0; e < W; e++) {
            // largest magnitude, and whether one is a NaN or an infinity (all bits of the exponent set)
            constexpr uint32_t ex = BF16 ? 0x7f80u : 0x7c00u;
            const uint32_t u = d[i][e];
            bad |= (u & ex) == ex || ((u >> 16) & ex) == ex;
            amax = fmaxf(amax, fmaxf(fabsf(half_to_f32<BF16>(u & 0xffffu)), fabsf(half_to_f32<BF16>(u >> 16))));
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    bad = __ballot(bad) != 0;
    float scale, mul;
    block_scale<CODE>(bad ? 0.f : amax, scale, mul);
    if (blk >= 0 && blk < c.blocks) {
        const int64_t at = (int64_t)blk * c.heads + h;
        if (lane == 0) c.scales[2 * at + which] = bad ? __builtin_nanf("") : scale;
        uint8_t* const out = (which ? c.v : c.k) + at * kKvBlock * D;
        auto val = [&](int i, int e) {
            const uint32_t u = d[i][e >> 1];
            const float f = half_to_f32<BF16>((e & 1) ? u >> 16 : u & 0xffffu) * mul;
            return bad ? 0.f : f;
        };
        if (which == 0) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int t = 16 * (i >> 2) + 4 * g + (i & 3);
                uint32_t* dst = reinterpret_cast<uint32_t*>(out + t * D + E * cl);
                const uint32_t w0 = encode4<CODE>(val(i, 0), val(i, 1), val(i, 2), val(i, 3));
                if constexpr (E == 4) *dst = w0;
                else
                    *reinterpret_cast<u32x2*>(dst) =
                        u32x2{w0, encode4<CODE>(val(i, E - 4), val(i, E - 3), val(i, E - 2), val(i, E - 1))};
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) {
                u32x4 word;  // words (c, a): tokens 32 c + 16 a + 4 g + 0..3
#pragma unroll
                for (int q = 0; q < 4; q++)
                    word[q] = encode4<CODE>(val(4 * q, e), val(4 * q + 1, e), val(4 * q + 2, e), val(4 * q + 3, e));
                *reinterpret_cast<u32x4*>(out + (E * cl + e) * kKvBlock + 16 * g) = word;
            }
        }
    }
    if (j == first && old_tail && s.total % kKvBlock != 0 && s.total / kKvBlock > j) to_tail(s.total / kKvBlock);
}

template <int CODE, bool BF16>
hipError_t append_d(const Kv8Append& p, int head_dim, hipStream_t s) {
    const int64_t waves = (int64_t)p.max_items * p.c.heads * 2, grid = (waves + 3) / 4;
    if (grid <= 0 || grid > 0x7fffffff) return hipErrorInvalidValue;
    if (head_dim == 64) hipLaunchKernelGGL((kv8_append<CODE, BF16, 64>), dim3((unsigned)grid), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((kv8_append<CODE, BF16, 128>), dim3((unsigned)grid), dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv8_plan(const Kv8Plan& p, hipStream_t s) {
    if (p.requests <= PT && p.max_tokens <= kFillTokens) {
        hipLaunchKernelGGL(plan_sums<true>, dim3(1), dim3(PT), 0, s, p);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(plan_sums<false>, dim3(1), dim3(PT), 0, s, p);
    const int64_t n = p.max_tokens > p.max_items ? p.max_tokens : p.max_items;
    hipLaunchKernelGGL(plan_fill, dim3((unsigned)((n + kFillTokens - 1) / kFillTokens)), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_kv8_release(const Kv8Release& p, hipStream_t s) {
    hipLaunchKernelGGL(release, dim3(1), dim3(PT), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_kv8_append(const Kv8Append& p, int code, bool bf16, int head_dim, hipStream_t s) {
    if (code == kCodeE4m3) return bf16 ? append_d<kCodeE4m3, true>(p, head_dim, s) : append_d<kCodeE4m3, false>(p, head_dim, s);
    return bf16 ? append_d<kCodeI8, true>(p, head_dim, s) : append_d<kCodeI8, false>(p, head_dim, s);
}

}  // namespace tsfm
