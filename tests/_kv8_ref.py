"""Plain models of the 8-bit serving operators, for the tests: quantisation and the cache's contents in numpy (f32
arithmetic where the definition says so, exact otherwise), attention and products in float64."""
import numpy as np

BLOCK = 64

# The non-negative e4m3 values by code (bias 7, 3 bits of mantissa, code 127 is NaN), and the midpoints between them.
E4M3 = np.array([(c & 7) * 2.0 ** -9 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) for c in range(127)])
_MID = (E4M3[1:] + E4M3[:-1]) / 2


def e4m3_encode(x):
    """float64 values to e4m3 codes: nearest, ties to the even code; NaN for what is no finite number."""
    x = np.asarray(x, np.float64)
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    low = np.searchsorted(_MID, a, side="left")  # up to and at a midpoint: the code below
    tie = (low < 126) & (a == _MID[np.minimum(low, 125)]) & (low % 2 == 1)
    code = np.minimum(low + tie, 126).astype(np.uint8)
    code = np.where(np.isfinite(x), code, 127).astype(np.uint8)
    return code | (np.signbit(x).astype(np.uint8) << 7)


def e4m3_decode(codes):
    codes = np.asarray(codes, np.uint8)
    v = np.append(E4M3, np.nan)[codes & 127]
    return np.where(codes & 128, -v, v)


def e4m3_scale(amax):
    """The smallest power of two s >= 2^-126 with amax / s <= 448; 1 for 0."""
    if amax == 0:
        return 1.0
    e = -126
    frac, ex = np.frexp(float(amax))  # amax = frac 2^ex
    e = max(e, ex - 9 + (1 if frac > 0.875 else 0))
    return float(2.0 ** e)


def quantise(x, code):
    """One block (any shape) of f32-exact values -> (codes, scale). A block that is not finite: codes 0, scale NaN."""
    x = np.asarray(x, np.float32)
    if not np.isfinite(x).all():
        return np.zeros(x.shape, np.uint8), np.float32(np.nan)
    amax = np.abs(x).max() if x.size else np.float32(0)
    if code == "e4m3":
        s = e4m3_scale(amax)
        return e4m3_encode(x.astype(np.float64) / s), np.float32(s)
    one, top = np.float32(1), np.maximum(amax, np.float32(2.0 ** -100))
    s = np.float32(1) if amax == 0 else top * (one / np.float32(127))
    mul = np.float32(127) * (one / top)
    q = np.clip(np.rint(x * mul), -127, 127).astype(np.int8)
    return q.view(np.uint8), np.float32(s)


def decode(codes, code):
    return e4m3_decode(codes) if code == "e4m3" else np.asarray(codes, np.uint8).view(np.int8).astype(np.float64)


def v_byte(t):
    """Where token t of a block lies in V's row of a dim: token 32 c + 16 a + 4 g + i at byte 16 g + 8 c + 4 a + i."""
    c, a, g, i = t // 32, t // 16 % 2, t // 4 % 4, t % 4
    return 16 * g + 8 * c + 4 * a + i


V_BYTE = np.array([v_byte(t) for t in range(BLOCK)])


class Model:
    """What the cache of some requests must hold: their tokens, dealt to blocks in order."""

    def __init__(self, requests, kv_heads, head_dim, code, blocks, width):
        self.k = [np.zeros((0, kv_heads, head_dim), np.float32) for _ in range(requests)]
        self.v = [np.zeros((0, kv_heads, head_dim), np.float32) for _ in range(requests)]
        self.code, self.blocks, self.width = code, blocks, width
        self.free = list(range(blocks - 1, -1, -1))
        self.table = [[] for _ in range(requests)]

    def lengths(self):
        return [len(x) for x in self.k]

    def plan(self, n_new):
        """Takes blocks for the new tokens: (cu_tokens, cu_blocks, cu_items, slots, pos, items)."""
        cu, cb, ci, slots, pos, items = [0], [0], [0], [], [], []
        for r, n in enumerate(n_new):
            n = max(0, n)
            have = len(self.k[r])
            need = -(-(have + n) // BLOCK) - -(-have // BLOCK)
            for _ in range(need):
                self.table[r].append(self.free.pop())
            for p in range(have, have + n):
                slots.append(self.table[r][p // BLOCK] * BLOCK + p % BLOCK)
                pos.append(p)
            touched = sorted({p // BLOCK for p in range(have, have + n)})
            items += [(r, j) for j in touched]
            cu.append(cu[-1] + n)
            cb.append(cb[-1] + need)
            ci.append(ci[-1] + len(touched))
        return cu, cb, ci, slots, pos, items

    def append(self, n_new, k, v):
        at = 0
        for r, n in enumerate(n_new):
            n = max(0, n)
            self.k[r] = np.concatenate([self.k[r], k[at:at + n]])
            self.v[r] = np.concatenate([self.v[r], v[at:at + n]])
            at += n

    def release(self, drop):
        for r, d in enumerate(drop):
            if d:
                self.free += self.table[r]
                self.table[r] = []
                self.k[r], self.v[r] = self.k[r][:0], self.v[r][:0]

    def block(self, r, j, h, which):
        """(codes (64, D), scale) of whole block j of request r."""
        x = (self.k if which == 0 else self.v)[r][j * BLOCK:(j + 1) * BLOCK, h]
        return quantise(x, self.code)

    def values(self, r, h):
        """K and V of request r as attention reads them, float64."""
        out = []
        for which, x in ((0, self.k[r]), (1, self.v[r])):
            parts = []
            for j in range(len(x) // BLOCK):
                codes, s = self.block(r, j, h, which)
                parts.append(decode(codes, self.code) * np.float64(s))
            parts.append(x[len(x) // BLOCK * BLOCK:, h].astype(np.float64))
            out.append(np.concatenate(parts))
        return out


def attend(q, k, v, last, scale):
    """Rows q (n, D) over keys k, v (m, D); row i reads keys 0 .. last[i]. Returns (o, A, S): the result, the same with
    |v| (what a relative error of a weight is multiplied with), and the largest sum of |q_c k_c| scale (what a relative
    error of a product's terms is)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    o, a, s = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1])), np.zeros(len(q))
    for i in range(len(q)):
        m = min(max(int(last[i]) + 1, 0), len(k))
        if m == 0:
            continue
        x = k[:m] @ q[i] * scale
        w = np.exp(x - x.max())
        w /= w.sum()
        o[i], a[i] = w @ v[:m], w @ np.abs(v[:m])
        s[i] = (np.abs(k[:m]) @ np.abs(q[i])).max() * scale
    return o, a, s


def attend_bound(o, a, s, vmax, keys, half, f16):
    """How far a row of the kernel's may be from attend()'s. half: half a step of the 16-bit type, relative.
    - the result's rounding: half |o|;
    - the weights' rounding to the 16-bit type: half a;
    - f16 weights below 2^-14 are rounded to multiples of 2^-24: 2^-25 each, of a largest weight of 1, times the
      values in units of the largest block scale: 2^-25 * 2 vmax * keys (a scale is at most twice what its values need);
    - f32 arithmetic: a score is a sum of at most 128 products, 2^-24 of each partial sum: 130 * 2^-24 s, a shift
      of the exponent and so a relative error of the weight; the exponential, sums over keys, the joins: 64 * 2^-24."""
    f32 = (130 * s + 64)[:, None] * 2.0 ** -24
    return half * np.abs(o) + (half + f32) * (1 + half) * a + (2.0 ** -24 * vmax * keys if f16 else 0.0) + 1e-30
