"""Plain numpy forms of the 8-bit KV cache's operators, row by row and page by page, and seeded inputs for them."""
import numpy as np

PAGE = 16
SMALLEST = np.float32(2.0 ** -126)
OK, NO_PAGES, LENGTH, NO_TOKENS = range(4)


def from_bf16(bits):
    return (np.asarray(bits, dtype=np.uint32) << 16).view(np.float32)


def to_bf16(values):
    u = np.ascontiguousarray(values, dtype=np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


# ---- codes ---------------------------------------------------------------------------------------------------------------

def _e4m3_values():
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v[c] = (-1.0) ** (c >> 7) * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    v[0x7f] = v[0xff] = np.nan
    return v


E4M3 = _e4m3_values()


def decode(codes, e4m3):
    codes = np.asarray(codes, dtype=np.uint8)
    return E4M3[codes] if e4m3 else codes.view(np.int8).astype(np.float64)


def encode(values, e4m3):
    """Nearest code, ties to even; the largest one for what lies beyond."""
    v = np.asarray(values, dtype=np.float64)
    if not e4m3:
        return np.clip(np.rint(v), -127, 127).astype(np.int8).view(np.uint8)
    a = np.abs(v)
    step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    a = np.minimum(np.rint(a / step) * step, 448.0)
    e = np.floor(np.log2(np.maximum(a, 2.0 ** -6))).astype(int)
    normal = ((e + 7) << 3) | (np.rint(a / 2.0 ** (e - 3)).astype(int) & 7)
    code = np.where(a < 2.0 ** -6, np.rint(a * 512).astype(int), normal)
    return (code | (np.signbit(v).astype(int) << 7)).astype(np.uint8)


# ---- block tables --------------------------------------------------------------------------------------------------------

def page_tables(lengths, changes, table, free_pages, free_count, capacity):
    """As q3t_ops.h has it, a row at a time."""
    rows, stride = table.shape
    table, lengths = table.copy(), [int(n) for n in lengths]
    stack = [int(p) for p in free_pages[:free_count]]
    pages = lambda n: -(-n // PAGE)  # noqa: E731
    status, new, starts, positions, slots = [], list(lengths), [0], [], []
    legal = [0 <= n <= stride * PAGE and 0 <= n + int(c) <= stride * PAGE for n, c in zip(lengths, changes)]
    for r in range(rows):
        if legal[r] and changes[r] < 0:
            new[r] = lengths[r] + int(changes[r])
            stack += [int(p) for p in table[r, pages(new[r]):pages(lengths[r])]]
    stack = stack[:len(free_pages)]
    asked = needed = 0
    room = len(stack)
    for r in range(rows):
        c = int(changes[r])
        if not legal[r]:
            status.append(LENGTH)
        elif c <= 0:
            status.append(OK)
        else:
            want = lengths[r] + c
            need = pages(want) - pages(lengths[r])
            asked, needed = asked + c, needed + need
            if asked > capacity:
                status.append(NO_TOKENS)
            elif need and needed > room:
                status.append(NO_PAGES)
            else:
                status.append(OK)
                for p in range(pages(lengths[r]), pages(want)):
                    table[r, p] = stack.pop()
                positions += range(lengths[r], want)
                slots += [int(table[r, p // PAGE]) * PAGE + p % PAGE for p in range(lengths[r], want)]
                new[r] = want
        starts.append(len(slots))
    return dict(page_table=table, free=stack, lengths=np.array(new), status=np.array(status), starts=np.array(starts),
                positions=np.array(positions, dtype=np.int64), slots=np.array(slots, dtype=np.int64))


# ---- append --------------------------------------------------------------------------------------------------------------

def finite(bits):
    """What is not finite as the largest finite bf16 of its sign."""
    bits = np.asarray(bits, dtype=np.uint16)
    return np.where((bits & 0x7fff) >= 0x7f80, (bits & 0x8000) | 0x7f7f, bits).astype(np.uint16)


def append_plane(codes, scales, new, slots, e4m3):
    """codes [pages][heads][16][dim] and scales [pages][heads] after new [tokens][heads * dim] bf16 bits went to `slots`, a page at a
    time and every operation in fp32."""
    codes, scales = codes.copy(), scales.copy()
    pages, heads, _, dim = codes.shape
    x = from_bf16(finite(new)).reshape(-1, heads, dim)
    most = np.float32(448 if e4m3 else 127)
    first = 0
    while first < len(slots):
        page = slots[first] // PAGE
        last = first
        while last < len(slots) and slots[last] >= 0 and slots[last] // PAGE == page:
            last += 1
        if slots[first] < 0 or page >= pages:
            first += 1
            continue
        fill = {int(slots[t]) % PAGE: t for t in range(first, last)}          # the last one that names a slot
        held = min(fill)
        for h in range(heads):
            mine = {s: x[t, h] for s, t in fill.items()}
            scale = np.maximum(np.float32(max(np.abs(v).max() for v in mine.values())) / most, SMALLEST)
            if held:
                own = scales[page, h]
                scale = max(scale, own)
                if scale > own:
                    shrink = own * (np.float32(1) / scale)
                    old = decode(codes[page, h, :held], e4m3).astype(np.float32) * shrink
                    codes[page, h, :held] = encode(old, e4m3)
            inverse = np.float32(1) / scale
            for s, v in mine.items():
                codes[page, h, s] = encode(v * inverse, e4m3)
            scales[page, h] = scale
        first = last
    return codes, scales


# ---- attention -----------------------------------------------------------------------------------------------------------

def attention(q, planes, table, lengths, starts, e4m3, max_seq=None, scale=None):
    """(out, tolerance) in 64 bits, [tokens][query heads][dim].

    The tolerance of the fp32 value: with weights p_j (sum 1) and values v_j, an error e_j relative to each weight and one of the sum give
    at most 2 max|e| * sum p_j |v_j|.  A weight enters the product as fp16 (half a step: 2^-11), its exponent comes from a score in
    fp32: a sum of dim products (and one scale) is off by (dim + 8) * 2^-24 of the sum of magnitudes, and an error of the exponent is
    a relative error of the weight; 2^-21 for the exponential itself.  Sums over n tokens: n * 2^-24.  What multiplies the codes, p_j times
    the page's scale, is subnormal as fp16 (or, far below, zero) where it is less than 2^-20 of the largest such product: an absolute error of
    2^-31 of that one each, times a code of at most M in any dimension, whatever the dimension's own sum is.  Scales below 2^-80 count as
    that there."""
    kc, vc, ks, vs = planes
    heads, dim = kc.shape[1], kc.shape[3]
    qf = from_bf16(q).astype(np.float64).reshape(len(q), -1, dim)
    group = qf.shape[1] // heads
    scale = dim ** -0.5 if scale is None else scale
    out, tol = np.zeros(qf.shape), np.zeros(qf.shape)
    for r, length in enumerate(lengths):
        s0, s1 = (r, r + 1) if starts is None else (int(starts[r]), int(starts[r + 1]))
        for t in range(s0, s1):
            seen = length - (s1 - s0) + (t - s0) + 1
            seen = min(seen, seen if max_seq is None else max_seq)
            if seen <= 0:
                continue
            ids = table[r, :-(-seen // PAGE)]
            good = np.repeat((ids >= 0) & (ids < kc.shape[0]), PAGE)[:seen]
            ids = np.where((ids >= 0) & (ids < kc.shape[0]), ids, 0)
            for h in range(heads):
                k = (decode(kc[ids, h], e4m3) * ks[ids, h].astype(np.float64)[:, None, None]).reshape(-1, dim)[:seen][good]
                v = (decode(vc[ids, h], e4m3) * vs[ids, h].astype(np.float64)[:, None, None]).reshape(-1, dim)[:seen][good]
                if len(k) == 0:
                    continue
                g = slice(h * group, (h + 1) * group)
                s = qf[t, g] @ k.T * scale
                off = (np.abs(qf[t, g]) @ np.abs(k).T).max(axis=1) * scale * (dim + 8) * 2.0 ** -24
                p = np.exp(s - s.max(axis=1, keepdims=True))
                p /= p.sum(axis=1, keepdims=True)
                out[t, g] = p @ v
                size = p @ np.abs(v)
                each = 2.0 ** -11 + off[:, None] + 2.0 ** -21 + len(k) * 2.0 ** -24
                most = (448 if e4m3 else 127) * np.repeat(np.maximum(vs[ids, h].astype(np.float64), 2.0 ** -80), PAGE)[:seen][good]
                tol[t, g] = 2 * each * size + len(k) * 2.0 ** -31 * (p * most).max(axis=1)[:, None]
    return out, tol


def cache(rng, pages, heads, dim, e4m3, spread=0.5):
    """Planes of random codes and scales, a factor of e^(+-spread) apart."""
    def codes():
        x = rng.standard_normal((pages, heads, PAGE, dim))
        return encode(x * ((448 if e4m3 else 127) / np.abs(x).max(axis=(2, 3), keepdims=True)), e4m3)

    def scales():
        return (3.5 / (448 if e4m3 else 127) * np.exp(rng.uniform(-spread, spread, (pages, heads)))).astype(np.float32)
    return [codes(), codes(), scales(), scales()]


def tables_of(rng, lengths, pages, stride=None):
    """A page table of rows of these lengths over a pool of `pages`, ids in any order, nonsense behind the last page of a row."""
    counts = [-(-max(int(n), 0) // PAGE) for n in lengths]
    assert sum(counts) <= pages
    ids = rng.permutation(pages)
    table = np.full((len(lengths), stride or max(max(counts), 1)), -12345678, dtype=np.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = ids[at:at + c]
        at += c
    return table
