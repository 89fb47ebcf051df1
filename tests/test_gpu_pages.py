"""GPU tests of the paged KV cache and of attention over it: the formula in 64
bits on the values the cache holds, over types, head shapes, lengths, windows,
shared prefixes and strides; what stands in places a token does not see; the
cache's own copies and moves; captured calls; refusals.

Tolerances.  With u = 2^-24 (32-bit sums), h(T) half a step of a 16-bit type
(bf16 2^-9 of the value's binade at most 2^-8 relative: finfo.eps / 2), S the
largest sum |q_d k_d| * scale of a row, n its positions, A = sum_j p_j |v_j|:
  * a score is off by at most (head_dim + 4) u S from the 32-bit sum, and by
    what is left of a 32-bit query: h(page type) S where it is rounded to the
    page type (F16 pages, BF16 results), its square where it is split in two,
    2^-22 S for 32-bit results (BF16 in three, F16 in two);
  * a probability is off by that, by 2 u of its exponential, relatively; the
    sum of them by as much, so the quotient by twice that;
  * rounding it to the page type adds h(T); for 32-bit results h(T)^2 (F16, split
    in two) or h(T)^3 (BF16, in three);
  * F16 probabilities, 2^10 times larger, vanish below 2^-35: n 2^-35;
  * sums of n terms add n u; the result's own rounding h(output) |o|.
"""
import ctypes

import numpy as np
import pytest

from diskmule_amd import HipError, load_library

pytestmark = pytest.mark.gpu

F32, F16, BF16 = 0, 1, 30
HALF = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
PAGE = 64
U = 2.0 ** -24


def to_bits(x, kind):
    """f32 -> the type's stored form (numpy array), nearest even."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    if kind == F32:
        return x
    if kind == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, kind):
    if kind == F32:
        return b.astype(np.float64)
    if kind == F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Model:
    """A cache, and what each of its sequences should hold, layer by layer."""

    def __init__(self, ctx, kind, kvh, hd, pages=64, sequences=8, layers=1, context=4096):
        self.ctx, self.kind, self.kvh, self.hd, self.layers = ctx, kind, kvh, hd, layers
        self.pages = ctx.new_kv_pages(kind, layers, kvh, hd, context, pages, sequences)
        self.rows = {}  # sequence -> [layers][2][tokens, kvh, hd] in 64 bits
        self.keep = []

    def close(self):
        self.pages.free()

    def new(self):
        s = self.pages.new_sequence()
        self.rows[s] = [[np.zeros((0, self.kvh, self.hd))] * 2 for _ in range(self.layers)]
        return s

    def device(self, a):
        self.keep.append(self.ctx.device_array(a))
        return self.keep[-1].device_ptr

    def fork(self, parents, lengths):
        children = self.pages.fork(parents, lengths)
        for c, p, n in zip(children, parents, lengths):
            self.rows[c] = [[x[:n] for x in layer] for layer in self.rows[p]]
        return children

    def release(self, seqs):
        self.pages.release(seqs)
        for s in seqs:
            del self.rows[s]

    def write(self, plan, seqs, counts, rng, source=F32, make=None, pad=0, shift=0):
        """New tokens of every layer through the plan (set to them)."""
        n, width = sum(counts), self.kvh * self.hd
        for layer in range(self.layers):
            bits = []
            for which in range(2):
                x = rng.standard_normal((n, self.kvh, self.hd)) if make is None else make(which, layer, n)
                bits.append(to_bits(x, source))
                if source == F32:
                    held = from_bits(to_bits(bits[-1], self.kind), self.kind)
                else:
                    held = from_bits(bits[-1], source)
                lo = 0
                for s, c in zip(seqs, counts):
                    self.rows[s][layer][which] = np.concatenate([self.rows[s][layer][which], held[lo:lo + c]])
                    lo += c
            pitch = width + pad
            p = []
            for b in bits:
                wide = np.zeros(n * pitch + shift, dtype=b.dtype)
                wide[shift:].reshape(n, pitch)[:, :width] = b.reshape(n, width)
                p.append(self.device(wide) + shift * b.dtype.itemsize)
            self.ctx.write_kv_pages_device(plan, layer, source, p[0], pitch, p[1], pitch)

    def grow(self, seqs, counts, rng, **more):
        self.pages.extend(seqs, counts)
        if sum(counts):
            plan = self.pages.new_plan(self.kvh, None, F32, F32, sum(counts))
            plan.set(seqs, counts)
            self.write(plan, seqs, counts, rng, **more)
            self.ctx.synchronize()
            plan.free()

    def stored(self, seq, layer=0):
        """(keys, values) of a sequence as its pages hold them."""
        ids, n = self.pages.page_ids(seq), self.pages.length(seq)
        size, kvh, hd = self.pages.page_bytes(), self.kvh, self.hd
        k, v = [], []
        for p in ids:
            raw = self.ctx.copy_to_host(self.pages.layer_ptr(layer) + p * size, size, np.uint16).reshape(kvh, 2, -1)
            k.append(raw[:, 0].reshape(kvh, hd // 8, PAGE, 8).transpose(2, 0, 1, 3).reshape(PAGE, kvh, hd))
            c = raw[:, 1].reshape(kvh, 8, hd, 8)
            out = np.zeros((PAGE, kvh, hd), dtype=np.uint16)
            for chunk in range(8):
                for j in range(8):
                    out[16 * (chunk // 2) + 4 * (chunk % 2) + 8 * (j // 4) + j % 4] = c[:, chunk, :, j]
            v.append(out)
        join = lambda x: from_bits(np.concatenate(x)[:n] if x else np.zeros((0, kvh, hd), np.uint16), self.kind)  # noqa: E731
        return join(k), join(v)

    def check_stored(self, seqs=None):
        for s in self.rows if seqs is None else seqs:
            for layer in range(self.layers):
                k, v = self.stored(s, layer)
                assert np.array_equal(k, self.rows[s][layer][0], equal_nan=True), (s, layer)
                assert np.array_equal(v, self.rows[s][layer][1], equal_nan=True), (s, layer)

    def expect(self, seqs, counts, q, window, scale, layer=0):
        """(output, the bound's S, A and n of each row) in 64 bits; q [tokens, heads, hd]."""
        heads = q.shape[1]
        group = heads // self.kvh
        o, spread, size, count = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape), np.zeros(q.shape[0])
        t = 0
        for s, c in zip(seqs, counts):
            k, v = self.rows[s][layer]
            for i in range(c):
                p = k.shape[0] - c + i
                lo = max(0, p + 1 - window) if window else 0
                for h in range(heads):
                    kk, vv = k[lo:p + 1, h // group], v[lo:p + 1, h // group]
                    x = kk @ q[t, h] * scale
                    w = np.exp(x - x.max())
                    w /= w.sum()
                    o[t, h] = w @ vv
                    spread[t, h] = (np.abs(kk) @ np.abs(q[t, h])).max() * scale
                    size[t, h] = w @ np.abs(vv)
                count[t] = p + 1 - lo
                t += 1
        return o, spread, size, count

    def attend(self, seqs, counts, rng, heads, window=0, q_type=F32, out_type=F32, scale=None, layer=0, pad=0, shift=0,
               plan=None, q=None, check=True):
        hd = self.hd
        n, width = sum(counts), heads * hd
        scale = 1.0 / np.sqrt(hd) if scale is None else scale
        scale = float(np.float32(scale))
        if q is None:
            q = rng.standard_normal((n, heads, hd)) * 1.5 / (scale * np.sqrt(hd))
        bits = to_bits(q, q_type)
        mine = plan is None
        if mine:
            plan = self.pages.new_plan(heads, window or None, q_type, out_type, n)
            plan.set(seqs, counts)
        pitch = width + pad
        wide = np.zeros(n * pitch + shift, dtype=bits.dtype)
        wide[shift:].reshape(n, pitch)[:, :width] = bits.reshape(n, width)
        item = 4 if out_type == F32 else 2
        out = np.full((n + 2) * pitch + shift, 0x7B7B if item == 2 else 0x7B7B7B7B, dtype=np.uint16 if item == 2 else np.uint32)
        qp, op = self.device(wide) + shift * bits.dtype.itemsize, self.ctx.device_array(out)
        self.ctx.attention_pages_device(plan, layer, scale, qp, pitch, op.device_ptr + (shift + pitch) * item, pitch)
        self.ctx.synchronize()
        got = op.read(0, out.nbytes, out.dtype)
        rows = got[shift:].reshape(n + 2, pitch)
        # nothing beside the rows is touched
        guard = out[0]
        assert (got[:shift] == guard).all() and (rows[0] == guard).all() and (rows[-1] == guard).all()
        assert (rows[1:-1, width:] == guard).all()
        value = np.ascontiguousarray(rows[1:-1, :width])
        value = (value.view(np.float32).astype(np.float64) if item == 4 else from_bits(value, out_type)).reshape(n, heads, hd)
        if mine:
            plan.free()
        if check:
            self.close_to(value, seqs, counts, from_bits(bits, q_type), window, scale, q_type, out_type, layer)
        return value

    def close_to(self, got, seqs, counts, q, window, scale, q_type, out_type, layer=0):
        o, spread, size, n = self.expect(seqs, counts, q, window, scale, layer)
        n = n[:, None, None]
        exact = out_type == F32
        once = self.kind == F16 and out_type == BF16
        query = 2.0 ** -22 if exact else 0.0 if q_type != F32 else HALF[self.kind] if once else HALF[self.kind] ** 2
        score = ((self.hd + 4) * U + query) * spread[:, :, None]
        p = HALF[self.kind] ** ((3 if self.kind == BF16 else 2) if exact else 1)
        bound = (2 * (score + 2 * U) + p + (n + 8) * U) * size * 1.01 + n * 2.0 ** -35 * np.abs(o).max() + \
            HALF[out_type] * np.abs(o) * 1.01 + 1e-30
        worst = np.abs(got - o) / bound
        assert np.isfinite(got).all() and worst.max() <= 1.0, (worst.max(), np.unravel_index(worst.argmax(), worst.shape))


def expect_error(variant, fn, *args):
    with pytest.raises(HipError) as e:
        fn(*args)
    assert e.value.variant == variant, str(e.value)
    return e.value


@pytest.fixture(autouse=True)
def no_result_pending(ctx):
    """Each test's own calls alone are reported in it (and none in a later file's)."""
    yield
    try:
        ctx.attention_result()
    except HipError:
        pass


# ---- pages ------------------------------------------------------------------------

@pytest.mark.parametrize("kind,source", [(BF16, F32), (F16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("kvh,hd", [(1, 8), (3, 80), (8, 128), (2, 512)])
def test_written_rows_stand_in_the_documented_places(ctx, kind, source, kvh, hd):
    rng = np.random.default_rng(1)
    m = Model(ctx, kind, kvh, hd, layers=2)
    a, b, c = m.new(), m.new(), m.new()
    # starts and ends inside pages, chunks and the half pages that the kernel stages
    for counts in ([1, 0, 64], [1, 70, 3], [2, 1, 29], [59, 33, 1], [1, 1, 100], [130, 5, 31]):
        m.grow([a, b, c], counts, rng, source=source, pad=hd, shift=1)
    m.check_stored()
    m.close()


def test_rows_beyond_a_sequence_keep_what_they_held(ctx):
    rng = np.random.default_rng(2)
    m = Model(ctx, BF16, 2, 16, pages=4)
    a = m.new()
    m.grow([a], [64], rng)
    held = m.rows[a]
    m.pages.truncate(a, 10)
    m.rows[a] = [[x[:10] for x in layer] for layer in held]
    m.grow([a], [7], rng)
    new = m.rows[a]
    m.pages.extend([a], [47])
    m.rows[a] = [[np.concatenate([n, o[17:]]) for n, o in zip(x, y)] for x, y in zip(new, held)]
    m.check_stored()
    m.close()


def test_forks_share_whole_pages_and_own_the_last_one(ctx):
    rng = np.random.default_rng(3)
    m = Model(ctx, F16, 2, 40, pages=60, sequences=12, layers=3)
    a = m.new()
    m.grow([a], [150], rng)
    used = m.pages.used_pages()
    kids = m.fork([a, a, a, a], [150, 128, 70, 0])  # the same parent again and again
    assert m.pages.used_pages() == used + 2
    m.grow(kids + [a], [3, 1, 100, 65, 1], rng)
    m.check_stored()
    more = m.fork([kids[2], a, kids[2]], [100, 151, 170])
    m.release([kids[0], a])
    m.grow(more, [1, 200, 7], rng)
    m.check_stored()
    m.close()


def test_compaction_moves_pages_and_not_their_contents(ctx):
    rng = np.random.default_rng(4)
    # more pages than one launch moves
    m = Model(ctx, BF16, 1, 8, pages=1200, sequences=34, layers=2, context=64 * 100)
    seqs = [m.new() for _ in range(28)]
    m.grow(seqs, [64 * 41 + i for i in range(28)], rng)
    kids = m.fork(seqs[20:23], [64 * 40 + 9] * 3)
    m.release(seqs[0:14])
    plan = m.pages.new_plan(2, None, F32, F32, 64)
    plan.set(kids, [5, 5, 5])  # plans survive
    moved = m.pages.compact()
    assert moved > 480
    used = m.pages.used_pages()
    assert all(p < used for s in m.rows for p in m.pages.page_ids(s))
    m.check_stored()
    m.attend(kids, [5, 5, 5], rng, 2, plan=plan)
    assert m.pages.compact() == 0
    m.grow(kids, [100, 1, 64], rng)
    m.check_stored()
    plan.free()
    m.close()


def test_pages_behind_four_gigabytes(ctx):
    rng = np.random.default_rng(5)
    kvh, hd = 8, 128  # 256 KiB a page
    m = Model(ctx, BF16, kvh, hd, pages=17000, sequences=2, layers=2, context=64 * 16990)
    far = m.new()
    m.pages.extend([far], [64 * 16980])  # room that is never written
    a = m.new()
    m.grow([a], [100], rng)
    assert min(m.pages.page_ids(a)) >= 16980
    m.check_stored([a])
    for layer in range(2):
        m.attend([a], [3], rng, 32, layer=layer)
    m.close()


# ---- attention --------------------------------------------------------------------

SHAPES = [(1, 1, 8), (8, 2, 64), (6, 2, 80), (32, 8, 128), (71, 1, 64), (4, 2, 256), (4, 1, 512), (3, 3, 136)]
TYPES = [(BF16, F32, F32), (BF16, BF16, BF16), (F16, F32, F32), (F16, F16, F16), (BF16, F32, F16), (F16, F32, BF16),
         (BF16, BF16, F32)]


@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
@pytest.mark.parametrize("kind,q_type,out_type", TYPES)
def test_prompts_of_different_lengths(ctx, heads, kvh, hd, kind, q_type, out_type):
    rng = np.random.default_rng(hd + heads)
    m = Model(ctx, kind, kvh, hd)
    lengths = [1, 2, 33, 64, 65, 130] if heads * hd < 2000 else [1, 63, 97]
    seqs = [m.new() for _ in lengths]
    m.grow(seqs, lengths, rng)
    m.attend(seqs, lengths, rng, heads, q_type=q_type, out_type=out_type)
    m.close()


@pytest.mark.parametrize("window", [1, 2, 31, 64, 65, 1000])
@pytest.mark.parametrize("kind,out_type", [(BF16, F32), (F16, F16)])
@pytest.mark.parametrize("hd", [64, 256, 512])
def test_windows(ctx, window, kind, out_type, hd):
    rng = np.random.default_rng(window)
    m = Model(ctx, kind, 2, hd)
    seqs = [m.new() for _ in range(4)]
    m.grow(seqs, [300, 1, 200, 64], rng)
    m.attend(seqs, [300, 1, 90, 2], rng, 6, window=window, out_type=out_type)
    kids = m.fork([seqs[0]] * 3, [300, 260, 256])
    m.grow(kids, [2, 1, 70], rng)
    m.attend(kids, [2, 1, 3], rng, 6, window=window, out_type=out_type)
    m.close()


@pytest.mark.parametrize("kind,q_type,out_type", TYPES)
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (16, 2, 256), (8, 1, 512), (5, 5, 24)])
def test_sequences_behind_a_shared_prefix(ctx, heads, kvh, hd, kind, q_type, out_type):
    rng = np.random.default_rng(hd)
    m = Model(ctx, kind, kvh, hd, pages=80, sequences=16)
    root = m.new()
    m.grow([root], [519], rng)
    kids = m.fork([root] * 5, [519, 519, 512, 300, 519])
    m.grow(kids, [1, 200, 30, 2, 64], rng)
    inner = m.fork([kids[1]] * 3, [719, 700, 719])  # a prefix of a prefix
    m.grow(inner, [1, 5, 9], rng)
    seqs = [root, kids[0]] + inner + [kids[4], kids[2], kids[3], kids[1]]
    for counts in ([1] * 9, [1, 2, 1, 5, 7, 3, 1, 2, 4]):
        m.attend(seqs, counts, rng, heads, q_type=q_type, out_type=out_type)
    m.close()


@pytest.mark.parametrize("positions", [1, 63, 5000, 70001])
@pytest.mark.parametrize("kind,out_type", [(BF16, F32), (F16, F32), (F16, F16)])
def test_single_tokens_over_long_caches(ctx, positions, kind, out_type):
    rng = np.random.default_rng(positions)
    m = Model(ctx, kind, 2, 64, pages=1100, sequences=2, context=80000)
    a = m.new()
    m.grow([a], [positions], rng)
    m.attend([a], [1], rng, 8, out_type=out_type)
    m.close()


@pytest.mark.parametrize("kind", [BF16, F16])
def test_a_long_prompt_in_parts(ctx, kind):
    """Chunks of a prompt over what is cached already, and its last rows at once."""
    rng = np.random.default_rng(9)
    m = Model(ctx, kind, 2, 128)
    a = m.new()
    for n in (700, 1, 513):
        m.grow([a], [n], rng)
        for out_type in (F32, kind):
            m.attend([a], [min(n, 150)], rng, 4, out_type=out_type)
    m.close()


@pytest.mark.parametrize("kind,q_type,out_type", [(BF16, F32, BF16), (F16, F16, F32), (BF16, F32, F32)])
def test_strides_and_alignments(ctx, kind, q_type, out_type):
    rng = np.random.default_rng(10)
    m = Model(ctx, kind, 2, 72)
    a, b = m.new(), m.new()
    m.grow([a, b], [70, 5], rng, pad=13, shift=1)
    for pad, shift in ((0, 1), (1, 0), (7, 3), (1000, 5)):
        m.attend([a, b], [40, 5], rng, 4, q_type=q_type, out_type=out_type, pad=pad, shift=shift)
    m.close()


@pytest.mark.parametrize("kind", [BF16, F16])
def test_queries_of_any_size_in_32_bits(ctx, kind):
    """F16 products of queries that F16 cannot hold, and of ones below its smallest value."""
    rng = np.random.default_rng(11)
    m = Model(ctx, kind, 1, 64)
    a = m.new()
    m.grow([a], [100], rng)
    for size in (1e6, 1e-9, 1e-30):
        q = rng.standard_normal((9, 2, 64)) * size
        for out_type in (F32, kind):
            m.attend([a], [9], rng, 2, q=q, scale=1.5 / (8 * size), out_type=out_type)
    m.attend([a], [9], rng, 2, q=np.zeros((9, 2, 64)))
    m.close()


def test_a_row_of_many_small_probabilities(ctx):
    """One key far ahead of 60000 equal ones that weigh 2^-22 each: together 1.4 % of the row."""
    rng = np.random.default_rng(12)
    m = Model(ctx, F16, 1, 64, pages=1000, context=64000)
    a = m.new()

    def make(which, layer, n):
        x = np.zeros((n, 1, 64))
        if which == 0:
            x[7, 0, 0] = 22 * np.log(2.0)
        else:
            x[:, 0] = 1.0 + rng.random((n, 64))
            x[7] = -1.0
        return x

    m.grow([a], [60000], rng, make=make)
    q = np.zeros((1, 2, 64))
    q[0, :, 0] = 1.0
    for out_type in (F32, F16):
        m.attend([a], [1], rng, 2, q=q, scale=1.0, out_type=out_type)
    m.close()


# ---- what is not seen, and what is not finite -----------------------------------------

@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("kind,out_type", [(BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)])
@pytest.mark.parametrize("hd", [24, 64, 72, 128, 136, 256, 264, 512])
def test_unseen_places_reach_no_result(ctx, bad, kind, out_type, hd):
    rng = np.random.default_rng(13)
    m = Model(ctx, kind, 1, hd, pages=30, sequences=6)
    old = m.new()
    m.grow([old], [30 * 64], rng, make=lambda which, layer, n: np.full((n, 1, hd), bad))
    m.release([old])  # every free page is full of it
    a, b = m.new(), m.new()
    m.grow([a, b], [200, 65], rng)
    m.attend([a, b], [200, 65], rng, 4, out_type=out_type)
    m.attend([a, b], [1, 1], rng, 4, out_type=out_type)
    # keys and values of later tokens, and ones that the window has passed
    c = m.new()

    def make(which, layer, n):
        x = rng.standard_normal((n, 1, hd))
        x[150:] = bad
        x[:20] = bad
        return x

    m.grow([c], [170], rng, make=make)
    q = rng.standard_normal((170, 2, hd)) * 1.5
    got = m.attend([c], [170], rng, 2, window=64, q=q, out_type=out_type, check=False)
    held = m.rows[c]
    m.rows[c] = [[x[:150] for x in layer] for layer in held]
    o, _, _, _ = m.expect([c], [150], from_bits(to_bits(q, F32), F32)[:150], 64, float(np.float32(1 / np.sqrt(hd))))
    fine = slice(83, 150)  # rows that see tokens 20 .. 149 alone
    assert np.isfinite(got[fine]).all()
    assert np.abs(got[fine] - o[fine]).max() <= (2e-4 if out_type == F32 else 0.1)
    m.rows[c] = held
    m.close()


def test_scores_that_are_not_finite_are_reported(ctx):
    rng = np.random.default_rng(14)
    for kind, out_type in ((BF16, F32), (F16, F16), (BF16, BF16)):
        m = Model(ctx, kind, 1, 64, pages=200, context=9000)
        a, b = m.new(), m.new()
        m.grow([a, b], [100, 8000], rng)
        q = rng.standard_normal((2, 2, 64))
        m.attend([a, b], [1, 1], rng, 2, q=q, out_type=out_type)
        ctx.attention_result()  # fine so far
        for at in (0, 1):  # a row of one unit, and one that is joined
            for value in (np.nan, np.inf):
                bad = q.copy()
                bad[at, 1, 3] = value
                got = m.attend([a, b], [1, 1], rng, 2, q=bad, out_type=out_type, check=False)
                expect_error("NonFinite", ctx.attention_result)
                good = m.attend([a, b], [1, 1], rng, 2, q=q, out_type=out_type)
                ctx.attention_result()
                assert np.array_equal(got[1 - at], good[1 - at]) and np.array_equal(got[at, 0], good[at, 0])
        expect_error("InvalidArgument", ctx.attention_result)
        m.close()


@pytest.mark.parametrize("kind,out_type", [(BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)])
def test_infinite_keys_and_values_that_are_seen(ctx, kind, out_type):
    """A key that scores -inf has no weight; an infinite value that has some makes its dim infinite."""
    rng = np.random.default_rng(15)
    m = Model(ctx, kind, 1, 64)
    a = m.new()

    def make(which, layer, n):
        x = np.abs(rng.standard_normal((n, 1, 64)))
        if which == 0:
            x[5, 0, 2] = -np.inf
        else:
            x[9, 0, 7] = np.inf
        return x

    m.grow([a], [70], rng, make=make)
    q = np.abs(rng.standard_normal((3, 2, 64))) * 0.2
    q[..., 2] = 0.5
    got = m.attend([a], [3], rng, 2, q=q, out_type=out_type, check=False)
    ctx.attention_result()
    assert (got[:, :, 7] == np.inf).all()
    seen = [np.delete(x, 5, axis=0) for x in m.rows[a][0]]
    seen[1][8, 0, 7] = 0.0
    m.rows[a] = [seen]
    got[:, :, 7] = 0.0
    o, _, _, _ = m.expect([a], [3], q, 0, float(np.float32(0.125)))
    o[:, :, 7] = 0.0
    assert np.abs(got - o).max() <= (1e-4 if out_type == F32 else 0.05)
    m.close()


def test_only_minus_infinite_scores_are_reported(ctx):
    rng = np.random.default_rng(16)
    m = Model(ctx, BF16, 1, 64)
    a = m.new()
    m.grow([a], [70], rng, make=lambda which, layer, n: np.full((n, 1, 64), -np.inf if which == 0 else 1.0))
    for out_type in (F32, BF16):
        m.attend([a], [3], rng, 2, q=np.ones((3, 2, 64)), out_type=out_type, check=False)
        expect_error("NonFinite", ctx.attention_result)
    m.close()


# ---- together, captured, refused ------------------------------------------------------

def test_a_serving_run(ctx):
    """Prompts, a shared prefix, decode steps, drafted tokens of which some are
    dropped, sequences that leave, compaction: every step's results, two layers."""
    rng = np.random.default_rng(17)
    m = Model(ctx, BF16, 2, 128, pages=120, sequences=12, layers=2)
    plan = m.pages.new_plan(8, None, F32, F32, 700)
    prompts = m.pages.new_plan(8, None, F32, BF16, 700)
    root = m.new()

    def step(seqs, counts, which=None):
        which = which or plan
        m.pages.extend(seqs, counts)
        which.set(seqs, counts)
        m.write(which, seqs, counts, rng)
        for layer in range(2):
            m.attend(seqs, counts, rng, 8, layer=layer, plan=which, out_type=BF16 if which is prompts else F32)

    step([root], [600], prompts)
    users = m.fork([root] * 4, [600] * 4)
    step(users, [50, 1, 130, 7], prompts)
    for _ in range(3):
        step(users, [1, 1, 1, 1])
    step(users, [5, 5, 5, 5])  # drafted
    for u, keep in zip(users, (1, 4, 2, 5)):
        n = m.pages.length(u) - 5 + keep
        m.pages.truncate(u, n)
        m.rows[u] = [[x[:n] for x in layer] for layer in m.rows[u]]
    step(users, [1, 1, 1, 1])
    best = m.fork([users[2], users[2], users[0]], [m.pages.length(users[2])] * 2 + [m.pages.length(users[0])])
    m.release([users[1], users[0], root])
    m.pages.compact()
    step(best + [users[3]], [1, 2, 1, 1])
    m.check_stored()
    ctx.attention_result()
    m.close()


class Graph:
    """A graph of what is enqueued on the context's stream, by the runtime that the library is linked to."""

    def __init__(self, ctx):
        self.hip = ctypes.CDLL("libamdhip64.so.7")
        self.stream = ctypes.c_void_p(load_library().dmhip_stream(ctx.handle))

    def __enter__(self):
        assert self.hip.hipStreamBeginCapture(self.stream, 0) == 0
        return self

    def __exit__(self, *exc):
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        assert self.hip.hipStreamEndCapture(self.stream, ctypes.byref(graph)) == 0
        assert self.hip.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0)) == 0
        assert self.hip.hipGraphDestroy(graph) == 0

    def replay(self):
        assert self.hip.hipGraphLaunch(self.exec, self.stream) == 0

    def free(self):
        assert self.hip.hipGraphExecDestroy(self.exec) == 0


@pytest.mark.parametrize("kind,out_type", [(BF16, F32), (BF16, BF16), (F16, F16)])
def test_captured_steps_follow_the_plan(ctx, kind, out_type):
    """One capture of a step, replayed for steps of other lengths, other
    sequences and other prefixes, each against the same calls made eagerly."""
    rng = np.random.default_rng(18)
    heads, kvh, hd, most = 8, 2, 64, 420
    m = Model(ctx, kind, kvh, hd, pages=150, sequences=12, context=3000)
    root = m.new()
    m.grow([root], [1000], rng)
    seqs = m.fork([root] * 4, [1000, 700, 1000, 64])
    plan = m.pages.new_plan(heads, None, F32, out_type, most)
    size = most * heads * hd * (4 if out_type == F32 else 2)
    k, v, q, o = (ctx.new_owned_buffer(n) for n in (most * kvh * hd * 4, most * kvh * hd * 4, most * heads * hd * 4, size))

    def calls():
        ctx.write_kv_pages_device(plan, 0, F32, k.device_ptr, kvh * hd, v.device_ptr, kvh * hd)
        ctx.attention_pages_device(plan, 0, 0.125, q.device_ptr, heads * hd, o.device_ptr, heads * hd)

    m.pages.extend(seqs, [1] * 4)
    plan.set(seqs, [1] * 4)
    with Graph(ctx) as graph:
        calls()
        for refused in (lambda: m.pages.extend(seqs, [1] * 4), lambda: m.pages.fork([root], [1]),
                        lambda: plan.set(seqs, [1] * 4), lambda: m.pages.compact(),
                        lambda: m.pages.new_plan(heads, None, F32, F32, 1),
                        lambda: ctx.new_kv_pages(kind, 1, 1, 8, 64, 1, 1)):
            expect_error("InvalidArgument", refused)
    assert [m.pages.length(s) for s in seqs] == [1001, 701, 1001, 65]
    for s in seqs:  # the capture's own token was enqueued by no one
        m.pages.truncate(s, m.pages.length(s) - 1)
    kids = None
    for names, counts in ((seqs, [1] * 4), (seqs[:1], [1]), (seqs, [1, 9, 40, 2]), (seqs[::-1], [1] * 4),
                          (kids, [1] * 3), (seqs[2:], [400, 1]), (seqs, [1] * 4)):
        if names is None:
            names = kids = m.fork([seqs[0]] * 3, [m.pages.length(seqs[0])] * 3)
        m.pages.extend(names, counts)
        plan.set(names, counts)
        n = sum(counts)
        for _ in range(2):
            new = [rng.standard_normal((n, w, hd)).astype(np.float32) for w in (kvh, kvh, heads)]
            for buf, x in zip((k, v, q), new):
                buf.write(0, x)
            o.write(0, np.full(size, 0x55, dtype=np.uint8))
            graph.replay()
            ctx.synchronize()
            replayed = o.as_bytes()
            used = n * size // most
            assert (replayed[used:] == 0x55).all()
            o.write(0, np.full(size, 0xAA, dtype=np.uint8))
            calls()
            ctx.synchronize()
            assert np.array_equal(o.as_bytes()[:used], replayed[:used])
        lo = 0
        for s, c in zip(names, counts):
            m.rows[s][0] = [np.concatenate([have, from_bits(to_bits(x[lo:lo + c], kind), kind)])
                            for have, x in zip(m.rows[s][0], new)]
            lo += c
        got = replayed[:used].view(np.float32).astype(np.float64) if out_type == F32 else \
            from_bits(replayed[:used].view(np.uint16), out_type)
        m.close_to(got.reshape(n, heads, hd), names, counts, new[2].astype(np.float64), 0, 0.125, F32, out_type)
    m.check_stored()
    graph.free()
    m.close()


def test_a_replayed_write_leaves_shared_pages_alone(ctx):
    rng = np.random.default_rng(19)
    m = Model(ctx, BF16, 2, 16, pages=20, sequences=6)
    root = m.new()
    m.grow([root], [128], rng)
    a, b = m.fork([root] * 2, [128, 128])
    plan = m.pages.new_plan(2, None, F32, F32, 4)
    k = m.device(rng.standard_normal((4, 32)).astype(np.float32))
    m.pages.extend([a], [1])
    plan.set([a], [1])
    with Graph(ctx) as graph:
        ctx.write_kv_pages_device(plan, 0, F32, k, 32, k, 32)
    m.pages.truncate(a, 128)
    for _ in range(3):
        plan.set([a, b], [2, 2])  # the root's own pages
        expect_error("InvalidArgument", ctx.write_kv_pages_device, plan, 0, F32, k, 32, k, 32)
        graph.replay()
        ctx.synchronize()
        m.check_stored()
    plan.free()
    graph.free()
    m.close()


def test_a_plan_is_refused_once_its_sequences_have_changed(ctx):
    m = Model(ctx, BF16, 1, 8, sequences=6)
    a, b, other = m.new(), m.new(), m.new()
    m.pages.extend([a, b, other], [100, 100, 100])
    plan = m.pages.new_plan(1, None, F32, F32, 200)
    buf = ctx.new_owned_buffer(200 * 8 * 4).device_ptr

    def calls():
        ctx.write_kv_pages_device(plan, 0, F32, buf, 8, buf, 8)
        ctx.attention_pages_device(plan, 0, 1.0, buf, 8, buf + 3200, 8)

    expect_error("InvalidArgument", calls)  # not set
    for change in (lambda: m.pages.extend([b], [1]), lambda: m.pages.truncate(b, 90), lambda: m.pages.fork([b], [50])):
        plan.set([a, b], [1, 2])
        calls()
        m.pages.extend([other], [1])  # not its own: no matter
        m.pages.extend([a], [0])
        calls()
        change()
        expect_error("InvalidArgument", calls)
    plan.set([a, b], [1, 2])
    m.pages.release([b])
    expect_error("InvalidArgument", calls)
    assert m.pages.new_sequence() == b  # the number again, another sequence
    expect_error("InvalidArgument", calls)
    # tokens in shared pages are read, not written
    kid = m.pages.fork([a], [64])[0]
    plan.set([kid], [1])
    expect_error("InvalidArgument", ctx.write_kv_pages_device, plan, 0, F32, buf, 8, buf, 8)
    ctx.attention_pages_device(plan, 0, 1.0, buf, 8, buf + 3200, 8)
    ctx.synchronize()
    plan.set([a], [1])
    m.close()
    expect_error("InvalidArgument", calls)
    expect_error("InvalidArgument", plan.set, [a], [1])
    plan.free()


def test_refusals(ctx):
    for args, variant in [((F32, 1, 1, 8, 64, 1, 1), "UnsupportedTensorType"), ((12, 1, 1, 8, 64, 1, 1), "UnsupportedTensorType"),
                          ((BF16, 0, 1, 8, 64, 1, 1), "InvalidAttentionShape"), ((BF16, 1, 0, 8, 64, 1, 1), "InvalidAttentionShape"),
                          ((BF16, 1, 1, 0, 64, 1, 1), "InvalidAttentionShape"), ((BF16, 1, 1, 12, 64, 1, 1), "InvalidAttentionShape"),
                          ((BF16, 1, 1, 520, 64, 1, 1), "InvalidAttentionShape"), ((BF16, 1, 1, 8, 0, 1, 1), "InvalidAttentionShape"),
                          ((BF16, 1, 1, 8, 64, 0, 1), "InvalidAttentionShape"), ((BF16, 1, 1, 8, 64, 1, 0), "InvalidAttentionShape"),
                          ((BF16, 1, 1, 8, 2 ** 31, 1, 1), "VectorTooLarge"), ((BF16, 1, 1, 8, 64, 2 ** 31, 1), "VectorTooLarge"),
                          ((BF16, 1, 1, 8, 2 ** 30, 1, 2 ** 8), "VectorTooLarge"), ((BF16, 1, 2 ** 16, 8, 64, 1, 1), "VectorTooLarge"),
                          ((BF16, 1, 32768, 512, 64, 1, 1), "VectorTooLarge"), ((BF16, 2 ** 16, 1, 8, 64, 1, 1), "VectorTooLarge"),
                          ((BF16, 65535, 1024, 512, 64, 2 ** 30, 1), "Overflow"), ((BF16, 1, 1024, 512, 64, 2 ** 20, 1), "BufferAllocation")]:
        expect_error(variant, ctx.new_kv_pages, *args)
    p = ctx.new_kv_pages(BF16, 2, 2, 16, 130, 5, 3)
    a = p.new_sequence()
    expect_error("InvalidArgument", p.extend, [a, a], [1, 1])
    expect_error("InvalidArgument", p.extend, [1], [1])
    expect_error("InvalidArgument", p.release, [2])
    expect_error("InvalidArgument", p.truncate, 2, 0)
    expect_error("InvalidArgument", p.page_ids, 9)
    e = expect_error("KvContext", p.extend, [a], [131])
    assert e.detail["limit"] == 130 and e.detail["position"] == 131
    p.extend([a], [130])
    b = p.new_sequence()
    e = expect_error("BufferAllocation", p.extend, [b], [129])
    assert e.detail["bytes"] == p.page_bytes() * 2
    expect_error("KvContext", p.fork, [a], [131])
    expect_error("NoSlots", p.fork, [a, a], [1, 1])
    p.extend([b], [100])
    expect_error("BufferAllocation", p.fork, [a], [1])
    p.fork([a], [128])
    expect_error("NoSlots", p.new_sequence)
    assert p.layer_ptr(2) == 0 and p.layer_ptr(1) - p.layer_ptr(0) == 5 * p.page_bytes()
    assert p.allocated_bytes() == 10 * p.page_bytes() and p.length(77) == 0
    for args, variant in [((3, None, F32, F32, 9), "InvalidAttentionShape"), ((0, None, F32, F32, 9), "InvalidAttentionShape"),
                          ((4, 0, F32, F32, 9), "EmptyInput"), ((4, None, F16, F32, 9), "UnsupportedTensorType"),
                          ((4, None, F32, 12, 9), "UnsupportedTensorType"), ((4, None, F32, F32, 0), "EmptyInput"),
                          ((4, None, F32, F32, 2 ** 30), "VectorTooLarge"),
                          ((2, None, F32, F32, 2 ** 30 - 1), "VectorTooLarge")]:  # lists of 6 GiB
        expect_error(variant, p.new_plan, *args)
    plan = p.new_plan(4, None, F32, BF16, 9)
    expect_error("EmptyInput", plan.set, [a], [0])
    expect_error("EmptyInput", plan.set, [], [])
    expect_error("KvContext", plan.set, [a], [131])
    expect_error("InvalidVectorLength", plan.set, [a], [10])
    expect_error("InvalidArgument", plan.set, [a, a], [1, 1])
    expect_error("InvalidArgument", plan.set, [7], [1])
    plan.set([a, b], [1, 3])
    buf = ctx.new_owned_buffer(1 << 16).device_ptr
    ok = (plan, 1, 1.0, buf, 64, buf + 32768, 64)
    for i, value, variant in [(1, 2, "InvalidLayer"), (2, 0.0, "InvalidPositiveParameter"), (2, -1.0, "InvalidPositiveParameter"),
                              (2, float("nan"), "InvalidPositiveParameter"), (2, float("inf"), "InvalidPositiveParameter"),
                              (2, 2.0 ** 127, "InvalidPositiveParameter"),
                              (3, 0, "InvalidArgument"), (3, buf + 2, "InvalidArgument"), (4, 63, "InvalidVectorLength"),
                              (5, 0, "InvalidArgument"), (5, buf + 1, "InvalidArgument"), (6, 63, "InvalidVectorLength")]:
        args = list(ok)
        args[i] = value
        expect_error(variant, ctx.attention_pages_device, *args)
    ctx.attention_pages_device(*ok)
    ok = (plan, 0, F32, buf, 32, buf, 32)
    for i, value, variant in [(1, 2, "InvalidLayer"), (2, F16, "UnsupportedTensorType"), (2, 12, "UnsupportedTensorType"),
                              (3, 0, "InvalidArgument"), (3, buf + 2, "InvalidArgument"), (4, 31, "InvalidVectorLength"),
                              (5, 0, "InvalidArgument"), (6, 31, "InvalidVectorLength")]:
        args = list(ok)
        args[i] = value
        expect_error(variant, ctx.write_kv_pages_device, *args)
    lib = load_library()
    assert lib.dmhip_kv_plan_set(plan.handle, 1, None, None) == 24
    assert lib.dmhip_kv_sequences_extend(p.handle, 1, None, None) == 24
    assert lib.dmhip_kv_sequences_extend(p.handle, 0, None, None) == 0
    assert lib.dmhip_new_kv_plan(None, 1, 0, 0, 0, 0, 1, None) == 24
    lib.dmhip_kv_pages_free(None)
    lib.dmhip_kv_plan_free(None)
    ctx.synchronize()
    plan.free()
    p.free()


def test_another_context_is_refused(ctx):
    from diskmule_amd import HipContext
    other = HipContext(0)
    p = ctx.new_kv_pages(BF16, 1, 1, 8, 64, 1, 1)
    s = p.new_sequence()
    p.extend([s], [1])
    plan = p.new_plan(1, None, F32, F32, 1)
    plan.set([s], [1])
    buf = ctx.new_owned_buffer(4096).device_ptr
    expect_error("InvalidArgument", other.write_kv_pages_device, plan, 0, F32, buf, 8, buf, 8)
    expect_error("InvalidArgument", other.attention_pages_device, plan, 0, 1.0, buf, 8, buf, 8)
    plan.free()
    p.free()
    other.close()
