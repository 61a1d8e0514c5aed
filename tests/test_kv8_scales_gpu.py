"""The paged 8-bit attention where the V scales of a request's pages differ by many orders of magnitude, and where keys that a
row does not see hold anything: the error is measured against what the row itself attends to.

Bounds. W of a row and head = the sum over pages of (the row's softmax weight on the page) * (the largest |value| of V in
the page): the size of what is added up. fp32: q and the weights as fp16 pairs, scores up to 40: 4e-5 * W. fp16 / bf16: the
weights are rounded to fp16 and the output to its type: 2^-10 * W + 2^-10 / 2^-8 * |out|, and half of fp16's smallest step."""
import math

import pytest

from test_kv8_gpu import Batch, T, ref  # noqa: F401  (T and ref are fixtures)

pytestmark = pytest.mark.gpu


def sizes(b, ref):  # noqa: F811
    """W [tokens][query heads] in float64."""
    T, c = b.T, b.cache  # noqa: F811
    hq, page = b.hq, c.page
    W = T.zeros(b.n_tokens, hq, dtype=T.float64, device="cuda")
    q = b.q.reshape(b.n_tokens, hq, c.hd).double()
    for r, (kv, n) in enumerate(b.lens):
        if kv == 0 or n == 0:
            continue
        ids = T.tensor(b.table[r][:-(-kv // page)], device="cuda")
        K = (ref.values(c.k[ids], c.fmt) * c.ks[ids].double()[:, :, None, None]).transpose(1, 2).reshape(-1, c.hkv, c.hd)[:kv]
        big = ref.values(c.v[ids], c.fmt).abs().amax((2, 3)) * c.vs[ids].double()  # [pages][hkv]
        key = T.arange(kv, device="cuda")
        at = kv - n + T.arange(n, device="cuda")[:, None]
        hide = key > at
        if b.window > 0:
            hide = hide | (key <= at - b.window)
        rows = slice(b.start[r], b.start[r + 1])
        for h in range(hq):
            g = h // (hq // c.hkv)
            p = T.softmax((q[rows, h] @ K[:, g].T * b.scale).masked_fill(hide, -math.inf), 1).nan_to_num(0.0)
            W[rows, h] = p @ big[:, g].repeat_interleave(page)[:kv]
    return W


def check(b, ref):  # noqa: F811
    T = b.T  # noqa: F811
    out, lse = b.run()
    T.cuda.synchronize()
    want, wlse = b.want(ref)
    W = sizes(b, ref)[:, :, None]
    got = out.reshape(want.shape).double()
    tol = 4e-5 * W if b.type == 0 else 2.0 ** -10 * W + (2.0 ** -10 if b.type == 1 else 2.0 ** -8) * want.abs()
    if b.type == 1:
        tol = tol + 2.0 ** -25
    over = (got - want).abs() - tol
    if b.type == 1:  # past fp16's largest number the output is infinite
        over = T.where((want.abs() > 65504 * (1 - 2.0 ** -9)) & (got == want.sign() * math.inf), -1.0, over)
    assert bool((over <= 0).all()), ((got - want).abs() / W.clamp(min=1e-300)).max().item()
    assert bool(((lse.double() - wlse).abs() <= 4e-5 * wlse.abs().clamp(min=1)).all())


SHAPES = [(8, 2, 128, 32), (4, 1, 64, 16), (8, 2, 256, 64)]


@pytest.mark.parametrize("hq,hkv,hd,page", SHAPES)
@pytest.mark.parametrize("n", [1, 5, 60])
@pytest.mark.parametrize("type", [0, 1, 2])
@pytest.mark.parametrize("power", [14, 27])
def test_a_page_of_large_values_that_gets_little_weight(fb, T, ref, hq, hkv, hd, page, n, type, power):  # noqa: F811
    """One page's V scale is 2^power times the others', its scores are 0, and the others' largest are about 25 to 35."""
    for fmt in (0, 1):
        b = Batch(fb, T, [(1000, n), (200, n)], hq, hkv, hd, page, fmt, type, q_scale=8.0 if fmt == 0 else 4.0)
        for r in (0, 1):
            p = b.table[r][2 + r]
            b.cache.k[p] = 0
            b.cache.vs[p] *= 2.0 ** (power if type != 1 else power - 14)  # fp16 outputs: the others smaller instead
        if type == 1:
            for r in (0, 1):
                for j, p in enumerate(b.table[r][:-(-b.lens[r][0] // page)]):
                    if j != 2 + r:
                        b.cache.vs[p] *= 2.0 ** -14 * 4096  # still normal numbers of fp16
                    else:
                        b.cache.vs[p] *= 4096
        check(b, ref)


@pytest.mark.parametrize("hq,hkv,hd,page", SHAPES)
@pytest.mark.parametrize("n", [1, 5, 60])
@pytest.mark.parametrize("type", [0, 2])
@pytest.mark.parametrize("step", [-3, 3])
def test_scales_that_rise_or_fall_along_the_request(fb, T, ref, hq, hkv, hd, page, n, type, step):  # noqa: F811
    """V scales that change by 2^3 from page to page, under scores that grow against them page by page, and with them."""
    for grow in (0.0, 1.0):
        b = Batch(fb, T, [(14 * page, n), (9 * page + 3, n)], hq, hkv, hd, page, 0, type, q_scale=0.25)
        for r in (0, 1):
            for j, p in enumerate(b.table[r][:-(-b.lens[r][0] // page)]):
                b.cache.vs[p] *= 2.0 ** (step * (j - 7))
                b.cache.ks[p] *= 1 + grow * 2 * j
        check(b, ref)


@pytest.mark.parametrize("type", [0, 1, 2])
@pytest.mark.parametrize("n", [1, 5, 60])
def test_one_request_split_over_many_blocks(fb, T, ref, type, n):  # noqa: F811
    """A long request whose parts, joined at the end, have seen V scales of very different size."""
    b = Batch(fb, T, [(6000, n)], 8, 2, 128, 16, 0, type, q_scale=6.0)
    pages = b.table[0][:375]
    for j, p in enumerate(pages):
        if 100 <= j < 140:  # the largest values under scores of zero
            b.cache.k[p] = 0
            b.cache.vs[p] *= 2.0 ** 10
        elif j >= 300:
            b.cache.vs[p] *= 2.0 ** -8
    check(b, ref)


@pytest.mark.parametrize("hq,hkv,hd,page", SHAPES)
@pytest.mark.parametrize("type", [0, 1, 2])
@pytest.mark.parametrize("n", [5, 12, 200])
def test_what_a_row_does_not_see_does_not_change_a_bit(fb, T, ref, hq, hkv, hd, page, type, n):  # noqa: F811
    """The codes and scales of the last page: rows that stand before it stay as they were, to the bit."""
    kv = 320 + 3 if n > 12 else 64 + 3
    b = Batch(fb, T, [(kv, n), (kv + 1, n)], hq, hkv, hd, page, 0, type, q_scale=2.0)
    want = [x.clone() for x in b.run()]
    blind = []
    for r, (L, m) in enumerate(b.lens):
        first = (L - 1) // page * page  # the last page's first position
        blind += [b.start[r] + i for i in range(m) if L - m + i < first]
        p = b.table[r][first // page]
        b.cache.vs[p] *= 2.0 ** 20
        b.cache.ks[p] *= 30.0
        b.cache.k[p], b.cache.v[p] = b.cache.k[p].flip(-1).clone(), b.cache.v[p].flip(-1).clone()
    assert blind
    got = b.run()
    for g, w in zip(got, want):
        assert T.equal(g[blind], w[blind])


@pytest.mark.parametrize("n", [1, 60])
@pytest.mark.parametrize("type", [0, 2])
def test_scales_at_the_ends_of_the_float_range(fb, T, ref, n, type):  # noqa: F811
    """All V scales near the smallest and near the largest normal numbers, and pages of zeros among them."""
    for f in (2.0 ** -118, 2.0 ** 118):
        b = Batch(fb, T, [(300, n), (100, n)], 8, 2, 128, 32, 0, type)
        b.cache.vs *= f
        p = b.table[0][1]
        b.cache.v[p], b.cache.vs[p] = 0, 0
        check(b, ref)


@pytest.mark.parametrize("type", [1, 2])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 1, 128), (4, 1, 64), (4, 1, 256)])
def test_sums_over_very_many_keys_are_not_biased(fb, T, ref, type, hq, hkv, hd):  # noqa: F811
    """131000 keys under many rows, so that a block of threads goes through all of them, positive values: the mean relative error,
    in which roundings to nearest cancel, stays below half a step of the output type (2^-12 for fp16)."""
    kv, n = 131000, 16384 if hd != 256 else 8192
    b = Batch(fb, T, [(kv, n)], hq, hkv, hd, 64, 0, type, q_scale=0.5)
    c = b.cache
    c.v = c.v.view(T.int8).abs().view(T.uint8)
    c.vs.fill_(2.0 ** -7)
    out, _ = b.run()
    ids = T.tensor(b.table[0][:-(-kv // 64)], device="cuda")
    K = (ref.values(c.k[ids], 0) * c.ks[ids].double()[:, :, None, None])[:, 0].reshape(-1, hd)[:kv]
    V = (ref.values(c.v[ids], 0) * 2.0 ** -7)[:, 0].reshape(-1, hd)[:kv]
    off = []
    for r0 in range(0, n, 2048):
        rows = T.arange(r0, r0 + 32, device="cuda")
        x = b.q.reshape(n, hq, hd)[rows, 3].double() @ K.T * b.scale
        w = T.softmax(x.masked_fill(T.arange(kv, device="cuda") > (kv - n + rows)[:, None], -math.inf), 1) @ V
        off.append((out.reshape(n, hq, hd)[rows, 3].double() - w) / w)
    assert abs(T.cat(off).mean().item()) < 2.0 ** -12


def rows_of(b, ref, rows, heads):  # noqa: F811
    """The definition for some rows of a request alone in its batch: (got - want, want, W) [rows][heads][head_dim or 1]."""
    T, c, kv, n = b.T, b.cache, *b.lens[0]  # noqa: F811
    ids = T.tensor(b.table[0][:-(-kv // c.page)], device="cuda")
    G, at = b.hq // c.hkv, (kv - n + rows)[:, None]
    key = T.arange(kv, device="cuda")
    hide = (key > at) | (key <= at - b.window) if b.window > 0 else key > at
    got, want, W = [], [], []
    for h in heads:
        K = (ref.values(c.k[ids, h // G], c.fmt) * c.ks[ids, h // G].double()[:, None, None]).reshape(-1, c.hd)[:kv]
        V = (ref.values(c.v[ids, h // G], c.fmt) * c.vs[ids, h // G].double()[:, None, None]).reshape(-1, c.hd)[:kv]
        x = b.q.reshape(n, b.hq, c.hd)[rows, h].double() @ K.T * b.scale
        p = T.softmax(x.masked_fill(hide, -math.inf), 1)
        want.append(p @ V)
        W.append(p @ V.abs().amax(1, keepdim=True))
        got.append(b.out.reshape(n, b.hq, c.hd)[rows, h].double())
    return T.stack(got, 1) - T.stack(want, 1), T.stack(want, 1), T.stack(W, 1)


@pytest.mark.parametrize("hd,hq,hkv,type", [(64, 32, 4, 1), (128, 64, 8, 2), (256, 16, 4, 1)])
@pytest.mark.parametrize("window", [0, 33000])
def test_parts_longer_than_the_sums_stay_in_one_place(fb, T, ref, hd, hq, hkv, type, window):  # noqa: F811
    """Rows at positions around 32768 (with a window, from further on), where one half of a group of rows has a tile more than
    the other: the sums leave tensor memory there."""
    kv, n = (34816, 4096) if window == 0 else (70016, 4096)
    b = Batch(fb, T, [(kv, n)], hq, hkv, hd, 128, 0, type, window=window, q_scale=2.0)
    for j, p in enumerate(b.table[0][:kv // 128]):
        b.cache.vs[p] *= 1 + j % 5
    b.run()
    rows = T.arange(2048 - 160, 2048 + 160, 3, device="cuda")
    off, want, W = rows_of(b, ref, rows, (0, hq // 2 + 1, hq - 1))
    tol = 2.0 ** -10 * W + (2.0 ** -10 if type == 1 else 2.0 ** -8) * want.abs()
    assert bool((off.abs() <= tol).all()), (off.abs() / W).max().item()


@pytest.mark.parametrize("window", [0, 900, 1100, 1500, 2600])
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64)])
def test_fp32_rows_over_many_drains(fb, T, ref, hd, page, window):  # noqa: F811
    """fp32 prompts and chunks of many tiles, with windows whose first and last tiles fall anywhere between two drains."""
    lens = [(4000 + 128 * i + 37 * i, 60 + 11 * i) for i in range(8)]
    check(Batch(fb, T, lens, 8, 2, hd, page, 0, 0, window=window, q_scale=2.0), ref)
