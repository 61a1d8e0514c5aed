"""The batched-serving operators over a paged 8-bit KV cache (csrc/paged_plan.cu, kv8_store.cu, kv8_attn.cu)
against plain implementations (tests/kv8_ref.py).

Bounds. plan, load: equal. store: equal to the same float32 operations one at a time, and within half a
code step of the row (first writing). attention, with V the largest |value| in the cache: fp32 carries q
and the softmax weights as fp16 pairs (22 bits) and exp2 to 2^-22, scores up to about 40 in size, so
40 * 2^-21 = 2e-5, twice that allowed: 4e-5 * V. fp16 / bf16: the weights are rounded to fp16
(2^-11 of their sum, times V) and the output to its type (2^-11 / 2^-8 of itself, half of it to
nearest): 2^-10 * V + 2^-10 / 2^-8 * |out|. lse: 4e-5 * max(1, |lse|)."""
import ctypes
import math
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DT = {0: "float32", 1: "float16", 2: "bfloat16"}


@pytest.fixture(scope="module")
def T():
    import torch
    assert torch.cuda.is_available()
    return torch


@pytest.fixture(scope="module")
def ref():
    import kv8_ref
    return kv8_ref


def stream(T):
    return T.cuda.current_stream().cuda_stream


def i32(T, v):
    return T.tensor(v, dtype=T.int32, device="cuda")


# ------------------------------------------------------------------ plan
def run_plan(fb, T, ctx, new, table, free, n_tokens, page, max_pages, n_pages):
    n = len(ctx)
    cap = min(n_tokens, 2 * n + n_tokens // page)
    e = lambda *s: T.full(s, -77, dtype=T.int32, device="cuda")  # noqa: E731
    buf = dict(ctx_len=i32(T, ctx), new_len=i32(T, new), block_table=i32(T, table), n_free=i32(T, [len(free)]),
               free_pages=i32(T, list(free) + [-5] * (n_pages - len(free))), n_free_out=e(1), ctx_out=e(n), kv_len=e(n),
               new_start=e(n + 1), slot=e(max(1, n_tokens)), pos=e(max(1, n_tokens)), touch=e(max(1, cap), 4))
    b = fb.PagedBatch()
    b.n_req, b.n_tokens, b.page_tokens, b.max_pages, b.n_pages, b.n_touch = n, n_tokens, page, max_pages, n_pages, cap
    for k, v in buf.items():
        setattr(b, k, v.data_ptr())
    fb.call("fence_paged_plan", b, stream(T))
    T.cuda.synchronize()
    got = {k: v.tolist() for k, v in buf.items()}
    got["touch"] = got["touch"][:cap]
    got["slot"], got["pos"] = got["slot"][:n_tokens], got["pos"][:n_tokens]
    return got


def check_plan(fb, T, ref, ctx, new, page, max_pages, spare, extra_tokens=0, seed=0):
    rng = random.Random(seed)
    held = [ref.ceil(c, page) for c in ctx]
    ids = list(range(sum(held) + spare))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-3] * (max_pages - h))
        at += h
    free = ids[at:]
    n_tokens = sum(max(0, n) for n in new) + extra_tokens
    want = ref.plan(ctx, new, table, free, n_tokens, page, max_pages, max(1, len(ids)))
    got = run_plan(fb, T, ctx, new, table, free, n_tokens, page, max_pages, max(1, len(ids)))
    for k in ("n_free_out", "ctx_out", "kv_len", "new_start", "slot", "pos", "block_table"):
        assert got[k] == want[k], k
    assert got["free_pages"][:len(want["stack"])] == want["stack"]
    touched = len(want["touch"])
    assert got["touch"][:touched] == want["touch"]
    assert all(t == [-1, 0, 0, 0] for t in got["touch"][touched:])
    return want


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_plan_page_edges(fb, T, ref, page):
    """Contexts and new lengths around page boundaries, empty requests among them."""
    ctx = [0, 0, 0, 1, page - 1, page, page + 1, 2 * page - 1, 5, 0, 3 * page, page]
    new = [0, 1, page, 0, 1, 1, page - 1, 2 * page + 1, page, 3 * page + 7, 0, 2]
    check_plan(fb, T, ref, ctx, new, page, 9, 40)


def test_plan_one_request_and_padding(fb, T, ref):
    check_plan(fb, T, ref, [0], [1], 16, 1, 1)
    check_plan(fb, T, ref, [0], [0], 16, 1, 1)
    check_plan(fb, T, ref, [37], [1], 16, 4, 0, extra_tokens=9)
    check_plan(fb, T, ref, [10], [-1], 16, 4, 2)


def test_plan_pool_runs_out(fb, T, ref):
    """In request order: the first that does not get its pages, and all later ones that need some, wait."""
    want = check_plan(fb, T, ref, [16, 3, 0, 16, 0, 8], [1, 2, 64, 1, 1, 4], 16, 8, 3)
    assert want["kv_len"] == [17, 5, 0, 0, 0, 12]
    check_plan(fb, T, ref, [16, 3], [1, 2], 16, 8, 0)


def test_plan_ended_requests_pages_are_handed_out(fb, T, ref):
    want = check_plan(fb, T, ref, [33, 20, 16, 0], [-1, 30, 1, 40], 16, 8, 2)
    assert want["kv_len"] == [0, 50, 17, 0] and want["n_free_out"] == [2]
    check_plan(fb, T, ref, [100, 0, 50], [-1, 1, -1], 16, 8, 0)


def test_plan_too_long_for_its_table(fb, T, ref):
    want = check_plan(fb, T, ref, [30, 60, 64], [3, 5, 0], 16, 4, 10)
    assert want["kv_len"] == [33, 0, 64]


@pytest.mark.parametrize("seed", range(12))
def test_plan_random(fb, T, ref, seed):
    rng = random.Random(seed)
    page = rng.choice([16, 32, 64, 128])
    n = rng.choice([1, 2, 7, 100, 511, 513, 1024, 1025, 3000, 4096])
    most = rng.choice([4, 20])
    ctx = [rng.randint(0, most * page) for _ in range(n)]
    new = [rng.choice([-1, 0, 1, 1, 1, 1, 3, page, rng.randint(0, 3 * page)]) for _ in range(n)]
    check_plan(fb, T, ref, ctx, new, page, most + 2, rng.choice([0, 3, n, 3 * n]), extra_tokens=rng.randint(0, 5), seed=seed)


def test_plan_lengths_out_of_range_are_reported(fb, T):
    """More new tokens than the buffers hold, and a free count past the pool: the word is set, nothing is written past."""
    got = run_plan(fb, T, [0, 0], [3, 9], [[-3], [-3]], [0, 1, 2], 5, 16, 1, 3)
    assert fb.lib().fence_device_error() == -1
    assert len(got["slot"]) == 5
    n_free = T.tensor([99], dtype=T.int32, device="cuda")
    b = fb.PagedBatch()
    bufs = [T.zeros(64, dtype=T.int32, device="cuda") for _ in range(11)]
    b.n_req, b.n_tokens, b.page_tokens, b.max_pages, b.n_pages, b.n_touch = 1, 1, 16, 1, 3, 1
    for k, t in zip(("ctx_len", "new_len", "block_table", "free_pages", "n_free_out", "ctx_out", "kv_len", "new_start", "slot", "pos",
                     "touch"), bufs):
        setattr(b, k, t.data_ptr())
    b.n_free = n_free.data_ptr()
    fb.call("fence_paged_plan", b, stream(T))
    assert fb.lib().fence_device_error() == -1


# ------------------------------------------------------------------ caches
class Cache:
    """A cache of random codes with its struct."""

    def __init__(self, fb, T, n_pages, hkv, page, hd, fmt, seed=0):
        g = T.Generator(device="cuda").manual_seed(seed)
        shape = (n_pages, hkv, page, hd)
        self.fmt, self.page, self.hkv, self.hd, self.n_pages = fmt, page, hkv, hd, n_pages
        if fmt == 0:
            mk = lambda: T.randint(-127, 128, shape, generator=g, device="cuda", dtype=T.int8).view(T.uint8)  # noqa: E731
        else:
            mk = lambda: (T.randn(shape, generator=g, device="cuda") * 120).clamp(-448, 448).to(T.float8_e4m3fn).view(T.uint8)  # noqa: E731
        self.k, self.v = mk(), mk()
        mks = lambda: T.rand(n_pages, hkv, generator=g, device="cuda") * 0.02 + 0.005  # noqa: E731
        self.ks, self.vs = mks(), mks()
        if fmt == 1:
            self.ks *= 0.3
            self.vs *= 0.3
        self.fb = fb

    def struct(self):
        c = self.fb.KV8Cache()
        c.k, c.v, c.k_scale, c.v_scale = self.k.data_ptr(), self.v.data_ptr(), self.ks.data_ptr(), self.vs.data_ptr()
        c.n_pages, c.n_kv_heads, c.page_tokens, c.head_dim, c.format = self.n_pages, self.hkv, self.page, self.hd, self.fmt
        return c


# ------------------------------------------------------------------ store, load
def run_store(fb, T, cache, touch, k, v, type, n_tokens, n_req=4096):
    b = fb.PagedBatch()
    b.n_req, b.n_tokens, b.page_tokens, b.max_pages, b.n_pages = n_req, n_tokens, cache.page, 1, cache.n_pages
    t = i32(T, touch)
    b.n_touch, b.touch = len(touch), t.data_ptr()
    fb.call("fence_kv8_store", cache.struct(), b, k.data_ptr(), v.data_ptr(), type, k.stride(0), v.stride(0), stream(T))
    T.cuda.synchronize()


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("type", [0, 1, 2])
@pytest.mark.parametrize("hkv,hd,page", [(8, 128, 16), (1, 64, 64), (3, 256, 128), (2, 128, 128), (5, 64, 32)])
def test_store_matches_float32_steps(fb, T, ref, fmt, type, hkv, hd, page):
    cache = Cache(fb, T, 9, hkv, page, hd, fmt, seed=hd + page)
    dt = getattr(T, DT[type])
    # page, first row, first token, rows: whole pages, one row, the last row, a part in the middle
    touch = [[3, 0, 0, page], [7, page - 1, page, 1], [0, 5, page + 1, 7], [-1, 0, 0, 0], [8, 0, page + 8, 1], [5, 0, page + 9, page - 3]]
    n = 2 * page + 6
    g = T.Generator(device="cuda").manual_seed(1)
    qkv = T.randn(n, 4 + 2 * hkv * hd + 12, generator=g, device="cuda")
    qkv[page] *= 40  # a row that makes its page's scale grow
    qkv[page + 1:page + 8] *= 0.01  # rows below their page's scale
    qkv = qkv.to(dt)
    off = 4 if type != 1 else 0  # a first element that is not 16-byte aligned in some of the types
    k, v = qkv[:, off:off + hkv * hd], qkv[:, off + hkv * hd:off + 2 * hkv * hd]
    was = [x.clone() for x in (cache.k, cache.ks, cache.v, cache.vs)]
    run_store(fb, T, cache, touch, k, v, type, n)
    for codes, scale, c0, s0, rows in ((cache.k, cache.ks, was[0], was[1], k), (cache.v, cache.vs, was[2], was[3], v)):
        want_c, want_s = c0.cpu().clone(), s0.cpu().clone()
        x = rows.float().cpu().reshape(n, hkv, hd)
        for p, first, at, cnt in touch:
            for h in range(hkv if p >= 0 else 0):
                c, s = ref.store_page(c0[p, h].cpu(), s0[p, h].item(), x[at:at + cnt, h], first, fmt)
                want_c[p, h], want_s[p, h] = c, float(s)
        assert T.equal(scale.cpu(), want_s)
        assert T.equal(codes.cpu(), want_c)
        # a page written from row 0 on: every value within half a step of the row
        val = (ref.values(codes[3], fmt) * scale[3].double()[:, None, None]).cpu()
        err = (val - x[:page].transpose(0, 1).double()).abs()
        step = scale[3].double().cpu()[:, None, None]
        if fmt == 1:  # 3 mantissa bits; subnormals below 2^-6
            step = T.maximum(x[:page].transpose(0, 1).double().abs() * 2.0 ** -3, step * 2.0 ** -9)
        assert bool((err <= 0.5 * step * (1 + 1e-5)).all())


@pytest.mark.parametrize("fmt", [0, 1])
def test_store_zero_and_non_finite(fb, T, ref, fmt):
    """A page of zeros, one of tiny values, NaN, infinity; then a finite row after them."""
    page, hd = 16, 64
    cache = Cache(fb, T, 6, 1, page, hd, fmt)
    x = T.zeros(7, hd, device="cuda")
    x[1] = 1e-38 / 448
    x[2, 3] = math.nan
    x[3, 9] = math.inf
    x[4, 9] = -math.inf
    x[5] = 3.0e38
    x[6] = 2.0
    touch = [[0, 0, 0, 1], [1, 0, 1, 1], [2, 0, 2, 1], [3, 0, 3, 1], [4, 0, 4, 1], [5, 0, 5, 1]]
    run_store(fb, T, cache, touch, x, x, 0, 7)
    s = cache.ks[:, 0].tolist()
    assert s[0] == 0 and s[1] == 0 and math.isnan(s[2]) and s[3] == s[4] == math.inf
    assert s[5] == np.float32(3.0e38) * np.float32(1 / ref.LIMIT[fmt])
    assert not cache.k[:5, 0, 0].any()
    assert (ref.values(cache.k[5, 0, 0], fmt) == ref.LIMIT[fmt]).all()
    run_store(fb, T, cache, [[0, 1, 6, 1], [2, 1, 6, 1], [3, 1, 6, 1]], x, x, 0, 7)
    s = cache.ks[:, 0].tolist()
    assert s[0] == np.float32(2.0) * np.float32(1 / ref.LIMIT[fmt]) and math.isnan(s[2]) and s[3] == math.inf
    assert not cache.k[0, 0, 0].any() and (ref.values(cache.k[0, 0, 1], fmt) == ref.LIMIT[fmt]).all()
    run_store(fb, T, cache, [[2, 0, 6, 1]], x, x, 0, 7)  # the page starts anew
    assert cache.ks[2, 0].item() == s[0]


def test_store_grows_row_by_row(fb, T, ref):
    """Row after row, each larger than the page's largest so far: every growth rounds the older rows once."""
    page, hd = 16, 128
    for fmt in (0, 1):
        cache = Cache(fb, T, 1, 1, page, hd, fmt)
        x = T.randn(page, hd, generator=T.Generator(device="cuda").manual_seed(5), device="cuda")
        x *= T.linspace(1, 9, page, device="cuda")[:, None]
        c, s = cache.k[0, 0].cpu(), 0.0
        for i in range(page):
            run_store(fb, T, cache, [[0, i, i, 1]], x, x, 0, page)
            c, s = ref.store_page(c, s, x[i:i + 1].cpu(), i, fmt)
            assert T.equal(cache.k[0, 0].cpu(), c) and cache.ks[0, 0].item() == s


def test_store_refuses_bad_pages_on_the_device(fb, T):
    cache = Cache(fb, T, 3, 2, 16, 64, 0)
    was = cache.k.clone()
    x = T.ones(4, 2 * 64, device="cuda")
    for bad in ([3, 0, 0, 1], [0, 15, 0, 2], [0, 0, 3, 2], [0, -1, 0, 1], [0, 0, -1, 1]):
        run_store(fb, T, cache, [bad], x, x, 0, 4)
        assert fb.lib().fence_device_error() == -1
    assert T.equal(was, cache.k)


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("type", [0, 1, 2])
def test_load_gives_code_times_scale(fb, T, ref, fmt, type):
    for hkv, hd, page in ((8, 128, 16), (3, 256, 128), (1, 64, 64)):
        cache = Cache(fb, T, 7, hkv, page, hd, fmt)
        slots = [0, 6 * page + page - 1, -1, 3 * page + 5, 3 * page + 5, page]
        dt = getattr(T, DT[type])
        buf = T.full((len(slots), 2 * hkv * hd + 5), 9.0, dtype=dt, device="cuda")
        k, v = buf[:, 1:1 + hkv * hd], T.empty(len(slots), hkv * hd, dtype=dt, device="cuda")
        s = i32(T, slots)
        fb.call("fence_kv8_load", cache.struct(), s.data_ptr(), len(slots), k.data_ptr(), v.data_ptr(), type, k.stride(0),
                v.stride(0), stream(T))
        for got, codes, scale in ((k, cache.k, cache.ks), (v, cache.v, cache.vs)):
            val = (ref.values(codes, fmt).float() * scale[..., None, None]).transpose(1, 2).reshape(-1, hkv * hd)
            want = T.where((s >= 0)[:, None], val[s.clamp(min=0).long()], 0.0).to(dt)
            assert T.equal(got, want)
        assert bool((buf[:, 0] == 9).all()) and bool((buf[:, 1 + hkv * hd:] == 9).all())
        # one of the two alone
        v2 = T.empty_like(v)
        fb.call("fence_kv8_load", cache.struct(), s.data_ptr(), len(slots), None, v2.data_ptr(), type, 0, v2.stride(0), stream(T))
        assert T.equal(v, v2)
        bad = i32(T, [7 * page])
        fb.call("fence_kv8_load", cache.struct(), bad.data_ptr(), 1, None, v2.data_ptr(), type, 0, v2.stride(0), stream(T))
        assert fb.lib().fence_device_error() == -1 and not v2[0].any()


# ------------------------------------------------------------------ attention
class Batch:
    """lens: (tokens in the cache with the new ones, new tokens) of every request."""

    def __init__(self, fb, T, lens, hq, hkv, hd, page, fmt, type, window=0, pad=0, seed=0, spare=2, max_new=None, scale=None,
                 q_pad=0, out_pad=0, q_scale=1.0):
        g = T.Generator(device="cuda").manual_seed(seed + 1)
        self.fb, self.T = fb, T
        self.lens, self.hq, self.window, self.type = lens, hq, window, type
        held = [-(-max(0, kv) // page) for kv, _ in lens]
        self.cache = Cache(fb, T, sum(held) + spare, hkv, page, hd, fmt, seed)
        ids = list(range(sum(held) + spare))
        random.Random(seed).shuffle(ids)
        self.max_pages = max(1, max(held) + 1)
        self.table, at = [], 0
        for h in held:
            self.table.append(ids[at:at + h] + [-9] * (self.max_pages - h))  # entries past the length are never used
            at += h
        self.unused = ids[at:]
        self.start = [0]
        for _, n in lens:
            self.start.append(self.start[-1] + n)
        self.n_tokens = self.start[-1] + pad
        dt = getattr(T, DT[type])
        self.qbuf = (T.randn(self.n_tokens, hq * hd + q_pad, generator=g, device="cuda") * q_scale).to(dt)
        self.q = self.qbuf[:, q_pad:]
        self.obuf = T.full((self.n_tokens, hq * hd + out_pad), 7.0, dtype=dt, device="cuda")
        self.out = self.obuf[:, :hq * hd]
        self.lse = T.full((self.n_tokens, hq), 7.0, device="cuda")
        self.scale = hd ** -0.5 if scale is None else scale
        self.max_new = max_new or max(1, max(n for _, n in lens))
        self.d_table, self.d_kv, self.d_start = i32(T, self.table), i32(T, [kv for kv, _ in lens]), i32(T, self.start)
        self.ws = None

    def structs(self):
        fb = self.fb
        b, a = fb.PagedBatch(), fb.KV8Attn()
        b.n_req, b.n_tokens, b.page_tokens, b.max_pages, b.n_pages = (len(self.lens), self.n_tokens, self.cache.page, self.max_pages,
                                                                      self.cache.n_pages)
        b.block_table, b.kv_len, b.new_start = self.d_table.data_ptr(), self.d_kv.data_ptr(), self.d_start.data_ptr()
        a.q, a.out, a.lse = self.q.data_ptr(), self.out.data_ptr(), self.lse.data_ptr()
        a.q_stride, a.out_stride, a.type, a.n_q_heads = self.q.stride(0), self.out.stride(0), self.type, self.hq
        a.max_new, a.window, a.scale = self.max_new, self.window, self.scale
        c = self.cache.struct()
        need = fb.lib().fence_kv8_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), ctypes.byref(a))
        assert need > 0
        if self.ws is None or self.ws.numel() < need:
            self.ws = self.T.zeros(need, dtype=self.T.uint8, device="cuda")
        a.workspace, a.workspace_bytes = self.ws.data_ptr(), self.ws.numel()
        return c, b, a

    def run(self):
        self.fb.call("fence_kv8_attention", *self.structs(), stream(self.T))
        return self.out, self.lse

    def want(self, ref):
        c = self.cache
        return ref.attention(c.k, c.v, c.ks, c.vs, c.fmt, self.table, [kv for kv, _ in self.lens], self.start,
                             self.q.reshape(self.n_tokens, self.hq, c.hd), c.hkv, self.scale, self.window, c.page)

    def check(self, ref):
        T = self.T
        out, lse = self.run()
        T.cuda.synchronize()
        want, wlse = self.want(ref)
        used = [p for r, (kv, _) in enumerate(self.lens) for p in self.table[r][:-(-max(0, kv) // self.cache.page)]]
        V = max([(ref.values(self.cache.v[p], self.cache.fmt).abs().amax((1, 2)) * self.cache.vs[p].double()).max().item() for p in used[:400]]
                + [0.0]) if used else 0.0
        got = out.reshape(self.n_tokens, self.hq, -1).double()
        err = (got - want).abs()
        tol = 4e-5 * V if self.type == 0 else 2.0 ** -10 * V + (2.0 ** -10 if self.type == 1 else 2.0 ** -8) * want.abs()
        assert bool((err <= tol).all()), (err - tol).max().item()
        empty = wlse == -math.inf
        assert T.equal(lse == -math.inf, empty)
        e2 = (lse.double() - wlse).abs()[~empty]
        assert bool((e2 <= 4e-5 * wlse.abs()[~empty].clamp(min=1)).all()), e2.max().item()
        assert not got[empty].any()
        assert bool((self.obuf[:, self.hq * self.cache.hd:] == 7).all())


SHAPES = [(32, 8, 128, 16), (8, 8, 64, 64), (16, 2, 256, 128), (10, 2, 128, 32), (4, 4, 256, 16), (12, 1, 64, 32), (40, 8, 128, 64)]


@pytest.mark.parametrize("hq,hkv,hd,page", SHAPES)
@pytest.mark.parametrize("fmt,type", [(0, 0), (0, 1), (1, 2), (1, 0)])
def test_decode_lengths(fb, T, ref, hq, hkv, hd, page, fmt, type):
    """One token each over every kind of length: one, page and tile boundaries, long ones, a request not placed."""
    lens = [(1, 1), (2, 1), (page - 1, 1), (page, 1), (page + 1, 1), (0, 1), (63, 1), (64, 1), (65, 1), (127, 1), (128, 1), (129, 1),
            (1000, 1), (2049, 1), (5, 0), (7, 1)]
    Batch(fb, T, lens, hq, hkv, hd, page, fmt, type).check(ref)


@pytest.mark.parametrize("hq,hkv,hd,page", SHAPES)
@pytest.mark.parametrize("fmt,type", [(0, 0), (0, 2), (1, 1), (1, 0)])
def test_several_tokens_each(fb, T, ref, hq, hkv, hd, page, fmt, type):
    """Drafts and chunks of every size in one batch, with padding rows at the end."""
    lens = [(2, 2), (300, 3), (17, 17), (700, 5), (0, 4), (130, 130), (1, 1), (900, 70), (33, 1), (257, 129)]
    Batch(fb, T, lens, hq, hkv, hd, page, fmt, type, pad=3).check(ref)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 300, 5000])
@pytest.mark.parametrize("hq,hkv,hd,page,type", [(32, 8, 128, 32, 1), (4, 2, 64, 128, 0), (8, 2, 256, 16, 2)])
def test_window(fb, T, ref, window, hq, hkv, hd, page, type):
    lens = [(1, 1), (64, 1), (65, 1), (700, 1), (1500, 40), (200, 200), (0, 2), (400, 4)]
    Batch(fb, T, lens, hq, hkv, hd, page, 0, type, window=window).check(ref)


@pytest.mark.parametrize("n,kv,page,hq,hkv,type", [(1, 70000, 64, 32, 8, 0), (1, 30011, 16, 8, 1, 2), (4, 20000, 128, 40, 8, 1),
                                                   (600, 9000, 64, 32, 8, 1), (2000, 2000, 32, 16, 4, 2), (300, 4000, 16, 32, 8, 0)])
def test_long(fb, T, ref, n, kv, page, hq, hkv, type):
    """One request whose keys are split over many blocks of threads and joined."""
    for fmt in (0, 1):
        Batch(fb, T, [(kv, n)], hq, hkv, 128, page, fmt, type).check(ref)


def test_many_requests(fb, T, ref):
    rng = random.Random(3)
    lens = [(rng.choice([0, 1, rng.randint(1, 200), rng.randint(1, 900)]), 1) for _ in range(300)]
    Batch(fb, T, lens, 8, 2, 128, 16, 0, 1).check(ref)
    lens = [(kv, 0 if kv == 0 else min(kv, rng.choice([0, 1, 2, 40]))) for kv, _ in lens]
    Batch(fb, T, lens, 8, 2, 64, 16, 1, 2).check(ref)


def test_more_rows_than_positions(fb, T, ref):
    """A caller's own lengths: more rows than tokens in the cache, so the first rows see nothing."""
    Batch(fb, T, [(3, 10), (0, 5), (1, 1), (50, 80)], 8, 2, 128, 16, 0, 0).check(ref)


@pytest.mark.parametrize("type", [0, 1, 2])
def test_strides_alignment_and_padding(fb, T, ref, type):
    """q inside a wider buffer at an odd element offset, out with a row pitch that is no multiple of 16 bytes."""
    for q_pad, out_pad in ((8, 0), (3, 5), (1, 8)):
        Batch(fb, T, [(100, 1), (300, 7), (90, 40)], 8, 2, 128, 32, 1, type, pad=2, q_pad=q_pad, out_pad=out_pad).check(ref)


@pytest.mark.parametrize("n", [1, 3, 100])
@pytest.mark.parametrize("fmt", [0, 1])
def test_rows_and_pages_out_of_sight_do_not_matter(fb, T, ref, n, fmt):
    """Unused pages and the rows after a request's last token hold anything: NaN codes, NaN scales."""
    b = Batch(fb, T, [(77, n), (130, 1), (200, n)], 8, 2, 128, 64, fmt, 0)
    want = [x.clone() for x in b.run()]
    for r, (kv, _) in enumerate(b.lens):
        p = b.table[r][kv // 64]
        for codes in (b.cache.k, b.cache.v):
            codes[p, :, kv % 64:] = 0x7f if fmt == 1 else 0x80
    for p in b.unused:
        b.cache.k[p], b.cache.v[p] = 0xff, 0xff
        b.cache.ks[p], b.cache.vs[p] = math.nan, math.nan
    got = b.run()
    assert T.equal(got[0], want[0]) and T.equal(got[1], want[1])
    # with a window, the pages before it are out of sight too
    b = Batch(fb, T, [(600, n)], 8, 2, 128, 64, fmt, 0, window=100)
    want = [x.clone() for x in b.run()]
    for p in b.table[0][:(600 - n - 100) // 64]:
        b.cache.k[p], b.cache.v[p], b.cache.ks[p], b.cache.vs[p] = 0x7f, 0x7f, math.nan, math.inf
    got = b.run()
    assert T.equal(got[0], want[0]) and T.equal(got[1], want[1])


@pytest.mark.parametrize("n", [1, 60])
def test_zero_pages_and_uneven_scales(fb, T, ref, n):
    """Pages of zeros (scale 0), and V scales that differ a thousandfold between the pages of one request."""
    for type in (0, 1):
        b = Batch(fb, T, [(1000, n), (64, min(n, 64)), (300, n)], 8, 2, 128, 32, 0, type)
        b.cache.v[b.table[0][3]], b.cache.vs[b.table[0][3]] = 0, 0
        b.cache.k[b.table[0][5]], b.cache.ks[b.table[0][5]] = 0, 0
        for p in b.table[1][:2]:
            b.cache.v[p], b.cache.vs[p] = 0, 0
        for j, p in enumerate(b.table[2][:10]):
            b.cache.vs[p] *= 10.0 ** -(j % 4)
        b.check(ref)
        for j, p in enumerate(b.table[0][:30]):
            b.cache.vs[p] *= 10.0 ** (j % 7 - 9)  # the scales grow along the request, all of them tiny
        b.check(ref)


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("scale", [0.0, 1e-3, 3.0])
def test_flat_and_sharp_softmax(fb, T, ref, n, scale):
    """Scores of 0 throughout, and scores of a size where one key takes all (their rounding then counts: scores of up
    to 400 * 22 bits)."""
    b = Batch(fb, T, [(500, n), (40, n)], 8, 2, 64, 16, 0, 1, scale=scale, q_scale=0.2)
    b.check(ref)


@pytest.mark.parametrize("n", [1, 40])
def test_large_and_small_queries(fb, T, ref, n):
    """Queries past fp16's range and far below it (fp32, bf16), with a scale that brings the scores back."""
    for type in (0, 2):
        for f in (2.0 ** 20, 2.0 ** -30):
            Batch(fb, T, [(300, n), (1, 1)], 8, 2, 128, 16, 0, type, scale=128 ** -0.5 / f, q_scale=f).check(ref)


@pytest.mark.parametrize("n", [1, 40])
def test_non_finite_stays_where_it_is(fb, T, ref, n):
    """A NaN or infinite scale of one page and head, and a NaN query row, reach their own rows alone."""
    b = Batch(fb, T, [(300, n), (300, n)], 8, 2, 128, 32, 0, 1)
    want = [x.clone().reshape(2, n, 8, -1) for x in b.run()]
    for where, bad in ((b.cache.ks, math.nan), (b.cache.vs, math.nan), (b.cache.ks, math.inf), (b.cache.vs, math.inf)):
        keep = where[b.table[0][2], 1].clone()
        codes = b.cache.k if where is b.cache.ks else b.cache.v
        kept = codes[b.table[0][2], 1].clone()
        codes[b.table[0][2], 1] = 0  # as the store leaves such a page
        where[b.table[0][2], 1] = bad
        out, lse = (x.clone().reshape(2, n, 8, -1) for x in b.run())
        assert T.equal(out[1], want[0][1]) and T.equal(out[0, :, :4], want[0][0, :, :4])
        assert T.equal(lse[1], want[1][1]) and T.equal(lse[0, :, :4], want[1][0, :, :4])
        assert bool(T.isnan(out[0, :, 4:]).all())
        where[b.table[0][2], 1] = keep
        codes[b.table[0][2], 1] = kept
    b.q[n:n + 1, 128:256] = math.nan  # the second request's first row, head 1
    out, _ = b.run()
    out = out.reshape(2, n, 8, -1)
    assert bool(T.isnan(out[1, 0, 1]).all())
    out[1, 0, 1] = want[0][1, 0, 1]
    assert T.equal(out, want[0])


def test_same_bits_every_time_and_any_workspace(fb, T):
    """Twice the same, after other work in the same workspace too, and with every hint of max_new within rounding."""
    b = Batch(fb, T, [(5000, 1), (70, 1), (900, 33)], 32, 8, 128, 64, 0, 1)
    first = [x.clone() for x in b.run()]
    other = Batch(fb, T, [(3000, 2)] * 5, 32, 8, 128, 64, 0, 1, seed=4)
    other.ws = b.ws
    for _ in range(3):
        other.run()
        out, lse = b.run()
        assert T.equal(out, first[0]) and T.equal(lse, first[1])
    for hint in (1, 2, 8, 33, 4000):
        b.max_new = hint
        out, lse = b.run()
        assert (out.float() - first[0].float()).abs().max().item() <= 2.0 ** -9 * first[0].float().abs().max().item() + 2.0 ** -9


def test_other_streams_and_graphs(fb, T, ref):
    """On a stream of its own, and captured in a graph whose lengths change between replays."""
    b = Batch(fb, T, [(400, 1), (50, 1), (900, 1)], 8, 2, 128, 32, 0, 0)
    want = [x.clone() for x in b.run()]
    T.cuda.synchronize()
    s = T.cuda.Stream()
    with T.cuda.stream(s):
        b.out.zero_()
        b.run()
    s.synchronize()
    assert T.equal(b.out, want[0])
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g):
        b.run()
    b.lens = [(33, 1), (50, 1), (0, 1)]
    b.d_kv.copy_(i32(T, [33, 50, 0]))
    g.replay()
    T.cuda.synchronize()
    w, _ = b.want(ref)
    V = (ref.values(b.cache.v, 0).abs().amax((1, 2, 3)) * b.cache.vs.double().amax(1)).max().item()
    assert (b.out.double().reshape(w.shape) - w).abs().max().item() <= 4e-5 * V


def test_bad_lengths_and_pages_are_reported_not_followed(fb, T):
    b = Batch(fb, T, [(100, 1), (60, 1), (200, 50)], 8, 2, 128, 32, 0, 0)
    for bad in ([100000, 60, 200], [-5, 60, 200]):
        b.d_kv.copy_(i32(T, bad))
        b.run()
        assert fb.lib().fence_device_error() == -1, bad
    b.d_kv.copy_(i32(T, [100, 60, 200]))
    for bad in (b.cache.n_pages, -1, 1 << 30):
        keep = b.d_table.clone()
        b.d_table[0, 0] = bad
        b.d_table[2, 1] = bad
        b.run()
        assert fb.lib().fence_device_error() == -1
        b.d_table.copy_(keep)
    b.d_start.copy_(i32(T, [0, 1, 2, 5000]))
    b.run()
    assert fb.lib().fence_device_error() == -1


@pytest.mark.parametrize("n", [1, 50])
def test_offsets_past_32_bits(fb, T, ref, n):
    """Pages at the end of a pool of more than 2^32 bytes of codes."""
    page, hkv, hd = 128, 8, 128
    n_pages = (1 << 32) // (page * hkv * hd) + 40
    b = Batch(fb, T, [(500, n)], 8, hkv, hd, page, 0, 1)
    small = b.cache
    big = Cache.__new__(Cache)
    big.__dict__.update(small.__dict__)
    big.n_pages = n_pages
    shift = n_pages - small.n_pages
    big.k = T.zeros(n_pages, hkv, page, hd, dtype=T.uint8, device="cuda")
    big.v = T.zeros_like(big.k)
    big.ks, big.vs = T.zeros(n_pages, hkv, device="cuda"), T.zeros(n_pages, hkv, device="cuda")
    for x in ("k", "v", "ks", "vs"):
        getattr(big, x)[shift:] = getattr(small, x)
    want = [x.clone() for x in b.run()]
    b.cache = big
    b.d_table.copy_(i32(T, [[p + shift if p >= 0 else p for p in r] for r in b.table]))
    out, lse = b.run()
    assert T.equal(out, want[0]) and T.equal(lse, want[1])
    rows = T.randn(3, hkv * hd, device="cuda")
    run_store(fb, T, big, [[n_pages - 1, 0, 0, 3]], rows, rows, 0, 3)
    back = T.empty(3, hkv * hd, device="cuda")
    slots = i32(T, [(n_pages - 1) * page + i for i in range(3)])
    fb.call("fence_kv8_load", big.struct(), slots.data_ptr(), 3, back.data_ptr(), None, 0, back.stride(0), 0, stream(T))
    # half a step of each head's scale
    step = big.ks[n_pages - 1].repeat_interleave(hd)
    assert bool(((back - rows).abs() <= 0.5 * step * (1 + 1e-5)).all())
