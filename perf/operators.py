"""The batched-serving operators over a paged 8-bit KV cache: what is measured, and their plain forms.

  plan    block tables, slot maps and page lists of one step, from request lengths (fence_paged_plan)
  store   the step's K/V rows quantised into the pages, one scale per page and head, and the touched
          pages' rows read back as the values they stand for (fence_kv8_store, fence_kv8_load)
  attn    causal grouped-query attention of a ragged batch over the pages (fence_kv8_attention)

A cache is two buffers of one-byte codes [n_pages][n_kv_heads][page][head_dim] and two of float
scales [n_pages][n_kv_heads]; a value is code * scale.
"""
import ctypes
import importlib.util
import math
import os
import random
import sys

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
TYPE = {"f32": 0, "f16": 1, "bf16": 2}  # FENCE_F32, FENCE_F16, FENCE_BF16
FMT = {"int8": 0, "e4m3": 1}            # FENCE_KV8_INT8, FENCE_KV8_E4M3
LIMIT = {"int8": 127.0, "e4m3": 448.0}  # the largest code
TINY = 1.1754943508222875e-38           # scales below the smallest normal float count as zero


# ------------------------------------------------------------------ cases
def _plan(name, n_req, ctx_hi, new, n_chunk, chunk, ended, page, spare, mix):
    return dict(name=name, op="plan", n_req=n_req, ctx_lo=1, ctx_hi=ctx_hi, new=new, n_chunk=n_chunk, chunk=chunk,
                ended=ended, page=page, spare=spare, mix=mix)


def _store(name, n_req, ctx_hi, new, page, hkv, hd, fmt, dt, mix):
    return dict(name=name, op="store", n_req=n_req, ctx_lo=1, ctx_hi=ctx_hi, new=new, n_chunk=0, chunk=0, idle=0,
                page=page, hq=4 * hkv, hkv=hkv, hd=hd, fmt=fmt, dt=dt, mix=mix)


def _attn(name, n_req, ctx_lo, ctx_hi, new, n_chunk, chunk, idle, page, hq, hkv, hd, window, fmt, dt, mix):
    return dict(name=name, op="attn", n_req=n_req, ctx_lo=ctx_lo, ctx_hi=ctx_hi, new=new, n_chunk=n_chunk, chunk=chunk,
                idle=idle, page=page, hq=hq, hkv=hkv, hd=hd, window=window, fmt=fmt, dt=dt, mix=mix)


def listed():
    return [
        # a decode step of 48 running requests
        _plan("plan decode 48", 48, 4096, 1, 0, 0, 0, 16, 64, 1),
        # a large scheduler step: many requests decode, some ended, 24 prompts enter
        _plan("plan mixed 2000", 2000, 8000, 1, 24, 2048, 60, 32, 1600, 2),
        # the decode step's rows of 61 requests, straight from an fp32 qkv buffer
        _store("store decode 61", 61, 4000, 1, 16, 8, 128, "int8", "f32", 3),
        # two prompts' chunks of one step
        _store("store prompts", 2, 1000, 4000, 64, 8, 128, "e4m3", "bf16", 4),
        # one user, a short chat: latency
        _attn("decode 1 short", 1, 700, 700, 1, 0, 0, 0, 16, 32, 8, 128, 0, "int8", "f32", 5),
        # a batch of chats of every length, one of them not placed this step
        _attn("decode 64", 64, 60, 8000, 1, 0, 0, 1, 32, 32, 8, 128, 0, "int8", "bf16", 6),
        # a few users with whole books in their contexts
        _attn("decode 3 long", 3, 90000, 131000, 1, 0, 0, 0, 64, 40, 8, 128, 0, "e4m3", "f16", 7),
        # drafts of 4 tokens checked at once, small heads, one KV head per query head
        _attn("drafts 17 of 4", 17, 200, 6000, 4, 0, 0, 0, 16, 8, 8, 64, 0, "e4m3", "bf16", 8),
        # a 4000-token prompt from nothing
        _attn("prompt 4000", 1, 0, 0, 4000, 0, 0, 0, 64, 32, 8, 128, 0, "int8", "f16", 9),
        # a later chunk of a long document
        _attn("chunk 2048 at 30000", 1, 30000, 30000, 2048, 0, 0, 0, 64, 32, 8, 128, 0, "e4m3", "bf16", 10),
        # decode and prompts' chunks in one step, fp32 activations
        _attn("mixed 14 + 2 chunks", 16, 100, 4000, 1, 2, 300, 1, 32, 40, 8, 128, 0, "int8", "f32", 11),
        # wide heads, sliding window
        _attn("window, wide heads", 5, 500, 9000, 1, 1, 700, 0, 128, 16, 2, 256, 1024, "int8", "bf16", 12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    mix = rng.randrange(100, 1 << 30)
    page = rng.choice([16, 32, 64, 128])
    kind = rng.choice(["plan", "store", "store", "decode", "decode", "drafts", "prompt", "prompt", "mixed"])
    if kind == "plan":
        n = _log(rng, 1, 2000)
        chunks = rng.randint(0, min(n, 24))
        c = _plan("", n, _log(rng, 8, 8000), rng.randint(0, 3), chunks, _log(rng, 2, 2048), rng.randint(0, (n - chunks) // 8), page,
                  _log(rng, 1, 1600), mix)
    else:
        hd = rng.choice([64, 128, 128, 128, 256])
        hkv = rng.choice([1, 2, 5, 8, 8])
        hq = hkv * rng.choice([1, 2, 4, 4, 5, 8])
        fmt, dt = rng.choice(["int8", "e4m3"]), rng.choice(["f32", "f16", "bf16"])
        window = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
        if kind == "store":
            n = _log(rng, 1, 128)
            c = _store("", n, _log(rng, 4, 4000), max(1, _log(rng, 1, 8000) // n), page, hkv, hd, fmt, dt, mix)
        elif kind == "decode":
            n = _log(rng, 1, 96)
            hi = _log(rng, 2, max(64, min(131000, 400000 // n)))
            c = _attn("", n, rng.randint(1, hi), hi, 1, 0, 0, rng.randint(0, n // 8), page, hq, hkv, hd, window, fmt, dt, mix)
        elif kind == "drafts":
            n = _log(rng, 1, 32)
            hi = _log(rng, 8, max(64, 100000 // n))
            c = _attn("", n, rng.randint(1, hi), hi, rng.randint(2, 12), 0, 0, rng.randint(0, n // 8), page, hq, hkv, hd, window,
                      fmt, dt, mix)
        elif kind == "prompt":
            n = rng.randint(1, 3)
            new = _log(rng, 17, 4000 // n)
            hi = _log(rng, 1, max(2, min(30000, 60000000 // (new * n))))
            c = _attn("", n, 0 if hi < 4 else rng.randint(1, hi), hi, new, 0, 0, 0, page, hq, hkv, hd, window, fmt, dt, mix)
        else:
            n = rng.randint(3, 24)
            c = _attn("", n, 1, _log(rng, 64, 4000), 1, rng.randint(1, 2), _log(rng, 17, 700), rng.randint(0, 1), page, hq, hkv, hd,
                      window, fmt, dt, mix)
    del c["name"]
    return c


def _lens(case):
    """(tokens in the cache, new tokens) of every request; new < 0: the request has ended."""
    rng = random.Random(case["mix"])
    got = []
    for r in range(case["n_req"]):
        lo, hi = case["ctx_lo"], max(case["ctx_lo"], case["ctx_hi"])
        ctx = min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1))))))
        new = rng.randint(max(1, case["chunk"] * 3 // 4), case["chunk"]) if r < case["n_chunk"] else case["new"]
        got.append((ctx, new))
    for r in range(case.get("ended", 0)):
        at = case["n_req"] - 1 - 3 * r % max(1, case["n_req"])
        if at >= case["n_chunk"]:
            got[at] = (got[at][0], -1)
    rng.shuffle(got)
    return got


def _idle(case):
    """Requests that were not placed: they bring tokens and see nothing."""
    return {(7 * k + 1) % case["n_req"] for k in range(case.get("idle", 0))}


def _ceil(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ inputs
def _pages(lens, page, spare, gen):
    """A pool of shuffled pages: the block table [n_req][max_pages] of `lens` tokens each, and the pages left over."""
    held = [_ceil(n, page) for n in lens]
    pool = torch.randperm(sum(held) + spare, generator=gen, device="cuda").to(torch.int32)
    most = max(held)
    h = torch.tensor(held, device="cuda")
    at = torch.cumsum(h, 0) - h
    j = torch.arange(max(1, most), device="cuda")
    table = torch.where(j < h[:, None], pool[(at[:, None] + j).clamp(max=pool.numel() - 1)], 0).to(torch.int32)
    return table.contiguous(), pool[sum(held):].contiguous(), pool.numel()


def _codes(n_pages, hkv, page, hd, fmt, gen):
    """Codes of K or V pages: a few channels stand out in every head, as in real keys."""
    wide = 1 + 3 * (torch.rand(hkv, 1, hd, generator=gen, device="cuda") < 0.04).float()
    out = torch.empty(n_pages, hkv, page, hd, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (hkv * page * hd))
    for p in range(0, n_pages, step):
        n = min(step, n_pages - p)
        x = torch.randn(n, hkv, page, hd, generator=gen, device="cuda") * wide
        if fmt == "int8":
            out[p:p + n] = (x * 25).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
        else:
            out[p:p + n] = (x * 90).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return out


def _scales(n_pages, hkv, fmt, gen):
    return torch.exp(0.3 * torch.randn(n_pages, hkv, generator=gen, device="cuda")) * (4.0 / LIMIT[fmt])


def _touch_cap(T, n_req, page):
    return min(T, 2 * n_req + T // page)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens, P = _lens(case), case["page"]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["op"] == "plan":
        ctx, new = [a for a, _ in lens], [b for _, b in lens]
        T = sum(max(0, b) for b in new) + 5  # the token buffers are a little longer than the step
        table, left, n_pages = _pages(ctx, P, case["spare"], gen)
        longest = max(_ceil(a + max(0, b), P) for a, b in lens) + 2
        table = torch.cat([table, torch.zeros(len(lens), longest - table.shape[1], dtype=torch.int32, device="cuda")], 1).contiguous()
        free = torch.cat([left, torch.zeros(n_pages - left.numel(), dtype=torch.int32, device="cuda")])
        cap = _touch_cap(T, len(lens), P)
        e = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        return dict(case=case, ctx_len=i32(ctx), new_len=i32(new), block_table=table, free_pages=free, n_free=i32([left.numel()]),
                    T=T, cap=cap, n_pages=n_pages, n_free_out=e(1), ctx_out=e(len(lens)), kv_len=e(len(lens)),
                    new_start=e(len(lens) + 1), slot=e(T), pos=e(T), touch=e(cap, 4))
    hq, hkv, hd, fmt, dt = case["hq"], case["hkv"], case["hd"], case["fmt"], DT[case["dt"]]
    idle = _idle(case)
    n = [b for _, b in lens]
    kv = [0 if r in idle else a + b for r, (a, b) in enumerate(lens)]
    T = sum(n)
    table, _, n_pages = _pages(kv, P, 3, gen)
    start = [0]
    for b in n:
        start.append(start[-1] + b)
    qkv = torch.randn(T, (hq + 2 * hkv) * hd, generator=gen, device="cuda").to(dt)
    s = dict(case=case, T=T, n_pages=n_pages, block_table=table, kv_len=i32(kv), new_start=i32(start), max_new=max(n),
             max_kv=max(kv), q=qkv[:, :hq * hd] * 2, k_new=qkv[:, hq * hd:(hq + hkv) * hd], v_new=qkv[:, (hq + hkv) * hd:],
             k=_codes(n_pages, hkv, P, hd, fmt, gen), v=_codes(n_pages, hkv, P, hd, fmt, gen),
             k_scale=_scales(n_pages, hkv, fmt, gen), v_scale=_scales(n_pages, hkv, fmt, gen))
    if case["op"] == "store":
        pages, first, rows, at = [], [], [], []
        for r, (a, b) in enumerate(lens):
            for j in range(a // P, (a + b - 1) // P + 1 if kv[r] else 0):
                lo, hi = max(a, j * P), min(a + b, (j + 1) * P)
                pages.append((r, j))
                first.append(lo - j * P)
                rows.append(hi - lo)
                at.append(start[r] + lo - a)
        rj = torch.tensor(pages, device="cuda")
        ids = table[rj[:, 0], rj[:, 1]]
        cap = _touch_cap(T, len(lens), P)
        touch = torch.zeros(cap, 4, dtype=torch.int32, device="cuda")
        touch[:, 0] = -1
        touch[:len(pages)] = torch.stack([ids, i32(first), i32(at), i32(rows)], 1)
        filled = i32(first) + i32(rows)
        grid = ids[:, None] * P + torch.arange(P, device="cuda", dtype=torch.int32)
        slots = grid[torch.arange(P, device="cuda") < filled[:, None]].contiguous()  # every filled row of the touched pages
        e = lambda: torch.empty(slots.numel(), hkv, hd, dtype=dt, device="cuda")  # noqa: E731
        s.update(touch=touch, cap=cap, n_touch=len(pages), slots=slots, k_back=e(), v_back=e())
    else:
        s.update(out=torch.empty(T, hq, hd, dtype=dt, device="cuda"), lse=torch.empty(T, hq, device="cuda"))
    return s


# ------------------------------------------------------------------ the framework's calls
_fb = None


def _framework():
    """The package's binding (its folder's name is no Python identifier)."""
    global _fb
    if _fb is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        pkg = os.path.join(root, "-damn-low-level-fence-inference-version-1_b200")
        spec = importlib.util.spec_from_file_location("fence_b200", os.path.join(pkg, "__init__.py"), submodule_search_locations=[pkg])
        _fb = importlib.util.module_from_spec(spec)
        sys.modules["fence_b200"] = _fb
        spec.loader.exec_module(_fb)
    return _fb


def _handles(s):
    """The structs that a program keeps beside its buffers."""
    fb, c = _framework(), s["case"]
    b = fb.PagedBatch()
    b.n_req, b.page_tokens, b.max_pages, b.n_pages, b.n_tokens = c["n_req"], c["page"], s["block_table"].shape[1], s["n_pages"], s["T"]
    b.n_touch = s.get("cap", 0)
    for name in ("ctx_len", "new_len", "block_table", "free_pages", "n_free", "n_free_out", "ctx_out", "kv_len", "new_start", "slot",
                 "pos", "touch"):
        if name in s:
            setattr(b, name, s[name].data_ptr())
    s["batch"] = b
    if c["op"] == "plan":
        return
    kv = fb.KV8Cache()
    kv.k, kv.v, kv.k_scale, kv.v_scale = (s[x].data_ptr() for x in ("k", "v", "k_scale", "v_scale"))
    kv.n_pages, kv.n_kv_heads, kv.page_tokens, kv.head_dim, kv.format = s["n_pages"], c["hkv"], c["page"], c["hd"], FMT[c["fmt"]]
    s["cache"] = kv
    if c["op"] == "store":
        return
    a = fb.KV8Attn()
    a.q, a.out, a.lse = s["q"].data_ptr(), s["out"].data_ptr(), s["lse"].data_ptr()
    a.q_stride, a.out_stride = s["q"].stride(0), s["out"].stride(0)
    a.type, a.n_q_heads, a.max_new, a.window, a.scale = TYPE[c["dt"]], c["hq"], s["max_new"], c["window"], c["hd"] ** -0.5
    need = fb.lib().fence_kv8_attention_workspace_bytes(ctypes.byref(kv), ctypes.byref(b), ctypes.byref(a))
    s["workspace"] = torch.zeros(need, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = s["workspace"].data_ptr(), need
    s["attn"] = a


def _run_own(s):
    fb, c = _framework(), s["case"]
    if "batch" not in s:
        _handles(s)
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "plan":
        fb.call("fence_paged_plan", s["batch"], stream)
        return {k: s[k] for k in PLANNED}
    if c["op"] == "store":
        k, v, kb, vb = s["k_new"], s["v_new"], s["k_back"], s["v_back"]
        fb.call("fence_kv8_store", s["cache"], s["batch"], k.data_ptr(), v.data_ptr(), TYPE[c["dt"]], k.stride(0), v.stride(0), stream)
        fb.call("fence_kv8_load", s["cache"], s["slots"].data_ptr(), s["slots"].numel(), kb.data_ptr(), vb.data_ptr(), TYPE[c["dt"]],
                kb.stride(0), vb.stride(0), stream)
        return {"k": kb, "v": vb, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    fb.call("fence_kv8_attention", s["cache"], s["batch"], s["attn"], stream)
    return {"out": s["out"], "lse": s["lse"]}


# ------------------------------------------------------------------ the plain forms
PLANNED = ("n_free_out", "ctx_out", "kv_len", "new_start", "slot", "pos", "touch", "block_table", "free_pages")


def _plan_plain(s):
    P, table, free, T, cap = s["case"]["page"], s["block_table"].long(), s["free_pages"].long(), s["T"], s["cap"]
    ctx, nl, n_free, n_pages = s["ctx_len"].long(), s["new_len"].long(), s["n_free"].long(), s["n_pages"]
    B, MP = table.shape
    ended, new, held = nl < 0, nl.clamp(min=0), (ctx + P - 1) // P
    fits = ctx + new <= MP * P
    need = torch.where(~ended & fits, (ctx + new + P - 1) // P - held, 0)
    back = torch.where(ended, held, 0)
    back_at = back.cumsum(0) - back
    avail = n_free + back.sum()
    N = need.cumsum(0)
    placed = ~ended & fits & ((need == 0) | (N <= avail))
    # the free stack with the ended requests' pages on top of it
    j = torch.arange(MP, device="cuda")
    idx = torch.where(j < back[:, None], n_free + back_at[:, None] + j, n_pages)
    stack = torch.cat([free, free[:1]]).scatter(0, idx.view(-1), table.view(-1))[:n_pages]
    fresh = placed[:, None] & (j >= held[:, None]) & (j < (held + need)[:, None])
    top = avail - 1 - ((N - need)[:, None] + j - held[:, None])
    table = torch.where(fresh, stack[top.clamp(0, n_pages - 1)], table)
    n_out = avail - torch.where(placed & (need > 0), N, 0).max()
    i = torch.arange(n_pages, device="cuda")
    free = torch.where((i >= n_free) & (i < n_out), stack, free)
    start = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), new.cumsum(0)])
    # tokens
    t = torch.arange(T, device="cuda")
    r = torch.searchsorted(start[1:], t, right=True).clamp(max=B - 1)
    real = (t < start[-1]) & placed[r]
    pos = torch.where(real, ctx[r] + t - start[r], -1)
    slot = torch.where(real, table[r, (pos // P).clamp(0, MP - 1)] * P + pos % P, -1)
    # pages that get tokens
    c = torch.where(placed & (new > 0), (ctx + new - 1) // P - ctx // P + 1, 0)
    C = c.cumsum(0)
    u = torch.arange(cap, device="cuda")
    q = torch.searchsorted(C, u, right=True)
    there, q = q < B, q.clamp(max=B - 1)
    at = ctx[q] // P + u - (C - c)[q]
    lo = torch.maximum(ctx[q], at * P)
    hi = torch.minimum((ctx + new)[q], (at + 1) * P)
    touch = torch.stack([table[q, at.clamp(0, MP - 1)], lo - at * P, start[q] + lo - ctx[q], hi - lo], 1)
    touch = torch.where(there[:, None], touch, torch.tensor([-1, 0, 0, 0], device="cuda"))
    got = dict(n_free_out=n_out, ctx_out=torch.where(ended, 0, torch.where(placed, ctx + new, ctx)), kv_len=torch.where(placed, ctx + new, 0),
               new_start=start, slot=slot, pos=pos, touch=touch, block_table=table, free_pages=free)
    return {k: v.to(torch.int32) for k, v in got.items()}


def _values(codes, fmt):
    return (codes.view(torch.int8) if fmt == "int8" else codes.view(torch.float8_e4m3fn)).float()


def _to_codes(x, fmt):
    if fmt == "int8":
        return x.round().nan_to_num(0.0).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return x.nan_to_num(0.0).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _store_plain(codes, scales, rows, touch, P, fmt):
    """One of K and V: the touched pages gathered, their new scales, their old rows brought to them, the new rows put in."""
    page, first, at, count = (touch[:, k].long() for k in range(4))
    hkv, hd = codes.shape[1], codes.shape[3]
    j = torch.arange(P, device="cuda")
    fresh = (j >= first[:, None]) & (j < (first + count)[:, None])
    old = j < first[:, None]
    t = (at[:, None] + j - first[:, None]).clamp(0, rows.shape[0] - 1)
    x = rows.view(rows.shape[0], hkv, hd)[t].float().permute(0, 2, 1, 3)                    # [pages][hkv][P][hd]
    x = torch.where(fresh[:, None, :, None], x, 0.0)
    s0 = torch.where(first[:, None] > 0, scales[page], 0.0)
    s1 = x.abs().amax((2, 3)) * torch.tensor(1.0 / LIMIT[fmt], device="cuda")
    s1 = torch.where(s1 < TINY, 0.0, s1)
    s1 = torch.where(s1 > s0, s1, s0)
    inv = torch.where(s1 > 0, 1.0 / s1, 0.0)[:, :, None, None]
    was = codes[page]
    moved = torch.where((s1 > s0)[:, :, None, None], _to_codes(_values(was, fmt) * s0[:, :, None, None] * inv, fmt), was)
    now = torch.where(fresh[:, None, :, None], _to_codes(x * inv, fmt), torch.where(old[:, None, :, None], moved, was))
    codes[page] = now
    scales[page] = s1


def _load_plain(codes, scales, slots, P, fmt, dt):
    page, row = slots.long() // P, slots.long() % P
    return (_values(codes[page, :, row], fmt) * scales[page][:, :, None]).to(dt)


def _attn_plain(s):
    c = s["case"]
    P, hq, hkv, hd, fmt = c["page"], c["hq"], c["hkv"], c["hd"], c["fmt"]
    B, G, N, C = c["n_req"], hq // hkv, s["max_new"], _ceil(max(1, s["max_kv"]), P)
    table = s["block_table"][:, :C].long()
    dense = lambda x, sc: (_values(x[table], fmt) * sc[table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(B, hkv, -1, hd)  # noqa: E731
    K, V = dense(s["k"], s["k_scale"]), dense(s["v"], s["v_scale"])
    start, kv = s["new_start"].long(), s["kv_len"].long()
    n = start[1:] - start[:-1]
    i = torch.arange(N, device="cuda")
    t = (start[:-1, None] + i).clamp(max=s["T"] - 1)
    q = s["q"].view(s["T"], hkv, G, hd)[t].float().permute(0, 2, 1, 3, 4).reshape(B, hkv, N * G, hd)
    x = torch.matmul(q, K.transpose(2, 3)).mul_(hd ** -0.5)
    pos = kv[:, None] - n[:, None] + i
    key = torch.arange(K.shape[2], device="cuda")
    seen = key <= pos[:, :, None]
    if c["window"] > 0:
        seen &= key > pos[:, :, None] - c["window"]
    x = x.view(B, hkv, N, G, -1).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = x.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hkv, N * G, -1), V).view(B, hkv, N, G, hd) / torch.where(l > 0, l, 1.0)
    lse = (m + l.log()).squeeze(-1)
    r = torch.searchsorted(start[1:], torch.arange(s["T"], device="cuda"), right=True)
    at = torch.arange(s["T"], device="cuda") - start[r]
    return {"out": o[r, :, at].reshape(s["T"], hq, hd).to(DT[c["dt"]]), "lse": lse[r, :, at].reshape(s["T"], hq)}


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["op"] == "plan":
        return _plan_plain(state)
    if c["op"] == "store":
        touch = state["touch"][:state["n_touch"]]
        _store_plain(state["k"], state["k_scale"], state["k_new"], touch, c["page"], c["fmt"])
        _store_plain(state["v"], state["v_scale"], state["v_new"], touch, c["page"], c["fmt"])
        return {"k": _load_plain(state["k"], state["k_scale"], state["slots"], c["page"], c["fmt"], DT[c["dt"]]),
                "v": _load_plain(state["v"], state["v_scale"], state["slots"], c["page"], c["fmt"], DT[c["dt"]]),
                "k_scale": state["k_scale"], "v_scale": state["v_scale"]}
    return _attn_plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    lens, P = _lens(case), case["page"]
    if case["op"] == "plan":
        T = sum(max(0, b) for _, b in lens) + 5
        fresh = sum(max(0, _ceil(a + b, P) - _ceil(a, P)) for a, b in lens if b >= 0)
        ended = sum(_ceil(a, P) for a, b in lens if b < 0)
        return {"bytes": 4.0 * (2 * len(lens) + 2 + 3 * len(lens) + 2 * T + 4 * _touch_cap(T, len(lens), P) + 2 * fresh + 2 * ended), "flops": 0}
    hkv, hd, es = case["hkv"], case["hd"], SIZE[case["dt"]]
    idle = _idle(case)
    live = [(a, b) for r, (a, b) in enumerate(lens) if r not in idle]
    if case["op"] == "store":
        new = sum(b for _, b in live)
        old = sum(a % P for a, _ in live)  # rows already in the touched pages: read back (and moved where the scale grows)
        return {"bytes": float(2 * hkv * hd * (new * (es + 1) + (new + old) * (1 + es))), "flops": float(4 * hkv * hd * new)}
    T, W = sum(b for _, b in lens), case["window"]
    keys = pairs = 0
    for a, b in live:
        keys += a + b if W <= 0 else min(a + b, W - 1 + b)
        pairs += sum(min(a + i + 1, W) if W > 0 else a + i + 1 for i in range(b))
    return {"bytes": float(2 * hkv * (keys * hd + 4 * _ceil(keys, P)) + 2 * T * case["hq"] * hd * es + 4 * T * case["hq"]),
            "flops": float(4 * hd * case["hq"] * pairs)}


# ------------------------------------------------------------------ the definition in 64 bits
def _round64(x, fmt):
    """x to the nearest code, ties to even, in 64 bits."""
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127)
    ulp = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / ulp) * ulp).clamp(-448, 448)


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s, P, fmt = prepare(case, seed), case["page"], case["fmt"]
    lens, hkv, hd = _lens(case), case["hkv"], case["hd"]
    start, table = s["new_start"].tolist(), s["block_table"].tolist()
    if case["op"] == "store":
        got = {}
        for what in "kv":
            codes, scales, rows = _values(s[what], fmt).double(), s[what + "_scale"].double(), s[what + "_new"].double()
            for r, (a, b) in enumerate(lens):
                for j in range(a // P, (a + b - 1) // P + 1):
                    lo, hi = max(a, j * P), min(a + b, (j + 1) * P)
                    x = rows[start[r] + lo - a:start[r] + hi - a].view(hi - lo, hkv, hd).transpose(0, 1)
                    page = table[r][j]
                    s0 = scales[page] if lo > j * P else torch.zeros_like(scales[page])
                    s1 = torch.maximum(s0, x.abs().amax((1, 2)) / LIMIT[fmt])
                    old = codes[page, :, :lo - j * P]
                    codes[page, :, :lo - j * P] = torch.where((s1 > s0)[:, None, None], _round64(old * (s0 / s1)[:, None, None], fmt), old)
                    codes[page, :, lo - j * P:hi - j * P] = _round64(x / s1[:, None, None], fmt)
                    scales[page] = s1
            slots = s["slots"].long()
            got[what] = codes[slots // P, :, slots % P] * scales[slots // P][:, :, None]
            got[what + "_scale"] = scales
        return got
    hq, W, T = case["hq"], case["window"], s["T"]
    out = torch.zeros(T, hq, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64, device="cuda")
    q = s["q"].double().view(T, hq, hd)
    for r, (a, b) in enumerate(lens):
        n = s["kv_len"][r].item()
        if n == 0:
            continue
        ids = torch.tensor(table[r][:_ceil(n, P)], device="cuda")
        for h in range(hq):
            g = h * hkv // hq
            K = (_values(s["k"][ids, g], fmt).double() * s["k_scale"][ids, g].double()[:, None, None]).view(-1, hd)[:n]
            V = (_values(s["v"][ids, g], fmt).double() * s["v_scale"][ids, g].double()[:, None, None]).view(-1, hd)[:n]
            for i0 in range(0, b, 1024):
                i1 = min(b, i0 + 1024)
                x = q[start[r] + i0:start[r] + i1, h] @ K.T / math.sqrt(hd)
                at = torch.arange(n - b + i0, n - b + i1, device="cuda")[:, None]
                key = torch.arange(n, device="cuda")
                x[(key > at) | ((key <= at - W) if W > 0 else (key < 0))] = -math.inf
                w = torch.logsumexp(x, 1)
                out[start[r] + i0:start[r] + i1, h] = torch.exp(x - w[:, None]) @ V
                lse[start[r] + i0:start[r] + i1, h] = w
    return {"out": out, "lse": lse}
