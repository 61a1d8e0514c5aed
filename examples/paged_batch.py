"""Several requests served at once over a paged 8-bit KV cache: prompts of different lengths enter while others decode,
requests end and give their pages back; what does not fit comes again.

A small attention-only decoder with random weights stands in for a model: per layer the q|k|v projection
(fence_gemm_f16), rotary embedding, fence_kv8_store, fence_kv8_attention and the output projection. One
fence_paged_plan per step serves all layers; a step copies its greedy ids and kv_len to the host, once.

    python examples/paged_batch.py
"""
import ctypes
import importlib.util
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "-damn-low-level-fence-inference-version-1_b200")


def load_package():
    """The binding (its folder's name is no Python identifier)."""
    if "fence_b200" not in sys.modules:
        spec = importlib.util.spec_from_file_location("fence_b200", os.path.join(PKG, "__init__.py"), submodule_search_locations=[PKG])
        sys.modules["fence_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["fence_b200"])
    return sys.modules["fence_b200"]


fb = load_package()


class Decoder:
    """Random weights; layers of attention over a paged cache."""

    def __init__(self, layers=2, hq=8, hkv=2, hd=64, vocab=512, n_pages=64, page=16, max_req=8, max_pages=16, max_tokens=256, fmt=None, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.layers, self.hq, self.hkv, self.hd, self.page, self.dim, self.max_tokens = layers, hq, hkv, hd, page, hq * hd, max_tokens
        self.embed = rnd(vocab, self.dim).half()
        self.wqkv = [(rnd((hq + 2 * hkv) * hd, self.dim) * self.dim ** -0.5).half() for _ in range(layers)]
        self.wo = [(rnd(self.dim, self.dim) * self.dim ** -0.5).half() for _ in range(layers)]
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        cap = min(max_tokens, 2 * max_req + max_tokens // page)
        # the plan's buffers: lengths and the free count in two sets, the one that is read and the one that is written
        self.ctx, self.n_free = [i32(max_req), i32(max_req)], [i32(1), i32(1)]
        self.new_len, self.kv_len, self.new_start = i32(max_req), i32(max_req), i32(max_req + 1)
        self.table, self.slot, self.pos, self.touch = i32(max_req, max_pages), i32(max_tokens), i32(max_tokens), i32(cap, 4)
        self.free = torch.arange(n_pages, dtype=torch.int32, device="cuda")
        self.n_free[0].fill_(n_pages)
        self.turn = 0
        b = self.batch = fb.PagedBatch(n_req=max_req, page_tokens=page, max_pages=max_pages, n_pages=n_pages)
        for name, t in (("new_len", self.new_len), ("block_table", self.table), ("free_pages", self.free), ("kv_len", self.kv_len),
                        ("new_start", self.new_start), ("slot", self.slot), ("pos", self.pos), ("touch", self.touch)):
            setattr(b, name, t.data_ptr())
        # a cache per layer
        fmt = fb.FENCE_KV8_INT8 if fmt is None else fmt
        self.store, self.cache = [], []
        for _ in range(layers):
            bufs = [torch.zeros(n_pages, hkv, page, hd, dtype=torch.uint8, device="cuda") for _ in range(2)]
            bufs += [torch.zeros(n_pages, hkv, device="cuda") for _ in range(2)]
            self.store.append(bufs)
            self.cache.append(fb.KV8Cache(*[t.data_ptr() for t in bufs], n_pages, hkv, page, hd, fmt))
        self.attn = fb.KV8Attn(type=fb.FENCE_F16, n_q_heads=hq, scale=hd ** -0.5)
        b.n_tokens, self.attn.max_new = max_tokens, max_tokens
        need = fb.lib().fence_kv8_attention_workspace_bytes(ctypes.byref(self.cache[0]), ctypes.byref(b), ctypes.byref(self.attn))
        self.workspace = torch.zeros(need, dtype=torch.uint8, device="cuda")
        self.attn.workspace, self.attn.workspace_bytes = self.workspace.data_ptr(), need

    def rope(self, x, pos):
        """Rotary embedding of x [tokens][heads][hd] at the plan's positions."""
        half = self.hd // 2
        angle = pos.clamp(min=0)[:, None].float() * 10000.0 ** (-torch.arange(half, device="cuda") / half)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    def gemm(self, x, w):
        y = torch.empty(x.shape[0], w.shape[0], device="cuda")
        fb.call("fence_gemm_f16", x.data_ptr(), w.data_ptr(), y.data_ptr(), x.shape[0], w.shape[0], w.shape[1], self.stream)
        return y

    def step(self, new_len, tokens, max_new):
        """One step: new_len[r] tokens of request r (0: waits, -1: has ended), `tokens` one after another. Returns the
        logits of every token row."""
        T, b, a = len(tokens), self.batch, self.attn
        if T > self.max_tokens:
            raise ValueError("%d tokens in a step of at most %d" % (T, self.max_tokens))
        self.stream = torch.cuda.current_stream().cuda_stream
        self.new_len.copy_(torch.tensor(new_len, dtype=torch.int32))
        b.n_tokens = T
        b.n_touch = min(T, 2 * b.n_req + T // self.page)
        b.ctx_len, b.ctx_out = self.ctx[self.turn].data_ptr(), self.ctx[1 - self.turn].data_ptr()
        b.n_free, b.n_free_out = self.n_free[self.turn].data_ptr(), self.n_free[1 - self.turn].data_ptr()
        self.turn = 1 - self.turn
        fb.call("fence_paged_plan", b, self.stream)
        if T == 0:
            return None
        x = self.embed[torch.tensor(tokens, device="cuda")].float()
        pos, nq, nk = self.pos[:T], self.hq * self.hd, self.hkv * self.hd
        for layer in range(self.layers):
            h = (x * x.pow(2).mean(-1, keepdim=True).add(1e-6).rsqrt()).half()
            qkv = self.gemm(h, self.wqkv[layer])
            q = self.rope(qkv[:, :nq].view(T, self.hq, self.hd), pos).half().view(T, nq)
            k = self.rope(qkv[:, nq:nq + nk].reshape(T, self.hkv, self.hd), pos).view(T, nk)
            v = qkv[:, nq + nk:]
            fb.call("fence_kv8_store", self.cache[layer], b, k.data_ptr(), v.data_ptr(), fb.FENCE_F32, k.stride(0), v.stride(0), self.stream)
            out = torch.empty_like(q)
            a.q, a.out, a.q_stride, a.out_stride, a.max_new = q.data_ptr(), out.data_ptr(), nq, nq, max_new
            fb.call("fence_kv8_attention", self.cache[layer], b, a, self.stream)
            x = x + self.gemm(out, self.wo[layer])
        return self.gemm((x * x.pow(2).mean(-1, keepdim=True).add(1e-6).rsqrt()).half(), self.embed)


def serve(dec, prompts, max_new=12, arrive_every=2):
    """Greedy decoding of all prompts; a prompt enters a free row every few steps. Returns the generated ids per prompt.

    A step sends at most max_tokens rows, so a long prompt goes in chunks. A request that the plan could not place brings the
    same tokens again, and none enters meanwhile. Where nothing could be placed, the request that entered last gives its
    pages back and starts over later, with what it has generated as part of its prompt."""
    b = dec.batch
    longest = min(b.max_pages, b.n_pages) * b.page_tokens
    for p in prompts:
        if not p or len(p) + max_new - 1 > longest:
            raise ValueError("a prompt of %d tokens with %d new ones: at least 1 and at most %d fit" % (len(p), max_new, longest))
    rows = [None] * b.n_req  # the prompt index that a row serves
    out, waiting, step = [[] for _ in prompts], list(range(len(prompts))), 0
    due = [list(p) for p in prompts]  # what each request has still to bring
    entered, ended = [], []  # rows in the order in which they were taken; rows whose request has ended
    short = False  # not all could be placed
    while waiting or entered or ended:
        new_len, tokens, sent = [0] * len(rows), [], {}
        for r in ended:
            new_len[r] = -1
        if waiting and step % arrive_every == 0 and not short:
            free = [r for r, p in enumerate(rows) if p is None and r not in ended]
            if free:
                rows[free[0]] = waiting.pop(0)
                entered.append(free[0])
        for r, p in enumerate(rows):
            if p is None:
                continue
            ids = due[p][:dec.max_tokens - len(tokens)]
            new_len[r] = len(ids)
            if ids:
                tokens += ids
                sent[r] = len(tokens) - 1
        freed, ended = bool(ended), []
        logits = dec.step(new_len, tokens, max([1] + new_len))
        step += 1
        if not sent:
            short = False
            continue
        # the step's only copy to the host: the greedy ids, and which requests were placed
        got = torch.cat([logits[list(sent.values())].argmax(-1).int(), dec.kv_len[list(sent)]]).tolist()
        placed = 0
        for r, t, kv in zip(sent, got, got[len(sent):]):
            if kv == 0:
                continue
            placed += 1
            p = rows[r]
            due[p] = due[p][new_len[r]:]
            if due[p]:
                continue  # more of its prompt to come
            out[p].append(t)
            due[p] = [t]
            if len(out[p]) == max_new:
                rows[r] = None
                entered.remove(r)
                ended.append(r)
        short = placed < len(sent)
        if not placed and not freed:
            r = entered.pop()
            waiting.insert(0, rows[r])
            due[rows[r]] = prompts[rows[r]] + out[rows[r]]
            rows[r] = None
            ended.append(r)
    return out


def main():
    g = torch.Generator().manual_seed(1)
    dec = Decoder()
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (3, 40, 17, 64, 1, 25)]
    for p, ids in zip(prompts, serve(dec, prompts)):
        print("prompt of %2d tokens ->" % len(p), ids)
    torch.cuda.synchronize()
    print("pages free at the end: %d of %d" % (dec.n_free[dec.turn].item(), dec.batch.n_pages))


if __name__ == "__main__":
    main()
