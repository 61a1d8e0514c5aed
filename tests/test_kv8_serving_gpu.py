"""The batched-serving operators together, as examples/paged_batch.py uses them: several requests that enter, decode and
end, against each of them alone through a dense float64 attention over the same (unquantised) keys and values.

The bound: int8 codes are off by at most half a step, 1 / 254 of their page's largest value, which is up to about 4
standard deviations, so 1.6 % of one at most and 0.9 % on average (uniform); q and the activations are fp16 (0.05 %).
The decoder's residual stream carries the embeddings unchanged, and two layers' attention averages its values, so logits
move by about 1 % of their spread: 5 % allowed on every logit's average over a row."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ex(fb):
    spec = importlib.util.spec_from_file_location("paged_batch", os.path.join(ROOT, "examples", "paged_batch.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def dense_logits(dec, ids):
    """Logits of every position of one request, float64."""
    import torch
    n, half = len(ids), dec.hd // 2
    x = dec.embed[torch.tensor(ids, device="cuda")].double()
    ang = torch.arange(n, device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(half, device="cuda").double() / half)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    rope = lambda y: torch.cat([y[..., :half] * c - y[..., half:] * s, y[..., :half] * s + y[..., half:] * c], -1)  # noqa: E731
    norm = lambda y: y * (y.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()  # noqa: E731
    hide = torch.ones(n, n, device="cuda").triu(1).bool()
    for wqkv, wo in zip(dec.wqkv, dec.wo):
        q, k, v = (norm(x) @ wqkv.double().T).split([dec.hq * dec.hd, dec.hkv * dec.hd, dec.hkv * dec.hd], 1)
        q, k, v = rope(q.view(n, dec.hq, -1)), rope(k.view(n, dec.hkv, -1)), v.view(n, dec.hkv, -1)
        k, v = (y.repeat_interleave(dec.hq // dec.hkv, 1) for y in (k, v))
        w = torch.softmax((torch.einsum("ihd,jhd->hij", q, k) * dec.hd ** -0.5).masked_fill(hide, float("-inf")), -1)
        x = x + torch.einsum("hij,jhd->ihd", w, v).reshape(n, -1) @ wo.double().T
    return norm(x) @ dec.embed.double().T


@pytest.mark.parametrize("fmt,page", [(0, 16), (1, 32)])
def test_requests_enter_decode_and_end(ex, fmt, page):
    import torch
    dec = ex.Decoder(fmt=fmt, page=page, n_pages=24 if page == 32 else 40, max_req=4, max_pages=8)
    seen = {}
    step = dec.step

    def spy(new_len, tokens, max_new):  # keeps every step's rows
        y = step(new_len, tokens, max_new)
        if y is not None:
            seen.setdefault("rows", []).append((list(new_len), list(tokens), y.double()))
        return y

    dec.step = spy
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (5, 33, 1, 70, 16, 48, 9)]
    out = ex.serve(dec, prompts, max_new=6)
    assert all(len(o) == 6 for o in out)
    assert dec.n_free[dec.turn].item() == dec.batch.n_pages  # all pages came back
    assert sorted(dec.free.tolist()) == list(range(dec.batch.n_pages))
    # the rows of each request, in order, against the request alone
    history = {}
    for new_len, tokens, y in seen["rows"]:
        at = 0
        for r, n in enumerate(new_len):
            if n < 0:
                history[r] = []
            for ids, logits in [(tokens[at:at + n], y[at:at + n])] if n > 0 else []:
                h = history.setdefault(r, [])
                h += ids
                want = dense_logits(dec, h)[-n:]
                off = (logits - want).norm(dim=1) / want.norm(dim=1)
                assert off.max().item() < 0.05, (r, len(h), off.max().item())
            at += max(0, n)
