"""The server loop of examples/paged_batch.py on the CPU, over a decoder whose plan is the plain one (tests/kv8_ref.py) and whose
next token is a function of all tokens that the cache holds: a token that was lost or stored twice changes what follows."""
import importlib.util
import os

import pytest
import torch

import kv8_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
VOCAB = 101


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("paged_batch_cpu", os.path.join(ROOT, "examples", "paged_batch.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def follows(history):
    return sum((i % 7 + 1) * t for i, t in enumerate(history)) % VOCAB


class Fake:
    """What serve() uses of a Decoder."""

    def __init__(self, fb, n_pages, max_pages, max_req, max_tokens, page=16):
        self.batch = fb.PagedBatch(n_req=max_req, page_tokens=page, max_pages=max_pages, n_pages=n_pages)
        self.max_tokens, self.page = max_tokens, page
        self.ctx, self.table, self.free = [0] * max_req, [[-1] * max_pages for _ in range(max_req)], list(range(n_pages))
        self.held = [[] for _ in range(max_req)]  # the tokens in each row's pages
        self.waits = self.chunks = 0

    def step(self, new_len, tokens, max_new):
        b = self.batch
        assert len(tokens) == sum(max(0, n) for n in new_len) <= self.max_tokens
        p = kv8_ref.plan(self.ctx, new_len, self.table, self.free, len(tokens), self.page, b.max_pages, b.n_pages)
        self.ctx, self.table, self.free = p["ctx_out"], p["block_table"], p["stack"]
        self.kv_len = torch.tensor(p["kv_len"], dtype=torch.int32)
        logits = torch.zeros(len(tokens), VOCAB)
        for r, n in enumerate(new_len):
            at = p["new_start"][r]
            if n < 0:
                self.held[r] = []
            elif n > 0 and p["kv_len"][r] == 0:
                self.waits += 1  # its rows attend to nothing: id 0
            elif n > 0:
                self.chunks += n > 1 and bool(self.held[r])
                for i in range(n):
                    self.held[r].append(tokens[at + i])
                    logits[at + i, follows(self.held[r])] = 1
        return logits if tokens else None


@pytest.mark.parametrize("n_pages,max_req,max_tokens,arrive", [(40, 4, 256, 2), (9, 4, 256, 1), (6, 4, 256, 2), (6, 7, 256, 1), (5, 3, 40, 1),
                                                               (7, 7, 10, 3), (12, 2, 9, 1)])
def test_every_request_gets_its_own_continuation(ex, fb, n_pages, max_req, max_tokens, arrive):
    g = torch.Generator().manual_seed(n_pages)
    prompts = [torch.randint(1, VOCAB, (n,), generator=g).tolist() for n in (5, 33, 1, 62, 16, 48, 9, 60)]
    dec = Fake(fb, n_pages, 6, max_req, max_tokens)
    out = ex.serve(dec, prompts, max_new=18, arrive_every=arrive)
    for p, ids in zip(prompts, out):
        h, want = list(p), []
        for _ in range(18):
            want.append(follows(h))
            h.append(want[-1])
        assert ids == want
    assert sorted(dec.free) == list(range(n_pages))
    assert dec.waits > 0 if n_pages < 10 else dec.waits == 0
    assert dec.chunks > 0 if max_tokens < 60 else True


def test_prompts_that_can_never_fit_are_refused(ex, fb):
    for n_pages, max_pages in ((3, 8), (8, 3)):
        with pytest.raises(ValueError):
            ex.serve(Fake(fb, n_pages, max_pages, 2, 64), [[1] * 40], max_new=10)
        assert len(ex.serve(Fake(fb, n_pages, max_pages, 2, 64), [[1] * 39], max_new=10)[0]) == 10
    with pytest.raises(ValueError):
        ex.serve(Fake(fb, 8, 8, 2, 64), [[]], max_new=10)


@pytest.mark.gpu
@pytest.mark.parametrize("n_pages,max_tokens", [(8, 256), (6, 24)])
def test_a_pool_too_small_for_all_requests_on_the_gpu(ex, n_pages, max_tokens):
    """The real decoder: every placed row's logits against the request alone, within the bound of test_kv8_serving_gpu.py."""
    from test_kv8_serving_gpu import dense_logits
    dec = ex.Decoder(n_pages=n_pages, max_req=4, max_pages=8, max_tokens=max_tokens)
    rows, step = [], dec.step

    def spy(new_len, tokens, max_new):
        y = step(new_len, tokens, max_new)
        rows.append((list(new_len), list(tokens), None if y is None else y.double(), dec.kv_len.clone()))
        return y

    dec.step = spy
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (5, 33, 1, 70, 16, 48, 9)]
    out = ex.serve(dec, prompts, max_new=12, arrive_every=1)
    assert all(len(o) == 12 for o in out)
    assert sorted(dec.free.tolist()) == list(range(n_pages))
    history, waits = {}, 0
    for new_len, tokens, y, kv in rows:
        at = 0
        for r, n in enumerate(new_len):
            if n < 0:
                history[r] = []
            elif n > 0 and kv[r] == 0:
                waits += 1
            elif n > 0:
                h = history.setdefault(r, [])
                h += tokens[at:at + n]
                assert kv[r] == len(h)
                want = dense_logits(dec, h)[-n:]
                off = (y[at:at + n] - want).norm(dim=1) / want.norm(dim=1)
                assert off.max().item() < 0.05
            at += max(0, n)
    assert waits > 0
