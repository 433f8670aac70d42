"""Paged cache, attention and token scores as a served model calls them, between the framework's
norms, FP8 products, rotary embedding and gated activation: a prompt's prefix, two questions on its pages,
then tokens chosen on the GPU in a replayed graph. Every call's outputs against the 64-bit
oracle on the inputs that the call really had."""
import pytest
import torch

from oracle import serving as S
from test_gpu_cache import close
from test_gpu_scores import _check

BF16, E4M3, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32
DEV = "cuda"
HIDDEN, HEADS, KV, D, WIDE, VOCAB, PAGE = 512, 8, 2, 128, 512, 1008, 16


def _product(g, n, k):
    from fastforward_amd.linear import FP8Linear
    return FP8Linear((torch.randn(n, k, generator=g) * k ** -0.5).to(DEV, BF16))


class Layer:
    def __init__(self, g, pages, dtype):
        from fastforward_amd import ops
        from fastforward_amd.cache import PagedCache

        def norm(d):
            return ops.RMSNorm((1 + 0.1 * torch.randn(d, generator=g)).to(DEV, BF16))
        self.qkv, self.out = _product(g, (HEADS + 2 * KV) * D, HIDDEN), _product(g, HIDDEN, HEADS * D)
        self.up, self.down = _product(g, 2 * WIDE, HIDDEN), _product(g, HIDDEN, WIDE)
        self.norm_in, self.norm_mid, self.norm_q, self.norm_k = norm(HIDDEN), norm(HIDDEN), norm(D), norm(D)
        self.cache = PagedCache(pages, PAGE, KV, D, dtype)

    def __call__(self, x, cos, sin, *rows):
        """x (T, HIDDEN); the sum after the layer, and what the attention read and wrote."""
        from fastforward_amd import ops
        t = x.shape[0]
        qkv = self.qkv(ops.fast_norm(x, self.norm_in))
        q, k, v = qkv.view(1, t, -1, D).split([HEADS, KV, KV], 2)
        q, k = (y[0].transpose(0, 1) for y in ops.qk_pair(q, k, self.norm_q, self.norm_k, cos, sin))
        self.cache.write(k, v[0], *rows)
        y = self.cache.attend(q, *rows)
        x = x + self.out(y.reshape(t, -1))
        gate, up = self.up(ops.fast_norm(x, self.norm_mid)).chunk(2, 1)
        return x + self.down(ops.swiglu(gate, up)), (q, k, v[0], y)


class Model:
    def __init__(self, dtype, pages):
        from fastforward_amd import ops
        g = torch.Generator().manual_seed(5)
        self.layers = [Layer(g, pages, dtype) for _ in range(2)]
        self.embed = torch.randn(VOCAB, HIDDEN, generator=g).to(DEV, BF16)
        self.head = _product(g, VOCAB, HIDDEN)
        self.norm = ops.RMSNorm(torch.ones(HIDDEN, device=DEV, dtype=BF16))
        self.freq = 1e4 ** (-torch.arange(0, D, 2, device=DEV).float() / D)
        self.held = []
        for layer in self.layers:
            c = {"k": layer.cache.k.cpu(), "v": layer.cache.v.cpu()}
            if dtype == E4M3:
                c.update(k_scale=layer.cache.k_scale.cpu(), v_scale=layer.cache.v_scale.cpu())
            self.held.append(c)

    def __call__(self, tokens, positions, *rows):
        """Logits (T, VOCAB) and every layer's (q, k, v, attended)."""
        from fastforward_amd import ops
        angle = (positions[:, None] * self.freq).repeat(1, 2)
        cos, sin = angle.cos().to(BF16), angle.sin().to(BF16)
        x, seen = self.embed[tokens.long()], []
        for layer in self.layers:
            x, of = layer(x, cos, sin, *rows)
            seen.append(of)
        return self.head(ops.fast_norm(x, self.norm)), seen

    def check(self, seen, table, lengths, starts):
        """The oracle's caches take the same rows; its attention is near, its pages are equal."""
        table, lengths = table.cpu(), lengths.cpu()
        starts = None if starts is None else starts.cpu()
        for layer, held, (q, k, v, y) in zip(self.layers, self.held, seen):
            S.write(held, k.cpu(), v.cpu(), table, lengths, starts)
            for name, want in held.items():
                assert torch.equal(getattr(layer.cache, name).cpu().view(torch.uint8), want.view(torch.uint8)), name
            close(y, *S.attend(held, q.cpu(), table, lengths, starts), D)


def _ints(*x):
    return torch.tensor(x, dtype=I32, device=DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_kept_prompt(gpu, dtype):
    from fastforward_amd.scores import token_scores
    model = Model(dtype, 12)
    prefix, questions = 70, (9, 4)
    # four full pages are the prefix's and shared; the fifth holds 6 tokens, and the second question has a copy
    table = _ints([7, 2, 11, 4, 0, 9, -1], [7, 2, 11, 4, 10, 1, -1])
    g = torch.Generator().manual_seed(6)
    prompt = torch.randint(0, VOCAB, (prefix,), generator=g).to(DEV)
    rows = (table[:1], _ints(prefix), _ints(0, prefix))
    logits, seen = model(prompt, torch.arange(prefix, device=DEV), *rows)
    model.check(seen, *rows)
    scored = token_scores(logits[:-1], prompt[1:], top=4)              # how likely the prompt itself is
    _check(logits[:-1].cpu(), prompt[1:].cpu(), 4)
    assert torch.equal(scored.logprobs, token_scores(logits, torch.cat([prompt[1:], prompt[:1]])).logprobs[:-1])
    for layer, held in zip(model.layers, model.held):
        for name in held:
            for pages in (getattr(layer.cache, name), held[name]):
                pages.view(torch.uint8)[10] = pages.view(torch.uint8)[0]

    # both questions at once, ragged, padded to 16 rows
    n = torch.tensor(questions)
    rows = (table, (n + prefix).to(DEV, I32), _ints(0, 9, 13))
    positions = torch.cat([prefix + torch.arange(i) for i in (*questions, 3)]).to(DEV)
    logits, seen = model(torch.randint(0, VOCAB, (16,), generator=g).to(DEV), positions, *rows)
    model.check(seen, *rows)
    last = logits[_ints(8, 12)]
    first = token_scores(last, torch.zeros(2, 0, dtype=torch.int64, device=DEV), top=3)
    assert torch.equal(first.top_ids.cpu(), S.token_scores(last.cpu(), torch.zeros(2, 0, dtype=torch.int64), 3)[3])

    # tokens one by one: the next ones are chosen, and the lengths raised, on the GPU
    token, lengths = first.top_ids[:, 0].contiguous(), rows[1].clone()

    def step():
        lengths.add_(1)
        logits, seen = model(token, lengths - 1, table, lengths)
        scores = token_scores(logits, token[:, None].long(), top=5)
        return logits, seen, scores

    before = [[getattr(layer.cache, name).clone() for name in held] for layer, held in zip(model.layers, model.held)]
    step()                                             # warms up; its writes are taken back
    lengths.sub_(1)
    for layer, held, kept in zip(model.layers, model.held, before):
        for name, x in zip(held, kept):
            getattr(layer.cache, name).copy_(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, seen, scores = step()
        chosen = scores.top_ids[:, 0].clone()
    for turn in range(6):
        fed = token.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert lengths.tolist() == [prefix + i + turn + 1 for i in questions]
        model.check(seen, table, lengths, None)
        _check(logits.cpu(), fed[:, None].long().cpu(), 5)
        eager = token_scores(logits, fed[:, None].long(), top=5)
        for a, b in zip(scores, eager):
            assert torch.equal(a, b)
        again, _ = model(fed, lengths - 1, table, lengths)             # the same positions written once more
        assert torch.equal(again, logits)
        token.copy_(chosen)
