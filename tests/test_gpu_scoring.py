"""Log probabilities, entropy and alternatives against float64.

Tolerances. Z sums up to 2^17 terms of one sign in f32 over 256 or more threads: each thread adds at
most 2^9 terms, the rest a tree, so Z is off by at most 2^-14 of itself in the worst order of
roundings, and the exponentials' arguments x log2 e - m log2 e by 2^-23 |x log2 e| each. Random
roundings stay far below; the bound taken is 2^-14 + 2^-22 max |x - m| absolute on log
probabilities, and on the entropy 2^-14 + 2^-20 of it times the same (its sum T has terms of one
sign as well). Indices and order are exact: they compare the logits themselves."""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def bound():
    from ppy_b200 import runtime

    if not torch.cuda.is_available():
        pytest.fail("a GPU test ran without a CUDA device")
    runtime.init(0)
    runtime.set_stream(torch.cuda.current_stream())


def _check(logits, tokens, top):
    from ppy_b200 import scoring

    got = scoring.token_logprobs(logits, tokens, top)
    x = logits.double()
    vocab = x.shape[-1]
    want = torch.log_softmax(x, -1)
    given = tokens if tokens.dim() == logits.dim() else tokens[..., None]
    valid = (given >= 0) & (given < vocab)
    ref = torch.where(valid, want.gather(-1, given.clamp(0, vocab - 1)), math.nan)
    finite = x.masked_fill(x.isinf(), 0.0)
    span = float((finite.amax(-1) - finite.amin(-1)).nan_to_num(0.0).max())
    tol = 2.0 ** -14 + 2.0 ** -22 * span

    def same(a, b, tol):
        a = a.double()
        assert a.shape == b.shape
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.isinf(), b.isinf())
        fine = b.isfinite()
        assert not fine.any() or float((a[fine] - b[fine]).abs().max()) <= tol

    same(got.logprobs.view(ref.shape), ref, tol)
    p = want.exp()
    entropy = -(torch.where(p > 0, p * want, 0.0)).sum(-1)
    entropy = torch.where(want.isnan().any(-1), math.nan, entropy)
    same(got.entropy, entropy, tol * (1 + float(entropy.nan_to_num(0.0).max())))
    # NaN sorts first, equal values by index
    order = x.sort(dim=-1, descending=True, stable=True).indices[..., :top]
    assert torch.equal(got.top_tokens, order)
    same(got.top_logprobs, want.gather(-1, order), tol)
    return got


def _tokens(shape, vocab, g):
    return torch.randint(0, vocab, shape, device="cuda", generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab,pitch,top", [
    (1, 1, 1, 1), (3, 7, 7, 7), (2, 33, 40, 5), (1, 50257, 50272, 5), (4, 50257, 50257, 64),
    (400, 1000, 1001, 20), (300, 50257, 50257, 3), (17, 4099, 4099, 64), (5, 129001, 129001, 0),
    (320, 63, 63, 63),
])
def test_rows(dtype, rows, vocab, pitch, top):
    g = torch.Generator(device="cuda").manual_seed(rows)
    store = 4 * torch.randn(rows * pitch + 3, device="cuda", generator=g)
    # rows that start anywhere
    logits = store.to(dtype)[3:].view(rows, pitch)[:, :vocab]
    _check(logits, _tokens((rows,), vocab, g), top)
    _check(logits, _tokens((rows, 3), vocab, g), top)


@pytest.mark.parametrize("rows", [2, 400])
def test_odd_rows(rows):
    """Infinities, NaN, equal logits in numbers, sharp and huge rows, tokens out of range."""
    g = torch.Generator(device="cuda").manual_seed(8)
    vocab, top = 5003, 20
    plain = torch.randn(rows, vocab, device="cuda", generator=g)
    tokens = _tokens((rows,), vocab, g)

    def with_(change):
        x = plain.clone()
        change(x)
        _check(x, tokens, top)

    with_(lambda x: x.fill_(0.25))                                  # all equal
    with_(lambda x: x.fill_(-0.0).__setitem__((..., slice(9, 2000)), 0.0))  # both zeros
    with_(lambda x: x[:, 7:].fill_(-math.inf))                      # fewer left than asked for
    with_(lambda x: x[:, :4990].fill_(-math.inf))
    with_(lambda x: x.fill_(-math.inf))
    with_(lambda x: x[:, 11::50].fill_(math.nan))
    with_(lambda x: x[:, 4000].fill_(math.inf))
    with_(lambda x: x[:, [3, 4001, 4002]].fill_(math.inf))
    with_(lambda x: x[:, 77].fill_(1e4))                            # one certain token
    with_(lambda x: x.mul_(1e30))
    with_(lambda x: x.fill_(torch.finfo(torch.float32).min))        # the lowest value everywhere
    with_(lambda x: x[:, 100:].fill_(torch.finfo(torch.float32).min))
    with_(lambda x: x.copy_(torch.arange(vocab, device="cuda") / 64))      # climbing
    with_(lambda x: x.copy_(-torch.arange(vocab, device="cuda") / 64))
    # a few slots hold everything large: more candidates than there is room for
    index = torch.arange(vocab, device="cuda")
    with_(lambda x: x.copy_(torch.where(index // 4 % 256 < 80, 100.0 + index / 8192, 0.0)))
    with_(lambda x: x.mul_(8).round_().div_(8))                     # many equal ones
    tokens[0] = -1
    tokens[1] = vocab
    _check(plain, tokens, top)


def test_leading_shapes_and_no_rows():
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(2, 5, 96, device="cuda", generator=g)[:, :, :70]
    _check(logits, _tokens((2, 5), 70, g), 4)
    _check(logits, _tokens((2, 5, 2), 70, g), 4)
    _check(logits[:, 2], _tokens((2,), 70, g), 4)       # rows further apart
    _check(logits[1, 3], _tokens((), 70, g), 4)         # one row
    from ppy_b200 import scoring

    none = scoring.token_logprobs(logits[:0], _tokens((0, 5), 70, g), 4)
    assert [tuple(t.shape) for t in none] == [(0, 5), (0, 5), (0, 5, 4), (0, 5, 4)]


def test_gpt2_scores_a_prompt():
    from ppy_b200 import gpt2

    model = gpt2.GPT2(gpt2.Config(layers=1), seed=1)
    ids = torch.randint(0, 50257, (2, 128), device="cuda")
    logits = model.forward(ids)
    scored = model.score(ids, top=3, logits=logits)
    want = torch.log_softmax(logits.double(), -1)[:, :-1]
    assert float((scored.logprobs.double() - want.gather(-1, ids[:, 1:, None])[..., 0]).abs()
                 .max()) < 1e-4
    assert float((scored.entropy.double() + (want.exp() * want).sum(-1)).abs().max()) < 1e-3
    assert torch.equal(scored.top_tokens[..., 0], logits[:, :-1].argmax(-1))
    assert scored.top_logprobs.shape == (2, 127, 3)
