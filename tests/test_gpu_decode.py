"""Generation with a MambaStack in 8 bits, and the stack with its head in 8 bits.

Bounds. An e4m3 value is off by at most 2^-4 of itself (rms about 2.6 %), so a
product of two such operands by about 3.7 % of its norm; two blocks and a head
stay below 15 % of the logits' norm. Two ways through the same 8-bit weights
(prompt and single tokens) differ by bfloat16 roundings (2^-8) and the codes
that those flip: below 4 %.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _stack(vocab=50, d=96, layers=2, seed=3, **kw):
    from mamba.block import MambaStack

    stack = MambaStack(vocab, d, layers, dtype=torch.bfloat16, seed=seed, **kw)
    with torch.no_grad():  # logits of order 1
        stack.head *= d ** 0.5
        stack.embed *= d ** 0.5
    return stack


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(21)


def _rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("batch,length", [(1, 1), (3, 7), (2, 40), (5, 130)])
def test_prefill_follows_the_stack(batch, length):
    from mamba import MambaDecoder

    stack = _stack()
    tokens = torch.randint(0, 50, (batch, length), device="cuda")
    logits, state = MambaDecoder(stack).prefill(tokens)
    assert logits.shape == (batch, 50) and logits.dtype == torch.float32 and len(state) == 2
    with torch.no_grad():
        assert _rel(logits, stack(tokens)[:, -1]) < 0.15


@pytest.mark.parametrize("start", [1, 3, 20])
def test_steps_continue_the_prompt(start):
    from mamba import MambaDecoder

    dec = MambaDecoder(_stack())
    tokens = torch.randint(0, 50, (4, 25), device="cuda")
    logits, state = dec.prefill(tokens[:, :start])
    for t in range(start, 25):
        logits = dec.step(tokens[:, t], state)
    want, want_state = dec.prefill(tokens)
    assert _rel(logits, want) < 0.04
    for (conv, scan), (wconv, wscan) in zip(state, want_state):
        assert _rel(conv, wconv) < 0.04 and _rel(scan, wscan) < 0.04


def test_padded_prompts():
    """Each row of a padded batch as the row alone."""
    from mamba import MambaDecoder

    dec = MambaDecoder(_stack())
    lens = torch.tensor([1, 2, 9, 30], dtype=torch.int32, device="cuda")
    tokens = torch.randint(0, 50, (4, 30), device="cuda")
    logits, state = dec.prefill(tokens, lens)
    nxt = torch.randint(0, 50, (4,), device="cuda")
    after = dec.step(nxt, state)
    for r, n in enumerate(lens.tolist()):
        alone, s = dec.prefill(tokens[r:r + 1, :n])
        assert _rel(logits[r:r + 1], alone) < 0.04
        assert _rel(after[r:r + 1], dec.step(nxt[r:r + 1], s)) < 0.04


def test_generate():
    from mamba import MambaDecoder, sample_tokens

    dec = MambaDecoder(_stack())
    tokens = torch.randint(0, 50, (3, 12), device="cuda")
    u = torch.rand(3, 6, device="cuda")
    kw = dict(temperature=0.8, top_k=10, top_p=0.95)
    got = dec.generate(tokens, 6, uniform=u, **kw)
    logits, state = dec.prefill(tokens)
    for t in range(6):
        tok = sample_tokens(logits, u[:, t].contiguous(), **kw)
        assert torch.equal(tok, got[:, t])
        logits = dec.step(tok, state)
    greedy = dec.generate(tokens, 4, temperature=0.0)
    assert torch.equal(greedy[:, 0], dec.prefill(tokens)[0].argmax(1))
    g = lambda: torch.Generator("cuda").manual_seed(5)  # noqa: E731
    assert torch.equal(dec.generate(tokens, 5, generator=g()), dec.generate(tokens, 5, generator=g()))
    assert dec.generate(tokens, 0).shape == (3, 0)


def test_head_in_8_bits_gradients():
    """The head alone on given hidden states and a given gradient of the logits:
    logits and all gradients beside the exact head's. Each is one product of
    8-bit operands (rms error 3.7 % of its norm, the roundings being independent),
    for the norm's weight and input followed by the norm's backward, which mixes
    columns but does not enlarge: below 10 %."""
    from mamba import fp8_linear, rms_norm_fn

    g = torch.Generator("cuda").manual_seed(11)
    h = torch.randn(4, 33, 96, generator=g, device="cuda")
    head = torch.randn(50, 96, generator=g, device="cuda")
    weight = torch.rand(96, generator=g, device="cuda") + 0.5
    dy = torch.randn(4, 33, 50, generator=g, device="cuda")
    got = []
    for exact in (True, False):
        x, w, n = (t.clone().requires_grad_() for t in (h, head, weight))
        if exact:
            y = torch.nn.functional.rms_norm(x, (96,), n, 1e-5) @ w.t()
        else:
            y = fp8_linear(rms_norm_fn(x.bfloat16(), n), w.bfloat16()).float()
        got.append((y, *torch.autograd.grad(y, (x, w, n), dy)))
    for a, b in zip(*got):
        assert _rel(b, a) < 0.1


def test_head_in_8_bits_trains():
    """Steps down the gradient lower the loss of a fixed batch."""
    torch.manual_seed(12)
    m = _stack(seed=9, fp8_head=True)
    tokens = torch.randint(0, 50, (4, 33), device="cuda")
    opt = torch.optim.SGD(m.parameters(), lr=0.02)
    losses = []
    for _ in range(12):
        out = m(tokens)
        assert out.dtype == torch.float32
        loss = torch.nn.functional.cross_entropy(out.flatten(0, 1), tokens.flatten())
        opt.zero_grad()
        loss.backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
        opt.step()
        losses.append(loss.item())
    assert losses[-1] < 0.9 * losses[0]


def test_refusals():
    from mamba import MambaDecoder

    with pytest.raises(ValueError, match="rmsnorm"):
        MambaDecoder(_stack(norm_type="layernorm"))
    with pytest.raises(ValueError, match="rmsnorm"):
        _stack(norm_type="layernorm", fp8_head=True)
    dec = MambaDecoder(_stack())
    with pytest.raises(ValueError, match="L >= 1"):
        dec.prefill(torch.zeros(2, 0, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="uniform"):
        dec.generate(torch.zeros(2, 3, dtype=torch.int64, device="cuda"), 4,
                     uniform=torch.rand(2, 3, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weights_are_copies(dtype):
    """A decoder answers the same after its stack has trained on."""
    from mamba import MambaDecoder

    stack = _stack()
    dec = MambaDecoder(stack, dtype=dtype)
    tokens = torch.randint(0, 50, (3, 9), device="cuda")
    want, state = dec.prefill(tokens)
    step = dec.step(tokens[:, 0], state)
    with torch.no_grad():
        for p in stack.parameters():
            p.add_(torch.rand_like(p) + 0.5)
    got, state = dec.prefill(tokens)
    assert torch.equal(got, want) and torch.equal(dec.step(tokens[:, 0], state), step)


def test_rows_with_nothing_to_draw():
    """-1 is no token of the vocabulary: a row that has it gives NaN, and -1 from there
    on; the other rows do not notice."""
    from mamba import MambaDecoder, sample_tokens

    stack = _stack()
    with torch.no_grad():
        stack.embed[7] = float("nan")
    dec = MambaDecoder(stack)
    tokens = torch.randint(8, 50, (4, 11), device="cuda")
    u = torch.rand(4, 5, device="cuda")
    want = dec.generate(tokens, 5, uniform=u)
    bad = tokens.clone()
    bad[1, 4] = 7
    got = dec.generate(bad, 5, uniform=u)
    assert (got[1] == -1).all() and torch.equal(got[[0, 2, 3]], want[[0, 2, 3]])
    bad[1, 4], bad[3, 10] = -1, -1
    logits, state = dec.prefill(bad)
    plain, plain_state = dec.prefill(tokens)
    for nxt in (tokens[:, 0], torch.tensor([3, -1, -1, 5], device="cuda"), tokens[:, 2]):
        gone = logits.isnan().all(1)
        assert not logits[~gone].isnan().any() and torch.equal(logits[~gone], plain[~gone])
        assert torch.equal(sample_tokens(logits, u[:, 0]) == -1, gone)
        logits, plain = dec.step(nxt, state), dec.step(nxt.clamp(min=0), plain_state)
    assert logits.isnan().all(1).tolist() == [False, True, True, True]


def test_lengths_outside_the_prompt():
    """A row of length 0 reads no other row's position: NaN logits and the state before
    any token; a length above L is L."""
    from mamba import MambaDecoder

    dec = MambaDecoder(_stack())
    tokens = torch.randint(0, 50, (5, 30), device="cuda")
    nxt = torch.randint(0, 50, (5,), device="cuda")
    logits, state = dec.prefill(
        tokens, torch.tensor([0, 5, 41, 0, -2], dtype=torch.int32, device="cuda"))
    assert logits.isnan().all(1).tolist() == [True, False, False, True, True]
    for conv, scan in state:
        assert (conv[[0, 3, 4]] == 0).all() and (scan[[0, 3, 4]] == 0).all()
    want, want_state = dec.prefill(
        tokens, torch.tensor([1, 5, 30, 7, 2], dtype=torch.int32, device="cuda"))
    assert torch.equal(logits[1:3], want[1:3])
    after, want_after = dec.step(nxt, state), dec.step(nxt, want_state)
    assert torch.equal(after[1:3], want_after[1:3])
    first = dec.prefill(nxt[:, None])[0]  # the rows' first token
    assert _rel(after[[0, 3, 4]], first[[0, 3, 4]]) < 0.04
    got = dec.generate(tokens, 3, seq_lens=torch.tensor([9, 0, 3, 1, 30], dtype=torch.int32,
                                                        device="cuda"))
    assert (got[1] == -1).all() and (got[[0, 2, 3, 4]] >= 0).all()


def test_lengths_that_are_refused():
    from mamba import MambaDecoder

    dec = MambaDecoder(_stack())
    tokens = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    for bad in (torch.ones(2, dtype=torch.int32), torch.ones(2, device="cuda"),
                torch.ones(3, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError, match="seq_lens"):
            dec.prefill(tokens, bad)


def test_head_in_8_bits_rounds_to_8_bits_alone():
    """Norm of the float32 stream, 8-bit operands from its float32 result and the float32
    weight, float32 sums and gradients: nothing passes through the stack's bfloat16."""
    from mamba import fp8_matmul, quantize_fp8, rms_norm_fn

    m = _stack(seed=9, fp8_head=True)
    tokens = torch.randint(0, 50, (4, 33), device="cuda")
    x = m.embed[tokens]
    for layer in m.layers:
        x = layer(x)
    y = rms_norm_fn(x, m.norm.weight, eps=1e-5).flatten(0, 1).detach()
    want = fp8_matmul(*quantize_fp8(y), *quantize_fp8(m.head.detach()), out_dtype=torch.float32)
    out = m(tokens)
    assert torch.equal(out.flatten(0, 1), want)
    dy = torch.randn(4 * 33, 50, device="cuda")
    dhead, = torch.autograd.grad(out, m.head, dy.view(4, 33, 50))
    assert torch.equal(dhead, fp8_matmul(*quantize_fp8(dy.t()), *quantize_fp8(y.t()),
                                         out_dtype=torch.float32))


def test_weights_are_rounded_once():
    """The 8-bit weights are those of the stack's float32 ones."""
    from mamba import MambaDecoder, quantize_fp8

    stack = _stack()
    dec = MambaDecoder(stack)
    pairs = [(dec.head, stack.head)]
    for a, b in zip(dec.layers, stack.layers):
        pairs += [(a.w_main, b.w_main), (a.w_skip, b.w_skip), (a.w_out, b.w_out)]
    for got, w in pairs:
        for a, b in zip(got, quantize_fp8(w.detach())):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
