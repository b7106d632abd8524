"""Token sampling against the float64 oracle. A draw is checked where its
uniform number lies in the middle of a kept token's interval (so that no
rounding can move it to a neighbour), and the filters at cutoffs between two
tokens; the answer is then a single token."""
import numpy as np
import pytest
import torch

from oracle import lm_ops_oracle as orc

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _logits(rows, vocab, seed, dtype, sharp=2.5):
    g = np.random.default_rng(seed)
    return torch.from_numpy(sharp * g.standard_normal((rows, vocab))).to(dtype).cuda()


def _run(logits, u, **kw):
    from mamba import sample_tokens

    dev = {k: torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v for k, v in kw.items()}
    return sample_tokens(logits, torch.from_numpy(np.asarray(u, np.float32)).cuda(), **dev).cpu().numpy()


def _middles(row, n, **kw):
    """Uniform numbers in the middle of kept tokens' intervals, and the tokens."""
    _, kept, prob = orc.sample(row, 0.0, **kw)
    end = np.cumsum(prob)
    wide = np.flatnonzero(prob > 1e-4)
    pick = wide[np.linspace(0, wide.size - 1, n).astype(int)]
    return end[pick] - prob[pick] / 2, kept[pick]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 17, 100, 2047, 4100, 10000, 50280, 131072])
@pytest.mark.parametrize("kw", [{}, {"temperature": 0.6}, {"top_k": 1}, {"top_k": 3}, {"top_k": 40},
                                {"top_k": 2000}, {"min_p": 0.05}, {"temperature": 0.0}],
                         ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()) or "plain")
def test_draws(vocab, dtype, kw):
    n = 9
    z = _logits(1, vocab, vocab, dtype)
    row = z.double().cpu().numpy()[0]
    u, want = _middles(row, n, **kw)
    got = _run(z.expand(n, vocab), u, **kw)
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("vocab", [5, 300, 5000, 50280])
@pytest.mark.parametrize("top_k", [0, 50])
def test_top_p_cutoffs(vocab, top_k):
    """top_p between two tokens' cumulative probabilities: the one before it is
    kept, the next is not. The last kept token's interval and, above it, u near
    1 (the last kept by index) tell."""
    z = _logits(1, vocab, 7 + vocab, F32)
    row = z.double().cpu().numpy()[0]
    order = np.argsort(-row, kind="stable")[:top_k or vocab]
    p = np.exp(row[order] - row.max())
    p /= p.sum()
    cum = np.cumsum(p)
    for at in sorted({0, 1, 2, min(7, order.size - 2), min(45, order.size - 2)}):
        if at < 0 or at + 1 >= order.size or p[at + 1] < 1e-5:
            continue
        top_p = float(np.float32(cum[at] - p[at] / 2))
        u, want = _middles(row, 5, top_k=top_k, top_p=top_p)
        _, kept, _ = orc.sample(row, 0.0, top_k=top_k, top_p=top_p)
        assert kept.size == at + 1
        np.testing.assert_array_equal(_run(z.expand(5, vocab), u, top_k=top_k, top_p=top_p), want)


def test_parameters_per_row():
    rows, vocab = 24, 3000
    z = _logits(rows, vocab, 3, F32)
    rng = np.random.default_rng(4)
    kw = {"temperature": rng.choice([0.0, 0.7, 1.0, 1.4], rows).astype(np.float32),
          "top_k": rng.choice([0, 1, 5, 200], rows).astype(np.int32),
          "top_p": rng.choice([1.0, 0.9, 0.4], rows).astype(np.float32),
          "min_p": rng.choice([0.0, 0.03], rows).astype(np.float32)}
    u, want = np.zeros(rows), np.zeros(rows, int)
    for r in range(rows):
        one = {k: v[r].item() for k, v in kw.items()}
        us, ws = _middles(z[r].double().cpu().numpy(), 3, **one)
        u[r], want[r] = us[1], ws[1]
    np.testing.assert_array_equal(_run(z, u, **kw), want)


@pytest.mark.parametrize("vocab", [700, 9000, 70000])
def test_ties_go_to_the_lowest_index(vocab):
    """Rows of equal logits: more in one bin than is ever sorted, and a cutoff
    that only the index decides."""
    z = torch.zeros(4, vocab, device="cuda")
    k = 300
    u = np.array([0.5 / k, (k - 0.5) / k, 0.0, 7.5 / k], np.float32)
    want = np.array([0, k - 1, 0, 7])
    np.testing.assert_array_equal(_run(z, u, top_k=k), want)
    top_p = (k - 0.5) / vocab  # k tokens: the k-th's predecessors hold (k - 1) / vocab
    np.testing.assert_array_equal(_run(z, u, top_p=top_p), want)
    np.testing.assert_array_equal(_run(z, u, temperature=0.0), 0)
    z[:, 5] = 1.0
    np.testing.assert_array_equal(_run(z, u, top_k=1), 5)
    # both filters: of the k first the ones ahead of half their mass
    z[:, 5] = 0.0
    np.testing.assert_array_equal(_run(z, [0.0, 0.999, 0.5, 0.25], top_k=k, top_p=0.5),
                                  [0, 149, 75, 37])


def test_masks_and_special_values():
    inf = float("inf")
    z = torch.full((8, 5000), -inf, device="cuda")
    z[0, 4000] = -3.0                       # one token left
    z[1, 10], z[1, 20] = 2.0, 2.0           # two
    z[2] = torch.nan                        # none
    z[4, 7], z[4, 9] = torch.nan, 1.0       # NaN is masked
    z[5] = torch.finfo(F32).min             # the type's lowest value everywhere: all equal
    z[6, 100], z[6, 200], z[6, 300] = inf, inf, 5.0   # only infinities have weight
    z[7] = torch.finfo(F32).min
    z[7, 42] = 0.0
    for kw in ({}, {"top_k": 3}, {"top_p": 0.9}, {"top_k": 3, "top_p": 0.9, "min_p": 0.1}):
        got = _run(z, [0.3, 0.75, 0.5, 0.5, 0.9, 0.0, 0.75, 0.99], **kw)
        np.testing.assert_array_equal(got, [4000, 20, -1, -1, 9, 0, 200, 42])
    got = _run(z, [0.5] * 8, temperature=0.0)
    np.testing.assert_array_equal(got, [4000, 10, -1, -1, 9, 0, 100, 42])
    assert _run(z[:0], np.zeros(0)).shape == (0,)


def test_uniform_numbers_at_the_ends():
    """0 is the first kept token, the largest float below 1 the last; 1 itself,
    outside the contract, stays inside the row."""
    z = _logits(3, 6000, 9, F32)
    for kw in ({}, {"top_k": 4}, {"top_p": 0.7}):
        kept = [orc.sample(r, 0.0, **kw)[1] for r in z.double().cpu().numpy()]
        np.testing.assert_array_equal(_run(z, [0.0] * 3, **kw), [k[0] for k in kept])
        for u in (1 - 2.0 ** -24, 1.0):
            got = _run(z, [u] * 3, **kw)
            if kw:
                np.testing.assert_array_equal(got, [k[-1] for k in kept])
            assert (got >= 0).all() and (got < 6000).all()


def test_strides_streams_and_sums_of_draws():
    from mamba import sample_tokens

    big = _logits(6, 9000, 11, BF16)
    u = torch.rand(6, device="cuda")
    for view in (big[:, :8001], big[:, 3:8000], big[::2, :64], big.t()[:6, :6].contiguous().t()):
        n = view.shape[0]
        want = sample_tokens(view.contiguous(), u[:n], top_k=20, top_p=0.9)
        assert torch.equal(sample_tokens(view, u[:n], top_k=20, top_p=0.9), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = sample_tokens(big * 1, u, top_k=20)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, sample_tokens(big, u, top_k=20))
    # many draws of one row: frequencies within 5 standard deviations
    p = torch.tensor([0.05, 0.5, 0.15, 0.3], device="cuda")
    n = 40000
    t = sample_tokens(p.log().expand(n, 4), torch.rand(n, device="cuda"))
    freq = torch.bincount(t, minlength=4) / n
    assert ((freq - p).abs() < 5 * (p * (1 - p) / n).sqrt()).all()


def test_refusals():
    from mamba import sample_tokens

    z, u = torch.randn(4, 100, device="cuda"), torch.rand(4, device="cuda")
    with pytest.raises(TypeError):
        sample_tokens(z.half(), u)
    with pytest.raises(ValueError, match="vocab"):
        sample_tokens(z[0], u)
    with pytest.raises(ValueError, match="vocab"):
        sample_tokens(torch.empty(1, 360449, device="cuda"), u[:1])
    with pytest.raises(ValueError, match="uniform"):
        sample_tokens(z, u[:3])
    with pytest.raises(ValueError, match="uniform"):
        sample_tokens(z, u.double())
    with pytest.raises(ValueError, match="top_k"):
        sample_tokens(z, u, top_k=torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="temperature"):
        sample_tokens(z, u, temperature=torch.ones(3, device="cuda"))


@pytest.mark.parametrize("rows,vocab", [(700, 900), (2100, 300), (300, 30000)])
def test_many_rows_of_mixed_cost(rows, vocab):
    """Rows in one call, more than run at once, as the same rows a few at a time:
    their order of execution does not show."""
    z = _logits(rows, vocab, rows, BF16)
    rng = np.random.default_rng(rows)
    kw = {"temperature": rng.choice([0.0, 0.7, 1.0], rows).astype(np.float32),
          "top_k": rng.choice([0, 1, 30, 600], rows).astype(np.int32),
          "top_p": rng.choice([1.0, 0.9, 0.4], rows).astype(np.float32),
          "min_p": rng.choice([0.0, 0.02], rows).astype(np.float32)}
    u = rng.random(rows).astype(np.float32)
    got = _run(z, u, **kw)
    for lo in range(0, rows, 50):
        part = slice(lo, lo + 50)
        np.testing.assert_array_equal(
            got[part], _run(z[part], u[part], **{k: v[part] for k, v in kw.items()}))


@pytest.mark.parametrize("vocab", [900, 5003, 50280, 131072])
@pytest.mark.parametrize("top_k", [0, 60, 500, 700])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_filters_together(vocab, top_k, dtype):
    """Every pair of top-p and min-p with each kind of top-k and a temperature."""
    z = _logits(1, vocab, vocab + top_k, dtype)
    # logit / temperature is defined in 32 bits: the oracle takes the quotients
    row = z.float().cpu().numpy()[0] / np.float32(1.3)
    for top_p in (1.0, 0.9, 0.35):
        for min_p in (0.0, 0.004, 0.3):
            kw = {"top_k": top_k, "top_p": float(np.float32(top_p)), "min_p": float(np.float32(min_p))}
            u, want = _middles(row, 6, **kw)
            np.testing.assert_array_equal(_run(z.expand(6, vocab), u, temperature=1.3, **kw), want)


@pytest.mark.parametrize("vocab", [1500, 2040, 9000])
@pytest.mark.parametrize("min_p", [0.0, float(np.float32(np.exp(-400.5 * 2.0 ** -20)))])
def test_cutoff_among_many_close_logits(vocab, min_p):
    """Distinct logits so close that the cutoff's bin holds hundreds to thousands:
    within one list, at its end, and past it; and min-p, halfway between two weights,
    cuts within the same bin."""
    rng = np.random.default_rng(vocab)
    row = rng.permutation(vocab) * np.float32(2.0 ** -20)
    z = torch.from_numpy(row.astype(np.float32))[None].cuda()
    row = z.double().cpu().numpy()[0]
    order = np.argsort(-row, kind="stable")
    p = np.exp(row[order])
    p /= p.sum()
    cum = np.cumsum(p)
    for at in (0, vocab // 3, vocab - 2):
        top_p = float(np.float32(cum[at] - p[at] / 2))
        u, want = _middles(row, 9, top_p=top_p, min_p=min_p)
        np.testing.assert_array_equal(_run(z.expand(9, vocab), u, top_p=top_p, min_p=min_p), want)
        u, want = _middles(row, 9, top_k=at + 1, min_p=min_p)
        np.testing.assert_array_equal(_run(z.expand(9, vocab), u, top_k=at + 1, min_p=min_p), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [50, 9000])
def test_quotients_past_the_largest_float(dtype, vocab):
    """Rows whose logit / temperature is not finite: the largest logits remain, all
    with the same weight; the type's lowest value is a value, not a mask."""
    z = torch.full((5, vocab), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    z[1] = -1.0
    z[1, 4], z[1, 40] = 3.0, 3.0                  # temperature 1e-39
    z[2, 7], z[2, 8], z[2, 9] = 3e38, 2e38, 3e38  # temperature 0.5
    z[3, 1] = float("inf")                        # temperature inf
    z[4] = -float("inf")
    t = np.array([0.7, 1e-39, 0.5, np.inf, 0.7], np.float32)
    u = [0.99, 0.75, 0.25, 0.5, 0.5]
    last = int(np.floor(np.float64(np.float32(0.99)) * vocab))
    for kw in ({}, {"top_k": vocab - 1}, {"top_p": 0.9999}, {"min_p": 0.5}):
        got = _run(z, u, temperature=t, **kw)
        # top_k leaves out the last of the equal ones, top_p at most one
        assert last - 1 <= got[0] <= last
        np.testing.assert_array_equal(got[1:], [40, 7, 1, -1])
    np.testing.assert_array_equal(_run(z, u, temperature=t, top_k=2), [1, 40, 7, 1, -1])
    np.testing.assert_array_equal(_run(z, u, temperature=t, top_k=1), [0, 4, 7, 1, -1])


@pytest.mark.parametrize("name", ["temperature", "top_k", "top_p", "min_p"])
def test_parameters_that_are_not_numbers(name):
    from mamba import sample_tokens

    z, u = torch.randn(2, 10, device="cuda"), torch.rand(2, device="cuda")
    for bad in ("1", None, [1.0, 1.0]):
        with pytest.raises(TypeError):
            sample_tokens(z, u, **{name: bad})
    one = np.float32(1.0) if name != "top_k" else np.int32(1)
    assert sample_tokens(z, u, **{name: one}).shape == (2,)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(200, 5000), (600, 5000), (300, 9001)])
@pytest.mark.parametrize("kw", [{"top_k": 2}, {"top_k": 50}, {"top_k": 300},
                                {"top_k": 50, "top_p": 0.5}, {"top_k": 300, "top_p": 0.5},
                                {"top_k": 500, "top_p": 0.9}],
                         ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()))
def test_more_candidates_than_a_list_holds(rows, vocab, kw, dtype):
    """Rows of one CTA each whose bound leaves more than 2048 candidates: all equal, all
    equal but a few above, and equal where a mask leaves them. The draw then goes from the
    list to the general way, in every thread of the CTA."""
    z = torch.zeros(rows, vocab, device="cuda", dtype=dtype)
    z[1::3, 7], z[1::3, vocab - 3] = 1.0, 2.0
    z[2::3, ::2] = -float("inf")
    u, want = np.zeros(rows), np.zeros(rows, int)
    for kind in range(3):
        us, ws = _middles(z[kind].double().cpu().numpy(), 31, **kw)
        at = np.arange(kind, rows, 3)
        u[at], want[at] = us[at % us.size], ws[at % ws.size]
    for _ in range(4):
        np.testing.assert_array_equal(_run(z, u, **kw), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_calls_from_several_host_threads(dtype):
    """Through the C interface, whose calls run at the same time in several host threads:
    rows that need most of an SM's shared memory, and rows that need little."""
    import threading

    from mamba import _native

    lib = _native.load()
    code = {F32: 0, BF16: 1}[dtype]
    failed = []

    def calls(vocab):
        z = torch.zeros(4, vocab, device="cuda", dtype=dtype)
        z[:, 5] = 9.0
        u = torch.rand(4, device="cuda")
        t = torch.empty(4, dtype=torch.int64, device="cuda")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        for _ in range(3000):
            if lib.mamba_ss_sample_tokens(s.cuda_stream, code, 4, vocab, z.data_ptr(), vocab,
                                          u.data_ptr(), None, None, None, None, 0.0, 0, 1.0, 0.0,
                                          t.data_ptr()):
                failed.append((vocab, lib.mamba_ss_last_error()))
                break
        s.synchronize()
        if not (t == 5).all():
            failed.append((vocab, t.tolist()))

    threads = [threading.Thread(target=calls, args=(v,)) for v in (360448, 64, 9000, 1000)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed
