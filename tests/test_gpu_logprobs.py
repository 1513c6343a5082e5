"""token_logprobs on the GPU against log_softmax in 64 bits, at the vocabularies, alignments, ties and
infinities where it can go wrong."""

import math

import pytest
import torch

from kernels.sample import token_logprobs

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def check(x, tokens, top):
    """x [rows, V] on the GPU. The order of the alternatives is exact; the values: every exponent y and its
    exp2 to a few 2^-24, V terms summed in order by at least 64 lanes, logarithms to 2^-22 of themselves."""
    r = token_logprobs(x, tokens, top)
    d = x.double()
    V = x.shape[1]
    logp = torch.log_softmax(d, -1)
    p = logp.exp()
    entropy = -torch.special.xlogy(p, p).sum(-1)
    sums = (V / 64 + 64) * 2.0 ** -24  # of the sums, relative: an absolute error of a logarithm
    want = logp.gather(1, tokens.clamp(0, V - 1)[:, None])[:, 0]
    want = torch.where((tokens >= 0) & (tokens < V), want, NAN)

    def near(got, ref, what):
        assert got.dtype == torch.float32 and got.shape == ref.shape
        assert torch.equal(got.isnan(), ref.isnan()), what
        ok = ref.isfinite()
        assert torch.equal(got[~ok & ~ref.isnan()].double(), ref[~ok & ~ref.isnan()]), what
        e = (got.double() - ref)[ok].abs() - (sums + 2.0 ** -21 * ref[ok].abs())
        assert not e.numel() or e.max() <= 0, (what, float(e.max()))

    near(r.logprob, want, "logprob")
    # entropy: ln s - sum / s, both of up to ln V and of the exponents' mean
    size = math.log(V) + 1
    ok = entropy.isfinite()
    assert torch.equal(r.entropy.isnan(), ~ok)
    assert not ok.any() or (r.entropy.double() - entropy)[ok].abs().max() <= 2 * sums * size + 2.0 ** -21 * size
    order = x.float()
    ids = torch.sort(torch.where(order.isnan(), INF, order), dim=-1, descending=True, stable=True).indices[:, :top]
    has_nan = order.isnan().any(-1) & (order == INF).any(-1)  # NaN before +inf: checked by itself
    assert torch.equal(r.top_ids[~has_nan], ids[~has_nan])
    near(r.top_logprobs, logp.gather(1, r.top_ids), "top")
    return r


def logits(rows, V, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 2.5 * torch.randn(rows, V, device="cuda", generator=g)
    x[:, ::97] += 6
    t = torch.randint(0, V, (rows,), device="cuda", generator=g)
    return x.to(dtype), t


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (1, 5, 5), (3, 17, 4), (1, 151936, 5), (2, 32003, 20), (9, 1024, 64),
                                        (5, 1025, 0), (300, 4097, 8), (7, 50257, 33), (1100, 5000, 20), (2, 9000, 64)])
def test_against_float64(dtype, rows, V, top):
    x, t = logits(rows, V, dtype)
    check(x, t, top)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_rows_of_any_alignment(dtype, shift):
    """A slice of wider rows: every row begins at another alignment, what surrounds it is NaN."""
    wide = torch.full((13, 2113), NAN, device="cuda", dtype=dtype)
    x, t = logits(13, 2100, dtype)
    wide[:, shift:shift + 2100] = x
    check(wide[:, shift:shift + 2100], t, 7)


def test_many_rows():
    x, t = logits(70001, 17, torch.float16)
    check(x, t, 3)


@pytest.mark.parametrize("V", [100, 3000, 40000])
@pytest.mark.parametrize("kind", ["constant", "two values", "rising", "falling", "peak last"])
def test_ties_and_orders(kind, V):
    """The lowest index wins a tie; logits in an order that raises the threshold at every tile."""
    i = torch.arange(V, device="cuda", dtype=torch.float32)
    x = {"constant": torch.zeros(V, device="cuda"), "two values": (i % 7 == 3).float(), "rising": i * (20.0 / V),
         "falling": -i * (20.0 / V), "peak last": (i == V - 1) * 50.0}[kind]
    for dtype in (torch.float32, torch.bfloat16):
        rows = torch.stack([x, x.flip(0)]).to(dtype)
        check(rows, torch.tensor([0, V - 1], device="cuda"), 20)
        check(rows, torch.tensor([0, V - 1], device="cuda"), 64)


def test_signed_zeros_tie():
    x = torch.tensor([[-1.0, -0.0, 0.0, -0.0, -2.0]], device="cuda")
    assert check(x, torch.tensor([1], device="cuda"), 4).top_ids.tolist() == [[1, 2, 3, 0]]


@pytest.mark.parametrize("V", [40, 5000, 40000])
def test_masked_words(V):
    """-inf logits have probability 0, also where a row has fewer others than are asked for, or one."""
    x, t = logits(4, V, torch.float32)
    x[0, 3:] = -INF
    x[1, :V - 2] = -INF
    x[2, ::2] = -INF
    x[3, :] = -INF
    x[3, V // 2] = 1.0
    check(x, torch.tensor([0, 5, 2, V // 2], device="cuda"), 9)


@pytest.mark.parametrize("V", [40, 5000])
def test_rows_without_a_distribution(V):
    """+inf, NaN, and nothing but -inf: NaN, and the rows beside them are untouched."""
    x, t = logits(5, V, torch.float16)
    x[0, 7] = INF
    x[1, 7] = NAN
    x[2, :] = -INF
    x[3, 5], x[3, 9] = INF, NAN
    r = check(x, t, 3)
    assert r.logprob[:4].isnan().all() and r.logprob[4].isfinite()
    assert r.top_ids[3, :2].tolist() == [9, 5] and r.top_ids[1, 0] == 7


def test_tokens_outside_the_vocabulary():
    x, _ = logits(4, 100, torch.float32)
    r = check(x, torch.tensor([-1, 100, 2 ** 40, 99], device="cuda"), 2)
    assert r.logprob.isnan().tolist() == [True, True, True, False]


def test_large_logits():
    """Far from 0: the maximum is taken out before any product is rounded."""
    x, t = logits(3, 5000, torch.float32)
    check(x + torch.tensor([[3e4], [-3e4], [100.0]], device="cuda"), t, 5)


LOWEST = {t: torch.finfo(t).min for t in (torch.float16, torch.bfloat16, torch.float32)}


def masked_rows(V, dtype, mask):
    """Rows whose masked words hold `mask`: the first 1024, the last, all but ten, a tail, all, the first half
    beside others at the type's lowest value; the given token masked in every second of two passes."""
    x, t = logits(6, V, dtype, seed=V)
    i = torch.arange(V, device="cuda")
    hidden = torch.stack([i < 1024, i == V - 1, i % (V // 10) != 3, i >= 3 * V // 4, i >= 0, i < V // 2])
    x = torch.where(hidden, torch.tensor(mask, device="cuda", dtype=dtype), x)
    x[5, V // 2:V // 2 + V // 4] = LOWEST[dtype]
    return x, t, hidden


@pytest.mark.parametrize("dtype,mask", [(torch.float32, -1e5), (torch.float32, -1e9), (torch.float32, -1e10),
                                        (torch.float32, -2e10), (torch.float32, -1e20), (torch.float32, -1e30),
                                        (torch.float32, -2.3e38), (torch.float32, LOWEST[torch.float32]),
                                        (torch.bfloat16, -1e10), (torch.bfloat16, -1e30),
                                        (torch.bfloat16, LOWEST[torch.bfloat16]), (torch.float16, LOWEST[torch.float16])])
@pytest.mark.parametrize("V,repeat", [(1025, 1), (5000, 1), (9000, 200), (40000, 1)])
def test_words_masked_with_finite_numbers(V, repeat, dtype, mask):
    """A finite mask is a logit like any other: alone in a wave's first tile, in the tile of the last logits,
    in whole slices, and in a row that holds nothing else (uniform, not NaN)."""
    x, t, hidden = masked_rows(V, dtype, mask)
    x, t = x.repeat(repeat, 1), t.repeat(repeat)
    for top in (0, 5, 64):
        r = check(x, t, top)
        assert r.logprob.isfinite().all() and r.entropy.isfinite().all()
        assert abs(r.entropy[4].item() - math.log(V)) <= 2.0 ** -20 * V / 64
    check(x, torch.where(hidden.repeat(repeat, 1).any(-1), hidden.repeat(repeat, 1).int().argmax(-1), 0), 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e5, 1e6, 1e7, 1e10, 1e20, 1e37])
def test_logits_of_any_size(size, dtype):
    """Finite logits of both signs, spread as widely as they are large; shifted to either side of 0."""
    x, t = logits(3, 9000, torch.float32, seed=3)
    wide = (x * size).to(dtype)
    check(wide, t, 20)
    check(wide[:, :1024].contiguous(), t % 1024, 20)
    if size <= 1e10:  # where a step of the type is left between them
        check((x + torch.tensor([[size], [-size], [2 * size]], device="cuda")).to(dtype), t, 20)


@pytest.mark.parametrize("V", [40, 5000, 40000])
def test_infinities_beside_finite_masks(V):
    """+inf and NaN give NaN, -inf beside a finite mask counts as less than it."""
    x, t = logits(4, V, torch.float32)
    x[:, V // 2:] = LOWEST[torch.float32]
    x[0, 3], x[1, 3], x[2, :V // 2] = INF, NAN, -INF
    x[3] = -INF
    x[3, V - 1] = LOWEST[torch.float32]
    r = check(x, torch.tensor([3, 3, V - 1, V - 1], device="cuda"), 5)
    assert r.logprob[:2].isnan().all() and r.logprob[2].isfinite() and r.logprob[3] == 0


def test_far_logits_of_every_slice():
    """Finite masks in slices that hold whole tiles, the last logits alone, and both; numbers on either side of
    what a near maximum is, one above the other by little."""
    for V in (4097, 12289, 16383, 16385, 20487):
        x = torch.full((4, V), -3e7, device="cuda")
        x[0, V - 1], x[1, 5], x[2, 1030] = -16777210.0, -16777217.0, 16777218.0
        x[0, 3], x[0, 9], x[1, 2000], x[2, V - 1] = -16777218.0, -16777212.0, -16777218.0, 16777216.0
        x[3] += 2 * (torch.arange(V, device="cuda") % 5)
        for top in (0, 6):
            check(x, torch.tensor([3, 2000, V - 1, 4], device="cuda"), top)


def test_leading_shapes_and_empty():
    x, t = logits(12, 300, torch.float16)
    r = token_logprobs(x.view(3, 4, 300), t.view(3, 4), 2)
    s = token_logprobs(x, t, 2)
    assert r.logprob.shape == (3, 4) and r.top_ids.shape == (3, 4, 2)
    for a, b in zip(r, s):
        assert torch.equal(a.reshape(-1), b.reshape(-1))
    one = token_logprobs(x[0], t[0], 2)
    assert one.logprob.shape == () and torch.equal(one.top_ids, s.top_ids[0])
    assert token_logprobs(x[:0], t[:0], 2).top_ids.shape == (0, 2)
    turned = token_logprobs(x.t().contiguous().t(), t, 2)
    assert torch.equal(turned.top_ids, s.top_ids) and torch.equal(turned.logprob, s.logprob)


def test_graphs_and_streams():
    """Two captured calls replayed in turn on two streams, with eager calls between, at new logits."""
    cases = []
    for seed, (rows, V) in enumerate([(1, 50000), (3, 20011)]):
        x, t = logits(rows, V, torch.float16, seed)
        token_logprobs(x, t, 5)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = token_logprobs(x, t, 5)
        cases.append((graph, r, x, t))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(4):
        want = []
        for graph, r, x, t in cases:
            x.copy_(x.roll(101, 1))
            want.append(token_logprobs(x, t, 5))
        torch.cuda.synchronize()
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                c[0].replay()
        torch.cuda.synchronize()
        for w, c in zip(want, cases):
            assert all(torch.equal(a, b) for a, b in zip(w, c[1])), step


def test_refusals():
    x, t = logits(2, 10, torch.float16)
    for bad in (dict(top=11), dict(top=65), dict(top=-1)):
        with pytest.raises((ValueError, RuntimeError)):
            token_logprobs(x, t, **bad)
    with pytest.raises(ValueError, match="int64"):
        token_logprobs(x, t.int())
    with pytest.raises(ValueError, match="shape"):
        token_logprobs(x, t[:1])
    with pytest.raises(ValueError, match="dtype"):
        token_logprobs(x.double(), t)
    with pytest.raises(RuntimeError, match="GPU"):
        token_logprobs(x.cpu(), t.cpu())
