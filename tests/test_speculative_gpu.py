"""Draft verification on the B200 against a plain 64-bit definition on the CPU.

Outputs are whole numbers.  The inputs are drawn with room around every decision:
a draw whose acceptance or race is closer than 1e-4 relative (fp32 probabilities
are good to about 1e-6) is drawn again, so the answers have to be equal."""
import math

import pytest
import torch

import block_cache_oracle as BO

pytestmark = pytest.mark.gpu


def _margin_ok(c):
    vocab = c["logits"].shape[1]
    for s in range(len(c["cu"]) - 1):
        heat = 1.0 if c["temperature"] is None else float(c["temperature"][s])
        for r in range(c["cu"][s], c["cu"][s + 1]):
            last = r == c["cu"][s + 1] - 1
            p = BO.probabilities(c["logits"][r], heat)
            q = torch.zeros(vocab, dtype=torch.float64)
            if not last:
                d = int(c["tokens"][r + 1])
                q = c["draft"][r].double() if c["draft"] is not None else q.index_fill(0, torch.tensor([d]), 1.0)
                if heat > 0 and abs(float(c["uniforms"][r]) * q[d] - p[d]) < 1e-4 * p[d]:
                    return False
            if heat > 0 and vocab > 1:
                for w in ((p - q).clamp_min(0), p):
                    top = (w / c["noise"][s].double()).topk(2).values
                    if top[0] > 0 and top[0] - top[1] < 1e-3 * top[0]:
                        return False
    return True


def _case(seed, counts, vocab, probs=True, temperature=True, half=False, greedy=()):
    g = torch.Generator().manual_seed(seed)
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    while True:
        rows = cu[-1]
        logits = torch.randn(rows, vocab, generator=g) * 3
        draft = torch.softmax(logits + torch.randn(rows, vocab, generator=g), 1)
        if half:
            logits = logits.to(torch.bfloat16)
        tokens = torch.randint(0, vocab, (rows,), generator=g)
        if rows > 1:
            tokens[1:] = torch.multinomial(draft, 1, generator=g)[:-1, 0]
        heat = 0.5 + torch.rand(len(counts), generator=g) if temperature else None
        for i in greedy:
            heat[i] = 0
        c = {"cu": cu, "logits": logits, "draft": draft if probs else None, "tokens": tokens, "temperature": heat,
             "uniforms": torch.rand(rows, generator=g),
             "noise": torch.empty(len(counts), vocab).exponential_(generator=g).clamp_min(1e-20)}
        if _margin_ok(c):
            return c


def _run(c, cuda, **over):
    import speculative
    a = {**c, **over}
    to = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    return speculative.verify(to(a["logits"]), to(a["tokens"]), torch.tensor(a["cu"], dtype=torch.int32, device=cuda),
                              to(a["uniforms"]), to(a["noise"]), to(a["temperature"]), to(a["draft"]))


def _check(c, got):
    out, accepted = BO.verify(c["logits"], c["tokens"], c["cu"], c["uniforms"], c["noise"], c["temperature"], c["draft"])
    assert torch.equal(got[1].cpu(), accepted), (got[1].cpu(), accepted)
    assert torch.equal(got[0].cpu(), out)


@pytest.mark.parametrize("counts", [[1], [2], [5], [1, 4, 8, 2], [17, 3], [9, 9]])
@pytest.mark.parametrize("vocab", [1, 2, 7, 100, 1000, 4099])
def test_verify(cuda, counts, vocab):
    c = _case(len(counts) * vocab, counts, vocab)
    _check(c, _run(c, cuda))


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("temperature", [True, False])
@pytest.mark.parametrize("half", [True, False])
def test_verify_forms(cuda, probs, temperature, half):
    c = _case(3, [4, 1, 6], 777, probs, temperature, half)
    _check(c, _run(c, cuda))


@pytest.mark.parametrize("half", [True, False])
def test_verify_greedy_and_ties(cuda, half):
    c = _case(4, [4, 3, 5], 333, greedy=(0, 2), half=half)
    c["logits"][0, 50:60] = 40.0          # ties: the lowest index
    c["logits"][1, [7, 300]] = 40.0
    c["tokens"][1] = 50                   # taken
    c["tokens"][2] = 300                  # not taken: 7 is emitted
    got = _run(c, cuda)
    _check(c, got)
    assert got[0][:3].tolist() == [50, 7, -1] and got[1][0].item() == 1


def test_verify_takes_all_and_none(cuda):
    c = _case(5, [6, 6], 500)
    c["uniforms"][:6] = 0.0
    c["draft"][6:] = 0
    c["draft"][6:, 3] = 1
    c["tokens"][7] = 3
    c["logits"][6, 3] = -math.inf         # the draft is impossible under the target
    got = _run(c, cuda)
    _check(c, got)
    assert got[1].tolist() == [5, 0] and got[0][7:].tolist() == [-1] * 5


def test_verify_equal_distributions(cuda):
    """p == q: every draft is taken below u = 1; a rejection cannot find a residual
    and falls back to p."""
    c = _case(6, [3], 64, temperature=False)
    c["logits"] = torch.zeros(3, 64)
    c["draft"] = torch.full((3, 64), 1 / 64)
    c["uniforms"][:] = 0.5
    _check(c, _run(c, cuda))
    c["uniforms"][0] = 1.0                # not below 1: the edge the random numbers exclude
    _check(c, _run(c, cuda))


def test_verify_masked_logits(cuda):
    """Rows with -inf, NaN and +inf; a row of -inf takes nothing and emits token 0."""
    c = _case(7, [3, 3, 2, 2], 129, probs=False)
    c["logits"][0, ::2] = -math.inf
    c["logits"][3, 5:] = math.nan
    c["logits"][6, 17] = math.inf
    c["tokens"][7] = 17
    c["logits"][8] = -math.inf
    got = _run(c, cuda)
    _check(c, got)
    assert got[0][6].item() == 17 and got[0][8].item() == 0 and got[1][3].item() == 0


def test_verify_drafts_outside_the_vocabulary(cuda):
    c = _case(8, [3, 3], 50, probs=False)
    c["tokens"][1], c["tokens"][4] = -1, 50
    got = _run(c, cuda)
    _check(c, got)
    assert got[1].tolist() == [0, 0]


def test_verify_strides_and_buffers(cuda):
    import speculative
    c = _case(9, [4, 2], 300)
    wide = torch.full((6, 400), 50.0, device=cuda)
    wide[:, 3:303] = c["logits"].to(cuda)  # rows start off 16 bytes
    noise = torch.full((2, 333), 1e-20, device=cuda)
    noise[:, 1:301] = c["noise"].to(cuda)
    draft = torch.ones(6, 301, device=cuda)
    draft[:, 1:] = c["draft"].to(cuda)
    out = torch.zeros(6, dtype=torch.int64, device=cuda)
    num = torch.zeros(2, dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = speculative.verify(wide[:, 3:303], c["tokens"].to(cuda), torch.tensor(c["cu"], dtype=torch.int32, device=cuda),
                                 c["uniforms"].to(cuda), noise[:, 1:301], c["temperature"].to(cuda), draft[:, 1:], out, num)
    side.synchronize()
    assert got[0] is out and got[1] is num
    _check(c, got)


def test_verify_large_vocabulary_and_graph(cuda):
    import speculative
    c = _case(10, [5, 1, 3], 128256)
    _check(c, _run(c, cuda))
    a = [c["logits"].to(cuda), c["tokens"].to(cuda), torch.tensor(c["cu"], dtype=torch.int32, device=cuda),
         c["uniforms"].to(cuda), c["noise"].to(cuda), c["temperature"].to(cuda), c["draft"].to(cuda)]
    buf = (torch.zeros(9, dtype=torch.int64, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        speculative.verify(*a, *buf)
    for u in (0.0, 0.999):
        c["uniforms"][:] = u
        a[3].copy_(c["uniforms"])
        graph.replay()
        _check(c, buf)


def test_verify_emits_the_targets_distribution(cuda):
    """20000 sequences of one draft over 8 tokens: the emitted first tokens are
    distributed as the target (each frequency within 5 standard deviations)."""
    import speculative
    n, vocab = 20000, 8
    g = torch.Generator(device=cuda).manual_seed(11)
    p = torch.softmax(torch.randn(vocab, device=cuda, generator=g), 0)
    q = torch.softmax(torch.randn(vocab, device=cuda, generator=g), 0)
    logits = p.log().expand(2 * n, vocab).contiguous()
    tokens = torch.multinomial(q.expand(2 * n, vocab), 1, generator=g)[:, 0]
    out, _ = speculative.verify(logits, tokens, torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=cuda),
                                torch.rand(2 * n, device=cuda, generator=g),
                                torch.empty(n, vocab, device=cuda).exponential_(generator=g), None,
                                q.expand(2 * n, vocab).contiguous())
    freq = torch.bincount(out[::2], minlength=vocab).double() / n
    sd = (p.double() * (1 - p.double()) / n).sqrt()
    assert ((freq - p.double()).abs() < 5 * sd).all()


def test_verify_refusals(cuda):
    from _b200kv import B200KVError
    c = _case(12, [2], 20)
    _run(c, cuda)
    for bad in (dict(logits=c["logits"].half()), dict(tokens=c["tokens"].int()), dict(noise=c["noise"].double()),
                dict(draft=c["draft"].double())):
        with pytest.raises(TypeError):
            _run(c, cuda, **bad)
    for bad in (dict(tokens=c["tokens"][:1]), dict(noise=c["noise"][:, :5]), dict(draft=c["draft"][:1]),
                dict(cu=[0, 1, 2]), dict(uniforms=c["uniforms"][:1])):
        with pytest.raises(ValueError):
            _run(c, cuda, **bad)
    with pytest.raises(ValueError):
        _run(c, cuda, logits=c["logits"].t().contiguous().t())
    assert B200KVError is not None
