"""The decoder with drafted tokens on a block-scaled cache (spec_decoder.py) on
the B200: the operators together, as a serving step makes the calls.

Tolerance: both paths compared here (a whole prompt at once; the same tokens in
steps) are within 2e-2 of their logits' maximum of the exact model on their
cache, the decoder tests' bound, so they are within 4e-2 of one another."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(cuda, batch=2, max_ctx=400, **kw):
    import decoder
    import spec_decoder
    cfg = decoder.DecoderConfig(layers=2, hidden=512, heads=4, kv_heads=2, head_dim=128, inter=1024, vocab=1000)
    return spec_decoder.SpeculativeDecoder(cfg, cuda, batch, max_ctx, seed=3, **kw)


def _prompts(cuda, lens, seed=1):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return [torch.randint(0, 1000, (n,), device=cuda, generator=g) for n in lens]


def _prompt_logits(m, prompts):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=m.dev)  # noqa: E731
    lens = [len(p) for p in prompts]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return m._logits(m.forward(torch.cat(prompts), i32(cu), i32(lens), max(lens))), cu


@pytest.mark.parametrize("window,sinks", [(0, 0), (60, 4)])
@pytest.mark.parametrize("K", [0, 3, 40])
def test_steps_match_the_whole_prompt(cuda, window, sinks, K):
    """The logits of drafts verified after a prompt equal those of one pass over
    prompt and drafts."""
    prompts = _prompts(cuda, [150, 33])
    a, b = _model(cuda, window=window, sinks=sinks), _model(cuda, window=window, sinks=sinks)
    heat = torch.zeros(2, device=cuda)
    first = a.prompt(prompts, heat).clone()
    drafts = torch.randint(0, 1000, (2, K), device=cuda)
    seen = {}
    keep = a._logits
    a._logits = lambda x: seen.setdefault("logits", keep(x))
    a.verify_step(drafts, heat)
    whole, cu = _prompt_logits(b, [torch.cat([p, t[None], d]) for p, t, d in zip(prompts, first, drafts)])
    for s in range(2):
        got = seen["logits"].view(2, K + 1, -1)[s]
        want = whole[cu[s + 1] - K - 1:cu[s + 1]]
        assert ((got - want).abs().max() / want.abs().max()).item() < 4e-2


def test_greedy_drafts_are_taken_as_the_model_would(cuda):
    """With temperature 0, the model's own greedy tokens are all accepted, a wrong
    one stops the row where it stands, and decoding goes on from there."""
    heat = torch.zeros(2, device=cuda)
    prompts = _prompts(cuda, [70, 40], seed=5)
    m = _model(cuda)
    m.prompt(prompts, heat)
    start = m.tokens.clone(), m.positions.clone()
    plain = []
    for _ in range(6):  # no drafts: one token a step
        out, accepted = m.verify_step(torch.empty(2, 0, dtype=torch.int64, device=cuda), heat)
        assert accepted.tolist() == [0, 0]
        plain.append(out[:, 0])
    plain = torch.stack(plain, 1)
    m.tokens.copy_(start[0])
    m.positions.copy_(start[1])
    drafts = plain[:, :4].clone()
    drafts[1, 2] = (drafts[1, 2] + 1) % 1000
    out, accepted = m.verify_step(drafts, heat)
    # the tokens before a draft that differs by a near tie between the two passes
    assert accepted[1] <= 2
    for s in range(2):
        n = int(accepted[s])
        assert out[s, :n].tolist() == drafts[s, :n].tolist()
        assert out[s, n + 1:].tolist() == [-1] * (4 - n)
    assert m.positions.tolist() == (start[1] + accepted + 1).tolist()
    assert m.tokens.tolist() == [out[s, int(accepted[s])].item() for s in range(2)]


def test_step_in_a_graph(cuda):
    """A captured step replays on the advanced state as the eager one does."""
    heat = torch.zeros(2, device=cuda)
    prompts = _prompts(cuda, [30, 50], seed=7)
    a, b = _model(cuda), _model(cuda)
    for m in (a, b):
        m.prompt(prompts, heat)
    drafts = torch.randint(0, 1000, (2, 2), device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up on a copy of the state, then restore it
        keep = a.tokens.clone(), a.positions.clone()
        a.verify_step(drafts, heat)
        a.tokens.copy_(keep[0])
        a.positions.copy_(keep[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, accepted = a.verify_step(drafts, heat)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        graph.replay()
        want, taken = b.verify_step(drafts, heat)
        assert torch.equal(out, want) and torch.equal(accepted, taken)
        assert torch.equal(a.positions, b.positions) and torch.equal(a.tokens, b.tokens)


def test_refuses_tensor_parallel_and_bad_prompts(cuda):
    with pytest.raises(ValueError):
        _model(cuda, tp=2)
    m = _model(cuda, max_ctx=64)
    for lens in ([10], [10, 64], [0, 3]):
        with pytest.raises(ValueError):
            m.prompt(_prompts(cuda, lens))
