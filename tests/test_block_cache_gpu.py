"""The block-scaled fp8 cache on the B200 (append, attention) against plain
64-bit definitions on the CPU.

Tolerances, from the operators' arithmetic:
* append: codes and scales are exact (one rounding of the same fp32 value; the
  scales are powers of two), q within one bf16 rounding of the fp32 rotation,
  which the oracle repeats: equal.
* attention: bf16 output (half a step is at most 2^-8 of a value), probabilities
  with at least 8 significant bits (2^-8 each, of either sign), q exact to 2^-13
  of a row's maximum.  An output is a convex combination of the values, so its
  error is at most 2^-8 |out| + 2^-8 max |v| over the keys it sees; of the second
  term a quarter is allowed, the roundings of many keys being of either sign.
  The 2-norm over a whole output is held to 4e-3 (bf16 alone: 1.7e-3).
"""
import math

import pytest
import torch

import block_cache_oracle as BO

pytestmark = pytest.mark.gpu

D = 128


def _case(seed, lens, new, hq=8, hkv=2, bs=16, extra=3, spread=3, table_pad=0, layout="nhd"):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // bs) for n in lens]
    nb = sum(need) + extra
    perm = torch.randperm(nb, generator=g).tolist()
    width = max(need + [1]) + table_pad
    table, at = [], 0
    for n in need:
        table.append(perm[at:at + n] + [nb + 7] * (width - n))  # past a sequence: ids outside the cache
        at += n
    codes = lambda: (torch.randn(nb, bs, hkv, D, generator=g) * 64).clamp(-448, 448).to(torch.float8_e4m3fn)  # noqa: E731
    scale = lambda: torch.exp2(torch.randint(-6 - spread, -6 + spread + 1, (nb, hkv), generator=g).float())  # noqa: E731
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return {"k": codes(), "v": codes(), "ks": scale(), "vs": scale(), "table": table, "cu": cu, "lens": list(lens),
            "q": torch.randn(cu[-1], hq, D, generator=g).to(torch.bfloat16), "hq": hq, "hkv": hkv, "bs": bs, "g": g,
            "layout": layout}


def _cache(t, cuda, layout):
    """The cache on the GPU, [NB, BS, HKV, D] by shape; "hnd" stores heads before
    slots, "kv" K and V of a block side by side."""
    if layout == "hnd":
        return t.view(torch.uint8).permute(0, 2, 1, 3).contiguous().to(cuda).permute(0, 2, 1, 3).view(torch.float8_e4m3fn)
    if layout == "kv":
        nb, bs, hkv, d = t.shape
        both = torch.zeros(nb, 2, bs, hkv, d, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
        both.view(torch.uint8)[:, 1] = t.view(torch.uint8).to(cuda)
        return both[:, 1]
    return t.view(torch.uint8).to(cuda).view(torch.float8_e4m3fn)


def _attend(c, cuda, window=0, sinks=0, workspace=None, q=None, out=None, sm_scale=D ** -0.5, **over):
    import block_cache
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    q = c["q"].to(cuda) if q is None else q
    out = torch.full_like(q, 7.0) if out is None else out
    a = dict(max_qlen=max(1, max(b - a for a, b in zip(c["cu"], c["cu"][1:]))), max_seq_len=max(max(c["lens"]), 1),
             window=window, sinks=sinks, workspace=workspace)
    a.update(over)
    return block_cache.attention(q, _cache(c["k"], cuda, c["layout"]), _cache(c["v"], cuda, c["layout"]),
                                 c["ks"].to(cuda), c["vs"].to(cuda), out, i32(c["cu"]), i32(c["lens"]),
                                 i32(c["table"]), sm_scale, **a)


def _check(got, c, window=0, sinks=0, sm_scale=D ** -0.5):
    ref = BO.attention(c["q"], c["k"].double(), c["v"].double(), c["ks"], c["vs"], c["cu"], c["lens"], c["table"],
                       sm_scale, window, sinks)
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    for s, total in enumerate(c["lens"]):
        rows = slice(c["cu"][s], c["cu"][s + 1])
        if rows.start == rows.stop:
            continue
        blocks = c["table"][s][:-(-total // c["bs"])] if total > 0 else []
        top = (c["v"][blocks].double().abs() * c["vs"][blocks][:, None, :, None]).max().item() if blocks else 0.0
        err = (got[rows] - ref[rows]).abs()
        assert (err <= 2 ** -8 * ref[rows].abs() + 2 ** -10 * top).all(), (s, err.max().item(), top)
    norm = ref.norm().item()
    if norm:
        assert (got - ref).norm().item() / norm < 4e-3


LENGTHS = [
    ([1], [1]), ([16], [1]), ([17], [1]), ([127, 128, 129], [1, 1, 1]), ([300, 1, 77], [1, 1, 1]),
    ([700, 33, 5, 256], [3, 1, 5, 2]), ([64, 100], [0, 4]), ([0, 40], [0, 1]), ([1000], [8]), ([260, 511], [4, 7]),
]


@pytest.mark.parametrize("lens,new", LENGTHS)
@pytest.mark.parametrize("bs", [16, 64])
def test_attention_short_queries(cuda, lens, new, bs):
    c = _case(len(lens) + sum(lens), lens, new, bs=bs)
    _check(_attend(c, cuda), c)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 4), (4, 2), (8, 1), (6, 2), (16, 1), (5, 1), (14, 2), (32, 8)])
@pytest.mark.parametrize("new", [1, 5])
def test_attention_head_layouts(cuda, hq, hkv, new):
    c = _case(hq * 10 + hkv, [203, 64, 130], [new] * 3, hq=hq, hkv=hkv, bs=32)
    _check(_attend(c, cuda), c)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (100, 4), (129, 0), (130, 130), (5000, 3), (64, 300)])
@pytest.mark.parametrize("new", [1, 6])
def test_attention_window_and_sinks(cuda, window, sinks, new):
    c = _case(window + sinks, [900, 131, 7, 400], [new] * 4, bs=16)
    _check(_attend(c, cuda, window, sinks), c, window, sinks)


@pytest.mark.parametrize("lens,new,hq,hkv,bs", [
    ([200], [200], 4, 1, 16), ([33, 129, 64], [33, 129, 64], 8, 2, 16), ([300, 450], [70, 129], 4, 2, 64),
    ([257], [40], 16, 2, 128), ([500, 90, 1], [100, 1, 1], 8, 8, 32), ([150, 80], [61, 3], 5, 1, 16),
    ([128, 300], [128, 257], 3, 1, 32), ([700], [65], 16, 1, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3), (140, 0)])
def test_attention_prompts(cuda, lens, new, hq, hkv, bs, window, sinks):
    c = _case(sum(lens), lens, new, hq=hq, hkv=hkv, bs=bs)
    _check(_attend(c, cuda, window, sinks), c, window, sinks)


@pytest.mark.parametrize("layout", ["hnd", "kv"])
@pytest.mark.parametrize("new", [2, 80])
def test_attention_cache_strides(cuda, layout, new):
    c = _case(5, [220, 100], [new, 1], layout=layout)
    _check(_attend(c, cuda), c)


@pytest.mark.parametrize("new", [1, 90])
def test_attention_q_and_out_strides(cuda, new):
    """q as the columns of a projection, out as a slice of a wider buffer."""
    c = _case(6, [222], [new])
    wide = torch.zeros(c["cu"][-1], (8 + 4) * D, dtype=torch.bfloat16, device=cuda)
    wide[:, :8 * D] = c["q"].to(cuda).view(-1, 8 * D)
    buf = torch.full((c["cu"][-1], 10, D), 3.0, dtype=torch.bfloat16, device=cuda)
    _check(_attend(c, cuda, q=wide[:, :8 * D].unflatten(1, (8, D)), out=buf[:, 1:9]), c)
    assert (buf[:, 0] == 3).all() and (buf[:, 9] == 3).all()


@pytest.mark.parametrize("new", [1, 70])
def test_attention_stale_slots_hold_nan(cuda, new):
    """Slots past a sequence, blocks of nobody and, under a window, the slots
    before it hold NaN codes: none reaches the output."""
    c = _case(8, [200, 90], [new, 1], bs=32)
    k, v = c["k"].view(torch.uint8), c["v"].view(torch.uint8)
    used = set()
    for s, total in enumerate(c["lens"]):
        for page in range(-(-total // 32)):
            used.add(c["table"][s][page])
            k[c["table"][s][page], max(0, total - page * 32):] = 0x7F
            v[c["table"][s][page], max(0, total - page * 32):] = 0xFF
    for b in set(range(k.shape[0])) - used:
        k[b] = v[b] = 0x7F
        c["ks"][b] = c["vs"][b] = math.nan
    got = _attend(c, cuda)
    for s, total in enumerate(c["lens"]):  # the oracle takes no NaN
        blk = c["table"][s][(total - 1) // 32]
        k[blk, (total - 1) % 32 + 1:] = v[blk, (total - 1) % 32 + 1:] = 0
    _check(got, c)
    first = c["table"][0][0]
    low = c["lens"][0] - new - 100 + 1  # keys below it are outside every query's window
    if low > 0:
        k[first, :min(low, 32)] = v[first, :min(low, 32)] = 0x7F
        got = _attend(c, cuda, window=100)
        k[first, :min(low, 32)] = v[first, :min(low, 32)] = 0
        _check(got, c, 100)


@pytest.mark.parametrize("new", [1, 3, 100])
def test_attention_scales_far_apart(cuda, new):
    """Block scales from 2^-30 to 2^10, a block of zero scale, and keys of a tiny
    block scale that carry the whole softmax: the output keeps its precision."""
    c = _case(9, [200, 170], [new, new], spread=0)
    c["ks"] = torch.full_like(c["ks"], 2.0 ** -6)
    c["vs"] = torch.exp2(torch.randint(-30, 11, c["vs"].shape, generator=c["g"]).float())
    c["vs"][c["table"][0][1]] = 0
    _check(_attend(c, cuda), c)
    # one block's keys win by a wide margin and its values are the smallest
    c["vs"] = torch.full_like(c["vs"], 4.0)
    b = c["table"][1][2]
    c["vs"][b] = 2.0 ** -22
    c["q"][c["cu"][1]:] = c["q"][c["cu"][1]:, :1]  # one direction for every head of the sequence
    for h in range(c["hkv"]):
        c["k"][b, :, h] = (c["q"][c["cu"][1], 0].float().sign() * 448).to(torch.float8_e4m3fn)
    got = _attend(c, cuda)
    ref = BO.attention(c["q"], c["k"].double(), c["v"].double(), c["ks"], c["vs"], c["cu"], c["lens"], c["table"],
                       D ** -0.5)
    row = c["cu"][1]
    assert (got[row].double().cpu() - ref[row]).norm() / ref[row].norm() < 4e-3


def test_attention_scores_far_apart(cuda):
    """Large scores (a one-hot softmax) and all-equal ones."""
    c = _case(10, [300], [4])
    c["ks"] *= 2 ** 6
    _check(_attend(c, cuda), c)
    c["q"].zero_()
    _check(_attend(c, cuda), c)


@pytest.mark.parametrize("new", [1, 4, 60])
def test_attention_queries_that_see_nothing(cuda, new):
    """A sequence shorter than its queries: those before its first token see no
    key and give zeros; an empty sequence gives zeros throughout."""
    c = _case(11, [40, max(new - 2, 0), 0], [1, new, new])
    got = _attend(c, cuda)
    _check(got, c)
    assert (got[c["cu"][2]:] == 0).all()
    assert (got[c["cu"][1]:c["cu"][1] + min(2, new)] == 0).all()


def test_attention_many_splits_and_reuse(cuda):
    """One workspace for calls of other sizes; the same bytes every time."""
    import block_cache
    ws = block_cache.Workspace(cuda, 16, 8)
    big = _case(12, [5000, 3, 1], [2, 1, 1], hq=4, hkv=1)
    small = _case(13, [40] * 16, [1] * 16, hq=8, hkv=8, bs=128)
    first = _attend(big, cuda, workspace=ws)
    _check(first, big)
    _check(_attend(small, cuda, workspace=ws), small)
    assert torch.equal(first, _attend(big, cuda, workspace=ws))
    assert torch.equal(first, _attend(big, cuda))


def test_attention_length_bound_is_a_bound(cuda):
    """max_qlen and max_seq_len larger than the batch's change nothing in the mathematics."""
    c = _case(14, [300, 20], [2, 1])
    _check(_attend(c, cuda, max_qlen=50, max_seq_len=10000), c)
    _check(_attend(c, cuda, max_seq_len=0), c)


def test_attention_offsets_past_32_bits(cuda):
    """Blocks beyond 4 GB of cache."""
    import block_cache
    nb, bs, hkv = 16500, 128, 16
    k = torch.zeros(nb, bs, hkv, D, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    assert k.numel() > 2 ** 32
    c = _case(15, [200], [3], hq=16, hkv=hkv, bs=bs)
    blocks = [nb - 1, nb - 3]
    ks = torch.ones(nb, hkv, device=cuda)
    vs = torch.ones(nb, hkv, device=cuda)
    v = torch.zeros_like(k)
    for i, b in enumerate(blocks):
        src = c["table"][0][i]
        k.view(torch.uint8)[b] = c["k"][src].view(torch.uint8).to(cuda)
        v.view(torch.uint8)[b] = c["v"][src].view(torch.uint8).to(cuda)
        ks[b], vs[b] = c["ks"][src].to(cuda), c["vs"][src].to(cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    q = c["q"].to(cuda)
    got = block_cache.attention(q, k, v, ks, vs, torch.empty_like(q), i32([0, 3]), i32([200]), i32([blocks]),
                                D ** -0.5, max_qlen=3)
    _check(got, c)


def test_attention_graph_and_stream(cuda):
    """Captured on a side stream; replays follow the lengths and the cache."""
    import block_cache
    c = _case(16, [200, 90], [1, 1])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    k, v = _cache(c["k"], cuda, "nhd"), _cache(c["v"], cuda, "nhd")
    ks, vs, cu, lens, bt = c["ks"].to(cuda), c["vs"].to(cuda), i32(c["cu"]), i32(c["lens"]), i32(c["table"])
    q = c["q"].to(cuda)
    out, ws = torch.zeros_like(q), block_cache.Workspace(cuda, 2, 2)
    call = lambda: block_cache.attention(q, k, v, ks, vs, out, cu, lens, bt, D ** -0.5, max_qlen=1, max_seq_len=256,  # noqa: E731
                                         workspace=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
    torch.cuda.current_stream().wait_stream(side)
    for new_lens in ([200, 90], [17, 64], [1, 2]):
        c["lens"] = new_lens
        lens.copy_(i32(new_lens))
        out.fill_(5)
        graph.replay()
        _check(out, c)


# ---- append ------------------------------------------------------------------------------------------------
def _append_case(seed, lens, new, hq=8, hkv=2, bs=16, size=1.0):
    c = _case(seed, lens, new, hq, hkv, bs)
    c["qkv"] = (torch.randn(c["cu"][-1], (hq + 2 * hkv) * D, generator=c["g"]) * size).to(torch.bfloat16)
    ang = torch.arange(max(max(lens), 1)).double()[:, None] * (1e4 ** (-torch.arange(0, D, 2).double() / D))[None]
    c["rope"] = torch.cat([ang.cos(), ang.sin()], 1).float()
    return c


def _append(c, cuda, in_place=False):
    import block_cache
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    k, v = _cache(c["k"], cuda, c["layout"]), _cache(c["v"], cuda, c["layout"])
    ks, vs, qkv = c["ks"].to(cuda), c["vs"].to(cuda), c["qkv"].to(cuda)
    q = None if in_place else torch.empty(c["cu"][-1], c["hq"], D, dtype=torch.bfloat16, device=cuda)
    got = block_cache.append(qkv, c["rope"].to(cuda), k, v, ks, vs, i32(c["cu"]), i32(c["lens"]), i32(c["table"]), q)
    return got, k, v, ks, vs, qkv


def _check_append(c, got):
    q, k, v, ks, vs, _ = got
    rk, rv, rks, rvs = c["k"].double(), c["v"].double(), c["ks"].double(), c["vs"].double()
    rq = BO.append(c["qkv"], c["rope"], rk, rv, rks, rvs, c["cu"], c["lens"], c["table"], c["hq"])
    assert torch.equal(q.cpu(), rq.to(torch.bfloat16))
    assert torch.equal(ks.cpu().double(), rks) and torch.equal(vs.cpu().double(), rvs)
    assert torch.equal(k.double().cpu(), rk) and torch.equal(v.double().cpu(), rv)


@pytest.mark.parametrize("lens,new", [([1], [1]), ([16], [1]), ([17], [1]), ([33, 5], [2, 5]), ([100, 64], [100, 30]),
                                      ([50, 20, 300], [0, 3, 129]), ([128, 129, 130], [1, 2, 3])])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
def test_append_exact(cuda, lens, new, bs):
    c = _append_case(sum(lens) + bs, lens, new, bs=bs)
    _check_append(c, _append(c, cuda))


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (8, 1), (6, 2), (16, 1), (32, 8)])
def test_append_head_layouts(cuda, hq, hkv):
    c = _append_case(hq + hkv, [40, 9], [25, 1], hq, hkv)
    _check_append(c, _append(c, cuda))


@pytest.mark.parametrize("size", [0.0, 1e-30, 1e-3, 448.0, 1e6, 1e30])
def test_append_sizes_of_values(cuda, size):
    """Zeros, values below the smallest scale, and far above the block's old one."""
    c = _append_case(3, [40, 21], [25, 3], size=size)
    _check_append(c, _append(c, cuda))


def test_append_scale_never_shrinks_within_a_block_and_restarts_with_it(cuda):
    import block_cache  # noqa: F401
    c = _append_case(4, [20], [4], size=1e-3)
    blk = c["table"][0][1]
    c["ks"][blk], c["vs"][blk] = 0.75, 1.0  # not a power of two: an older writer's
    # the block's first new token is at its start: the old scale is void
    got = _append(c, cuda)
    _check_append(c, got)
    assert (got[3][blk].cpu() < 1e-3).all()
    c = _append_case(4, [22], [4], size=1e-3)
    c["ks"][blk], c["vs"][blk] = 1.0, 1.0
    got = _append(c, cuda)
    _check_append(c, got)
    assert (got[3][blk].cpu() == 1).all()


def test_append_in_place_and_strided_cache(cuda):
    c = _append_case(5, [40, 70], [3, 20])
    c["layout"] = "kv"
    got = _append(c, cuda, in_place=True)
    _check_append(c, got)
    assert torch.equal(got[5][:, :8 * D].reshape(-1, 8, D), got[0])        # rotated where it stood
    assert torch.equal(got[5][:, 8 * D:].cpu(), c["qkv"][:, 8 * D:])       # k and v as they were


def test_append_not_finite(cuda):
    """An infinity saturates and leaves the scale to the finite values; NaN stays NaN."""
    c = _append_case(6, [20], [20])
    c["qkv"][3, (8 + 2) * D + 5] = math.inf      # v of head 0
    c["qkv"][4, (8 + 2) * D + 6] = math.nan
    _, k, v, ks, vs, _ = _append(c, cuda)
    fine = c["qkv"][:16, (8 + 2) * D:(8 + 3) * D].float()
    top = fine[torch.isfinite(fine)].abs().max().item()
    blk = c["table"][0][0]
    assert vs[blk, 0].item() == BO.power_of_two_scale(top)
    assert v[blk, 3, 0, 5].item() == 448 and math.isnan(v[blk, 4, 0, 6].item())


def test_append_then_attention_on_another_stream(cuda):
    """The two calls one after the other on a side stream, as a step makes them."""
    import block_cache
    c = _append_case(7, [130, 50], [5, 2])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q, k, v, ks, vs, _ = _append(c, cuda)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
        out = block_cache.attention(q, k, v, ks, vs, torch.empty_like(q), i32(c["cu"]), i32(c["lens"]),
                                    i32(c["table"]), D ** -0.5, max_qlen=5)
    side.synchronize()
    c.update(q=q.cpu(), k=k.cpu(), v=v.cpu(), ks=ks.cpu(), vs=vs.cpu())
    _check(out, c)


def test_append_skips_what_has_no_block(cuda, b200):
    """A position past the table and a block id outside the cache are skipped, q
    is rotated all the same, and the device status says so."""
    c = _append_case(8, [40, 20], [8, 4])
    c["table"] = [row[:2] for row in c["table"]]   # tokens 32.. of sequence 0 have no column
    c["table"][1][1] = 999
    got = _append(c, cuda)
    _check_append(c, got)
    torch.cuda.synchronize()
    assert b200.device_status() == 0x105
    b200.reset_device_status()


def test_refusals(cuda):
    import block_cache
    from _b200kv import B200KVError
    c = _append_case(9, [20], [2])
    dev = {n: _cache(c[n], cuda, "nhd") for n in ("k", "v")}
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    base = dict(q=torch.zeros(2, 8, D, dtype=torch.bfloat16, device=cuda), k=dev["k"], v=dev["v"], ks=c["ks"].to(cuda),
                vs=c["vs"].to(cuda), out=torch.zeros(2, 8, D, dtype=torch.bfloat16, device=cuda), cu=i32([0, 2]),
                lens=i32([20]), bt=i32(c["table"]), sm=1.0, max_qlen=2)

    def attend(**o):
        a = {**base, **o}
        kw = {n: a[n] for n in ("max_qlen", "window", "sinks", "workspace", "max_seq_len") if n in a}
        return block_cache.attention(a["q"], a["k"], a["v"], a["ks"], a["vs"], a["out"], a["cu"], a["lens"], a["bt"],
                                     a["sm"], **kw)

    attend()
    for bad in (dict(q=base["q"].half()), dict(k=base["k"].view(torch.uint8)), dict(ks=base["ks"].double()),
                dict(bt=base["bt"].long()), dict(cu=base["cu"].long())):
        with pytest.raises(TypeError):
            attend(**bad)
    for bad in (dict(ks=base["ks"][:, :1]), dict(cu=i32([0, 1, 2])), dict(out=base["out"][:1]),
                dict(q=base["q"].transpose(1, 2)), dict(workspace=block_cache.Workspace(cuda, 1, 1))):
        with pytest.raises(ValueError):
            attend(**bad)
    for bad in (dict(window=-1), dict(sinks=-1), dict(max_qlen=0), dict(q=base["q"][:, :7], out=base["out"][:, :7])):
        with pytest.raises(B200KVError):
            attend(**bad)
    wide = torch.zeros(2, 34, D, dtype=torch.bfloat16, device=cuda)   # 17 query heads a kv head
    with pytest.raises(B200KVError):
        attend(q=wide, out=wide.clone())
    odd = torch.zeros(4, 24, 2, D, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    with pytest.raises(B200KVError):
        attend(k=odd, v=odd, ks=torch.ones(4, 2, device=cuda), vs=torch.ones(4, 2, device=cuda))

    rope, qkv = c["rope"].to(cuda), c["qkv"].to(cuda)

    def put(**o):
        a = {**base, "qkv": qkv, "rope": rope, "q_out": None, **o}
        return block_cache.append(a["qkv"], a["rope"], a["k"], a["v"], a["ks"], a["vs"], a["cu"], a["lens"], a["bt"],
                                  a["q_out"])

    for bad in (dict(qkv=qkv.float()), dict(rope=rope.double()), dict(q_out=torch.zeros(2, 8, D, device=cuda))):
        with pytest.raises(TypeError):
            put(**bad)
    for bad in (dict(qkv=qkv[:, :-1]), dict(qkv=qkv[:, :4 * D]), dict(rope=rope[:, :64]),
                dict(q_out=base["q"][:1])):
        with pytest.raises(ValueError):
            put(**bad)
