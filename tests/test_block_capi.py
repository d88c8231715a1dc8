"""Refusals of the block-scaled cache's and the draft verification's entry points
that need no GPU: the C functions return their documented status before they
touch a device, the Python ones raise."""
import pytest
import torch

A = 0x10000  # never dereferenced: every call below fails validation first
INVALID, UNSUPPORTED, MISALIGNED, WORKSPACE, NO_DEVICE = 1, 2, 3, 4, 6
NEED_GPU_FREE = pytest.mark.skipif(torch.cuda.is_available(), reason="fake pointers are only safe without a GPU")


def _cache(b200, **over):
    f = dict(k=A, v=A, ks=A, vs=A, bt=A, sk0=16 * 8 * 128, sk1=8 * 128, sk2=128, sv0=16 * 8 * 128, sv1=8 * 128,
             sv2=128, ks0=8, ks1=1, vs0=8, vs1=1, bts=4, nb=100, bs=16, hkv=8, d=128, blocks=4, seqs=2)
    assert set(over) <= set(f)
    f.update(over)
    return b200.BLOCK_CACHE.pack(*f.values())


CACHE_FAULTS = [(dict(k=0), INVALID), (dict(v=0), INVALID), (dict(ks=0), INVALID), (dict(vs=0), INVALID),
                (dict(bt=0), INVALID), (dict(nb=0), INVALID), (dict(hkv=0), INVALID), (dict(blocks=0), INVALID),
                (dict(seqs=0), INVALID), (dict(bts=3), INVALID), (dict(d=64), UNSUPPORTED), (dict(bs=48), UNSUPPORTED),
                (dict(bs=256), UNSUPPORTED), (dict(k=A + 8), MISALIGNED), (dict(v=A + 1), MISALIGNED),
                (dict(sk0=8), MISALIGNED), (dict(sv2=136), MISALIGNED)]


def _append(b200, cache=None, **over):
    f = dict(qkv=A, st=48 * 128, cs=A, pos=64, q=A, q0=32 * 128, q1=128, cu=A, lens=A, T=4, hq=32)
    assert set(over) <= set(f)
    f.update(over)
    return b200.lib.b200kv_block_append(_cache(b200, **(cache or {})), *f.values(), None)


def _attention(b200, cache=None, **over):
    need = b200.lib.b200kv_block_attn_workspace_bytes(2, 8)
    f = dict(q=A, out=A, cu=A, lens=A, ws=A, wsb=need, q0=32 * 128, q1=128, o0=32 * 128, o1=128, sm=0.1, T=4, mq=2,
             msl=64, hq=32, window=0, sinks=0, reserved=0)
    assert set(over) <= set(f)
    f.update(over)
    return b200.lib.b200kv_block_attn(_cache(b200, **(cache or {})), b200.BLOCK_ATTN_ARGS.pack(*f.values()), None)


def _verify(b200, **over):
    f = dict(lg=A, ld=1000, half=0, tok=A, cu=A, u=A, noise=A, nld=1000, temp=None, draft=None, dld=0, out=A, acc=A,
             seqs=2, rows=6, vocab=1000, ws=A, wsb=b200.lib.b200kv_spec_verify_workspace_bytes(2, 6, 1000), st=None)
    assert set(over) <= set(f)
    f.update(over)
    return b200.lib.b200kv_spec_verify(*f.values())


@pytest.mark.parametrize("fault,status", CACHE_FAULTS)
def test_cache_refusals(b200, fault, status):
    assert _append(b200, fault) == status
    assert _attention(b200, fault) == status


@pytest.mark.parametrize("fault,status", [
    (dict(qkv=None), INVALID), (dict(cs=None), INVALID), (dict(q=None), INVALID), (dict(cu=None), INVALID),
    (dict(lens=None), INVALID), (dict(pos=0), INVALID), (dict(T=-1), INVALID), (dict(hq=0), INVALID),
    (dict(hq=30), INVALID), (dict(qkv=A + 8), MISALIGNED), (dict(q=A + 2), MISALIGNED), (dict(cs=A + 4), MISALIGNED),
    (dict(st=48 * 128 + 4), MISALIGNED), (dict(q0=12), MISALIGNED), (dict(q1=129), MISALIGNED)])
def test_append_refusals(b200, fault, status):
    assert _append(b200, **fault) == status


@pytest.mark.parametrize("fault,status", [
    (dict(q=0), INVALID), (dict(out=0), INVALID), (dict(cu=0), INVALID), (dict(lens=0), INVALID),
    (dict(T=-1), INVALID), (dict(mq=0), INVALID), (dict(msl=-1), INVALID), (dict(hq=12), INVALID),
    (dict(window=-1), INVALID), (dict(sinks=-1), INVALID), (dict(hq=8 * 17), UNSUPPORTED), (dict(q=A + 8), MISALIGNED),
    (dict(out=A + 2), MISALIGNED), (dict(q0=12), MISALIGNED), (dict(o1=100), MISALIGNED), (dict(ws=0), WORKSPACE),
    (dict(wsb=1024), WORKSPACE), (dict(ws=A + 128), MISALIGNED)])
def test_attention_refusals(b200, fault, status):
    assert _attention(b200, **fault) == status


@pytest.mark.parametrize("fault,status", [
    (dict(lg=None), INVALID), (dict(tok=None), INVALID), (dict(cu=None), INVALID), (dict(u=None), INVALID),
    (dict(noise=None), INVALID), (dict(out=None), INVALID), (dict(acc=None), INVALID), (dict(seqs=-1), INVALID),
    (dict(rows=-1), INVALID), (dict(vocab=0), INVALID), (dict(ld=999), INVALID), (dict(nld=999), INVALID),
    (dict(draft=A, dld=999), INVALID), (dict(ws=None), WORKSPACE), (dict(wsb=16), WORKSPACE),
    (dict(ws=A + 8), MISALIGNED), (dict(rows=1 << 30, wsb=1 << 60), UNSUPPORTED)])
def test_verify_refusals(b200, fault, status):
    assert _verify(b200, **fault) == status


@NEED_GPU_FREE
def test_valid_calls_report_the_missing_device(b200):
    assert _append(b200) == NO_DEVICE
    assert _attention(b200) == NO_DEVICE
    assert _verify(b200) == NO_DEVICE


def test_workspace_sizes(b200):
    lib = b200.lib
    assert lib.b200kv_block_attn_workspace_bytes(0, 8) == 0
    assert lib.b200kv_block_attn_workspace_bytes(2, 0) == 0
    assert lib.b200kv_block_attn_workspace_bytes(1, 1) > 0
    assert lib.b200kv_spec_verify_workspace_bytes(-1, 4, 10) == 0
    assert lib.b200kv_spec_verify_workspace_bytes(1, 4, 0) == 0
    assert lib.b200kv_spec_verify_workspace_bytes(2, 6, 128256) > lib.b200kv_spec_verify_workspace_bytes(1, 1, 128256)


def _cpu_cache():
    fp8 = lambda: torch.zeros(4, 16, 2, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    return fp8(), fp8(), torch.zeros(4, 2), torch.zeros(4, 2), i32(3), i32(2), i32(2, 2)


def test_python_refuses_tensors_of_the_host(b200):
    import block_cache
    import speculative
    cache = _cpu_cache()
    qkv = torch.zeros(4, 8 * 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        block_cache.append(qkv, torch.zeros(64, 128), *cache)
    q = torch.zeros(4, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        block_cache.attention(q, *cache[:4], torch.empty_like(q), *cache[4:], 0.1, 2)
    with pytest.raises(ValueError, match="GPU"):
        speculative.verify(torch.zeros(4, 100), torch.zeros(4, dtype=torch.int64), torch.zeros(3, dtype=torch.int32),
                           torch.zeros(4), torch.ones(2, 100))


def test_python_refuses_types(b200):
    import block_cache
    import speculative
    kc, vc, ks, vs, cu, lens, bt = _cpu_cache()
    qkv, table = torch.zeros(4, 8 * 128, dtype=torch.bfloat16), torch.zeros(64, 128)
    for args in ((qkv.half(), table, kc, vc, ks, vs, cu, lens, bt), (qkv, table.double(), kc, vc, ks, vs, cu, lens, bt),
                 (qkv, table, kc.float(), vc, ks, vs, cu, lens, bt), (qkv, table, kc, vc, ks.half(), vs, cu, lens, bt),
                 (qkv, table, kc, vc, ks, vs, cu.long(), lens, bt)):
        with pytest.raises(TypeError):
            block_cache.append(*args)
    with pytest.raises(TypeError):
        speculative.verify(torch.zeros(4, 100).half(), torch.zeros(4, dtype=torch.int64),
                           torch.zeros(3, dtype=torch.int32), torch.zeros(4), torch.ones(2, 100))
