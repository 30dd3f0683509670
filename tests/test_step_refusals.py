"""Host-side argument checks of the 8-bit cache, shared-prefix attention and logit adjustment (no GPU: a refused call
touches no pointer)."""
import ctypes as C

import pytest

import b200infer.capi as L

P = 1 << 20  # a 16-byte aligned address that no refused call follows
OK, INVALID, UNSUPPORTED = 0, 1, 2


def pool8(**kw):
    a = dict(k=P, v=P, ks=P + 1, vs=P + 3, n_blocks=4, block_tokens=16, block_stride=16 * 128, tok_stride=128, head_stride=64,
             sb=32, st=1, sh=16, n_head_kv=2, head_dim=64)
    a.update(kw)
    return L._KVPoolQ8(*a.values())


def append(p=None, **kw):
    a = dict(k=P, kt=128, kh=64, v=P, vt=128, vh=64, dtype=0, cu=P, lens=P, n=2, t=10, pool=C.byref(p or pool8()), table=P, stride=4,
             blocks=4, status=None, stream=None)
    a.update(kw)
    return L.lib().b200_paged_kv_append_q8(*a.values())


def read(p=None, **kw):
    a = dict(pool=C.byref(p or pool8()), table=P, stride=4, blocks=4, cu=P, lens=P, n=2, t=10, k=P, kt=128, kh=64, v=P, vt=128, vh=64,
             dtype=0, status=None, stream=None)
    a.update(kw)
    return L.lib().b200_paged_kv_read_q8(*a.values())


def decode(p=None, **kw):
    a = dict(q=P, qs=256, qh=64, out=P, os=256, oh=64, dtype=0, pool=C.byref(p or pool8()), table=P, stride=4, blocks=4, lens=P, n=2,
             Hq=4, scale=0.0, ws=P, wsb=1 << 40, status=None, stream=None)
    a.update(kw)
    return L.lib().b200_flash_attn_paged_batch_q8(*a.values())


def pool(**kw):
    a = dict(k=P, v=P, n_blocks=4, block_tokens=16, block_stride=16 * 128, tok_stride=128, head_stride=64, n_head_kv=2,
             head_dim=64, dtype=0)
    a.update(kw)
    return L._KVPool(*a.values())


def shared(p=None, **kw):
    a = dict(q=P, qs=256, qh=64, out=P, os=256, oh=64, pool=C.byref(p or pool()), ptable=P, pstride=4, pblocks=4, plens=P, cu=P, groups=2,
             table=P, stride=4, blocks=4, lens=P, n=2, Hq=4, scale=0.0, ws=P, wsb=1 << 40, status=None, stream=None)
    a.update(kw)
    return L.lib().b200_flash_attn_paged_shared(*a.values())


def adjust(**kw):
    a = dict(x=P, stride=100, out=P, ostride=100, n=2, vocab=100, dtype=0, tokens=P, T=5, cu=P, prompt=None, r=P, f=P, p=P, ids=P,
             values=P, m=5, cub=P, mask=P, ms=4, status=None, stream=None)
    a.update(kw)
    return L.lib().b200_adjust_logits(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), INVALID), (dict(ks=None), INVALID), (dict(vs=None), INVALID), (dict(n_blocks=0), INVALID),
    (dict(block_tokens=0), INVALID), (dict(n_head_kv=0), INVALID), (dict(head_dim=-64), INVALID), (dict(head_dim=32), UNSUPPORTED),
    (dict(head_dim=256), UNSUPPORTED), (dict(k=P + 8), UNSUPPORTED), (dict(v=P + 1), UNSUPPORTED), (dict(tok_stride=120), UNSUPPORTED),
    (dict(head_stride=72), UNSUPPORTED), (dict(block_stride=8), UNSUPPORTED), (dict(n_blocks=2 ** 31), UNSUPPORTED),
    (dict(block_tokens=2 ** 31), UNSUPPORTED), (dict(n_head_kv=2 ** 40), UNSUPPORTED)])
def test_bad_pools(kw, code):
    assert append(pool8(**kw)) == code and read(pool8(**kw)) == code and decode(pool8(**kw)) == code


@pytest.mark.parametrize("call", [append, read])
@pytest.mark.parametrize("kw,code", [(dict(k=None), INVALID), (dict(v=None), INVALID), (dict(lens=None), INVALID),
                                     (dict(cu=None), INVALID), (dict(table=None), INVALID), (dict(n=-1), INVALID),
                                     (dict(n=0), INVALID), (dict(t=-1), INVALID), (dict(blocks=0), INVALID),
                                     (dict(stride=3), INVALID), (dict(pool=None), INVALID), (dict(dtype=3), INVALID),
                                     (dict(dtype=-1), INVALID), (dict(k=P + 4), UNSUPPORTED), (dict(vt=129), UNSUPPORTED),
                                     (dict(dtype=2, kh=4), UNSUPPORTED), (dict(t=2 ** 31), UNSUPPORTED), (dict(n=2 ** 31), UNSUPPORTED),
                                     (dict(t=0, n=0), OK)])
def test_append_and_read(call, kw, code):
    assert call(**kw) == code


@pytest.mark.parametrize("kw,code", [(dict(q=None), INVALID), (dict(out=None), INVALID), (dict(Hq=3), INVALID), (dict(Hq=0), INVALID),
                                     (dict(lens=None), INVALID), (dict(table=None), INVALID), (dict(stride=1), INVALID),
                                     (dict(blocks=0), INVALID), (dict(n=-1), INVALID), (dict(dtype=5), INVALID),
                                     (dict(q=P + 4), UNSUPPORTED), (dict(oh=65), UNSUPPORTED), (dict(dtype=1, qh=4), UNSUPPORTED),
                                     (dict(Hq=2 ** 17), UNSUPPORTED), (dict(n=2 ** 31), UNSUPPORTED), (dict(n=0), OK)])
def test_decode(kw, code):
    assert decode(**kw) == code


def test_decode_workspace():
    need = L.lib().b200_flash_attn_paged_batch_q8_workspace_bytes(200, 64, 64, 4, 2)
    if need:
        assert decode(n=200, ws=None) == INVALID and decode(n=200, wsb=need - 1) == INVALID and decode(n=200, ws=P + 4) == INVALID


@pytest.mark.parametrize("kw,code", [(dict(q=None), INVALID), (dict(Hq=3), INVALID), (dict(Hq=0), INVALID), (dict(lens=None), INVALID),
                                     (dict(ptable=None), INVALID), (dict(plens=None), INVALID), (dict(cu=None), INVALID),
                                     (dict(pblocks=0), INVALID), (dict(pstride=3), INVALID), (dict(groups=-1), INVALID),
                                     (dict(stride=1), INVALID), (dict(n=-1), INVALID), (dict(pool=None), INVALID),
                                     (dict(q=P + 4), UNSUPPORTED), (dict(oh=65), UNSUPPORTED), (dict(n=2 ** 31), UNSUPPORTED),
                                     (dict(groups=2 ** 31), UNSUPPORTED), (dict(Hq=2 ** 17), UNSUPPORTED), (dict(n=0), OK)])
def test_shared(kw, code):
    assert shared(**kw) == code


def test_shared_pool_and_workspace():
    assert shared(pool(head_dim=96, head_stride=96, tok_stride=192)) == UNSUPPORTED
    assert shared(pool(dtype=7)) == INVALID and shared(pool(k=P + 8)) == UNSUPPORTED
    need = L.lib().b200_flash_attn_paged_shared_workspace_bytes(2, 64, 2, 64, 64, 4, 2, 0)
    if need:
        assert shared(ws=None) == INVALID and shared(wsb=need - 1) == INVALID and shared(ws=P + 4) == INVALID


@pytest.mark.parametrize("kw,code", [(dict(x=None), INVALID), (dict(out=None), INVALID), (dict(n=-1), INVALID), (dict(vocab=0), INVALID),
                                     (dict(dtype=3), INVALID), (dict(stride=-1), INVALID), (dict(ostride=99), INVALID),
                                     (dict(ostride=101), INVALID), (dict(tokens=None), INVALID), (dict(cu=None), INVALID),
                                     (dict(tokens=None, T=0, cu=None), INVALID), (dict(T=-1), INVALID), (dict(ids=None), INVALID),
                                     (dict(values=None), INVALID), (dict(cub=None), INVALID), (dict(m=-1), INVALID), (dict(ms=-1), INVALID),
                                     (dict(vocab=2 ** 21 + 1, stride=2 ** 22, ostride=2 ** 22), UNSUPPORTED), (dict(T=2 ** 31), UNSUPPORTED),
                                     (dict(m=2 ** 31), UNSUPPORTED), (dict(x=P + 2, out=P + 2), UNSUPPORTED),
                                     (dict(x=P + 1, out=P + 1, dtype=2), UNSUPPORTED), (dict(n=2 ** 40), UNSUPPORTED), (dict(n=0), OK)])
def test_adjust(kw, code):
    assert adjust(**kw) == code


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("heads", [(32, 8), (16, 8), (16, 1), (150, 1)])
def test_workspace_for_many_sequences_does_for_fewer(dtype, heads):
    size = L.lib().b200_flash_attn_paged_shared_workspace_bytes
    for keys, groups, prefix in ((1024, 1, 8192), (4096, 4, 1000), (16, 1, 100000)):
        sizes = [size(n, keys, groups, prefix, 128, *heads, dtype) for n in list(range(1, 200)) + [500, 5000]]
        assert sizes == sorted(sizes)
