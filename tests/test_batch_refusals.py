"""Host-side argument checks of the batched serving entry points (no GPU: a refused call
touches no pointer)."""
import ctypes as C

import pytest

import b200infer.capi as L

P = 1 << 20  # a 16-byte aligned address that no refused call follows
OK, INVALID, UNSUPPORTED = 0, 1, 2


def packed(**kw):
    a = dict(q=P, qt=256, qh=64, k=P, kt=128, kh=64, v=P, vt=128, vh=64, out=P, ot=256, oh=64, cu_q=P, cu_k=P, n=2, tq=10,
             tk=10, D=64, Hq=4, Hkv=2, scale=0.0, dtype=0, ws=P, wsb=1 << 40, status=None, stream=None)
    a.update(kw)
    return L.lib().b200_flash_attn_packed(*a.values())


def pool(**kw):
    a = dict(k=P, v=P, n_blocks=4, block_tokens=16, block_stride=16 * 128, tok_stride=128, head_stride=64, n_head_kv=2,
             head_dim=64, dtype=0)
    a.update(kw)
    return L._KVPool(*a.values())


def append(p=None, **kw):
    a = dict(k=P, kt=128, kh=64, v=P, vt=128, vh=64, cu=P, lens=P, n=2, t=10, pool=C.byref(p or pool()), table=P, stride=4,
             blocks=4, status=None, stream=None)
    a.update(kw)
    return L.lib().b200_paged_kv_append(*a.values())


def decode(p=None, **kw):
    a = dict(q=P, qs=256, qh=64, out=P, os=256, oh=64, pool=C.byref(p or pool()), table=P, stride=4, blocks=4, lens=P, n=2,
             Hq=4, scale=0.0, ws=P, wsb=1 << 40, status=None, stream=None)
    a.update(kw)
    return L.lib().b200_flash_attn_paged_batch(*a.values())


def sample(**kw):
    a = dict(x=P, stride=100, n=2, vocab=100, dtype=0, u=P, t=P, k=None, p=None, m=None, out=P, status=None, stream=None)
    a.update(kw)
    return L.lib().b200_sample(*a.values())


@pytest.mark.parametrize("kw", [dict(q=None), dict(k=None), dict(out=None), dict(cu_q=None), dict(cu_k=None), dict(n=-1),
                                dict(tq=-1), dict(D=0), dict(Hq=3), dict(Hkv=0), dict(dtype=3), dict(dtype=-1)])
def test_packed_invalid(kw):
    assert packed(**kw) == INVALID


@pytest.mark.parametrize("kw", [dict(D=32), dict(D=256), dict(q=P + 4), dict(kt=130), dict(vh=2), dict(out=P + 8), dict(ot=1),
                                dict(tq=2 ** 31), dict(tk=2 ** 31), dict(dtype=1, qh=4)])
def test_packed_unsupported(kw):
    assert packed(**kw) == UNSUPPORTED


def test_packed_workspace():
    need = L.lib().b200_flash_attn_packed_workspace_bytes(2, 10, 10, 64, 4, 2, 0)
    if need:
        assert packed(ws=None, wsb=0) == INVALID and packed(wsb=need - 1) == INVALID and packed(ws=P + 4) == INVALID
    assert packed(n=0) == OK and packed(tq=0) == OK


BAD_POOLS = [(dict(k=None), INVALID), (dict(n_blocks=0), INVALID), (dict(block_tokens=0), INVALID), (dict(dtype=7), INVALID),
             (dict(head_dim=-1), INVALID), (dict(k=P + 8), UNSUPPORTED), (dict(tok_stride=130), UNSUPPORTED),
             (dict(head_stride=66), UNSUPPORTED), (dict(block_stride=2), UNSUPPORTED), (dict(n_blocks=2 ** 31), UNSUPPORTED),
             (dict(head_dim=66), UNSUPPORTED)]


@pytest.mark.parametrize("kw,code", BAD_POOLS)
def test_bad_pools(kw, code):
    assert append(pool(**kw)) == code and decode(pool(**kw)) == code


@pytest.mark.parametrize("kw,code", [(dict(k=None), INVALID), (dict(lens=None), INVALID), (dict(table=None), INVALID),
                                     (dict(n=-1), INVALID), (dict(n=0), INVALID), (dict(t=-1), INVALID),
                                     (dict(blocks=0), INVALID), (dict(stride=3), INVALID), (dict(pool=None), INVALID),
                                     (dict(k=P + 4), UNSUPPORTED), (dict(vt=129), UNSUPPORTED), (dict(t=0, n=0), OK)])
def test_append(kw, code):
    assert append(**kw) == code


@pytest.mark.parametrize("kw,code", [(dict(q=None), INVALID), (dict(Hq=3), INVALID), (dict(Hq=0), INVALID),
                                     (dict(lens=None), INVALID), (dict(stride=1), INVALID), (dict(n=200, ws=None), INVALID),
                                     (dict(n=200, wsb=16), INVALID), (dict(n=200, ws=P + 4), INVALID),
                                     (dict(q=P + 4), UNSUPPORTED),
                                     (dict(oh=65), UNSUPPORTED), (dict(n=0), OK)])
def test_decode(kw, code):
    assert decode(**kw) == code


def test_decode_head_dim():
    assert decode(pool(head_dim=96, head_stride=96, tok_stride=192)) == UNSUPPORTED


@pytest.mark.parametrize("kw,code", [(dict(x=None), INVALID), (dict(u=None), INVALID), (dict(t=None), INVALID),
                                     (dict(out=None), INVALID), (dict(n=-1), INVALID), (dict(vocab=0), INVALID),
                                     (dict(dtype=9), INVALID), (dict(vocab=2 ** 21 + 1), UNSUPPORTED), (dict(n=0), OK)])
def test_sample(kw, code):
    assert sample(**kw) == code
