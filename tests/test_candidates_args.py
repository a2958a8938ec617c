"""What the operators for several candidates of a chunk refuse, checked without a GPU: the entry points answer bad sizes with
a status before anything is read, the Python forms raise ValueError before anything is launched."""

import inspect

import pytest
import torch

from viktor_b200 import _lib, ops

BF = torch.bfloat16
fake = 16  # any non-null, 16-byte-aligned address: nothing is dereferenced


def _good_attend():
    B, H, HK, D, P, S, N, page, M = 4, 8, 2, 64, 2, 40, 6, 16, 3
    return dict(q=torch.zeros(B, H, D, dtype=BF), k_prefix=torch.zeros(P, S, HK, D, dtype=BF),
                v_prefix=torch.zeros(P, S, HK, D, dtype=BF), prefix_lens=torch.zeros(P, dtype=torch.int32),
                group_offsets=torch.zeros(P + 1, dtype=torch.int32), k_pages=torch.zeros(N, page, HK, D, dtype=BF),
                v_pages=torch.zeros(N, page, HK, D, dtype=BF), page_table=torch.zeros(B, M, dtype=torch.int32),
                tail_lens=torch.zeros(B, dtype=torch.int32))


def test_python_forms_need_cuda():
    with pytest.raises(ValueError, match="CUDA"):
        ops.shared_prefix_attention(**_good_attend())
    with pytest.raises(ValueError, match="CUDA"):
        ops.penalize_logits(torch.zeros(2, 7))
    pages = ops.KVPages.empty(1, 4, 16, 2, 2, device="cpu")
    for f in (lambda: ops.pages_extend(pages), lambda: ops.pages_free(pages), lambda: ops.pages_compact(pages),
              lambda: ops.pages_fork(pages, torch.zeros(1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))):
        with pytest.raises(ValueError, match="CUDA"):
            f()


@pytest.mark.parametrize("name,bad", [
    ("q", torch.zeros(4, 8, 64)), ("q", torch.zeros(4, 8, 64, dtype=torch.float16)), ("q", torch.zeros(4, 8, 32, dtype=BF)),
    ("q", torch.zeros(4, 9, 64, dtype=BF)), ("q", torch.zeros(4, 64, 8, dtype=BF).transpose(1, 2)),
    ("q", torch.zeros(1, 8, 64, dtype=BF).expand(4, 8, 64)), ("q", torch.zeros(5, 8, 64, dtype=BF)),
    ("k_prefix", torch.zeros(2, 41, 2, 64, dtype=BF)), ("k_prefix", torch.zeros(2, 40, 2, 128, dtype=BF)[..., ::2]),
    ("k_prefix", torch.zeros(2, 2, 40, 64, dtype=BF).transpose(1, 2)), ("v_prefix", torch.zeros(2, 50, 2, 64, dtype=BF)[:, :40]),
    ("prefix_lens", torch.zeros(3, dtype=torch.int32)), ("prefix_lens", torch.zeros(2, dtype=torch.int64)),
    ("group_offsets", torch.zeros(2, dtype=torch.int32)), ("k_pages", torch.zeros(6, 12, 2, 64, dtype=BF)),
    ("k_pages", torch.zeros(6, 16, 1, 64, dtype=BF)), ("page_table", torch.zeros(3, 3, dtype=torch.int32)),
    ("page_table", torch.zeros(4, 3, dtype=torch.int64)), ("page_table", torch.zeros(1, 3, dtype=torch.int32).expand(4, 3)),
    ("tail_lens", torch.zeros(8, dtype=torch.int32)[::2]), ("scale", 0.0), ("scale", -1.0), ("scale", float("inf")),
    ("scale", float("nan")), ("out", torch.zeros(4, 8, 64)), ("out", torch.zeros(4, 64, 8, dtype=BF).transpose(1, 2)),
    ("workspace", torch.zeros(1, dtype=torch.uint8)),
])
def test_shared_prefix_attention_refuses(name, bad):
    with pytest.raises(ValueError) as e:
        ops.shared_prefix_attention(**{**_good_attend(), name: bad})
    assert "CUDA" not in str(e.value)


def test_shared_prefix_attention_refuses_overlapping_out():
    a = _good_attend()
    big = torch.zeros(8, 8, 64, dtype=BF)
    for q, out in ((big[:4], big[:4]), (big[:4], big[3:7]), (big[::2], big[4:])):
        with pytest.raises(ValueError, match="overlap"):
            ops.shared_prefix_attention(**{**a, "q": q, "out": out})


def test_kv_pages_refuse():
    def make(k=(2, 4, 16, 2, 64), v=None, table=(3, 2), lens=3, refs=4, dtype=BF, ints=torch.int32):
        return ops.KVPages(torch.zeros(k, dtype=dtype), torch.zeros(v or k, dtype=dtype), torch.zeros(table, dtype=ints),
                           torch.zeros(lens, dtype=ints), torch.zeros(refs, dtype=ints))

    make()
    make(dtype=torch.uint8)
    for bad in (dict(k=(2, 4, 12, 2, 64)), dict(k=(2, 4, 16, 2, 64), v=(2, 4, 16, 1, 64)), dict(k=(2, 4, 512, 2, 64)),
                dict(lens=2), dict(refs=3), dict(ints=torch.int64), dict(table=(0, 2)), dict(k=(2, 4, 16, 1, 3)),
                dict(k=(4, 16, 2, 64))):
        with pytest.raises(ValueError):
            make(**bad)
    pages, i32 = make(), torch.int32
    for bad in (lambda: ops.pages_extend(pages, 0), lambda: ops.pages_extend(pages, 33),
                lambda: ops.pages_extend(pages, 1, torch.zeros(2, dtype=torch.int64)),
                lambda: ops.pages_extend(pages, 1, torch.zeros(2, 1, dtype=i32)),
                lambda: ops.pages_fork(pages, torch.zeros(2, dtype=i32), torch.zeros(3, dtype=i32)),
                lambda: ops.pages_fork(pages, None, None), lambda: ops.pages_free(pages, torch.zeros(4, dtype=i32)[::2])):
        with pytest.raises(ValueError) as e:
            bad()
        assert "CUDA" not in str(e.value)


def _good_penal():
    return dict(logits=torch.zeros(3, 40), history=torch.zeros(3, 5, dtype=torch.int64), history_lens=torch.zeros(3, dtype=torch.int32),
                repetition=torch.ones(3), presence=torch.ones(3), frequency=torch.ones(3), bias=torch.zeros(40),
                mask=torch.zeros(2, 2, dtype=torch.int32), mask_index=torch.zeros(3, dtype=torch.int32))


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(3, 40, dtype=torch.float64)), dict(logits=torch.zeros(40)), dict(logits=torch.zeros(40, 3).T),
    dict(logits=torch.zeros(1, 40).expand(3, 40)), dict(history=torch.zeros(2, 5, dtype=torch.int64)),
    dict(history=torch.zeros(3, 5, dtype=torch.int32)), dict(history_lens=None), dict(history_lens=torch.zeros(3, dtype=torch.int64)),
    dict(history=None), dict(repetition=torch.ones(3, dtype=torch.float64)), dict(presence=torch.ones(4)), dict(frequency=torch.ones(1)),
    dict(bias=torch.zeros(41)), dict(bias=torch.zeros(40, dtype=BF)), dict(bias=torch.zeros(2, 40)),
    dict(mask=torch.zeros(2, 1, dtype=torch.int32)), dict(mask=torch.zeros(2, 2, dtype=torch.int64)), dict(mask=None),
    dict(mask_index=None), dict(mask_index=torch.zeros(2, dtype=torch.int32)), dict(out=torch.zeros(3, 41)),
    dict(out=torch.zeros(3, 40, dtype=BF)), dict(out=torch.zeros(1, 40).expand(3, 40)),
])
def test_penalize_logits_refuses(change):
    with pytest.raises(ValueError) as e:
        ops.penalize_logits(**{**_good_penal(), **change})
    assert "CUDA" not in str(e.value)


def test_penalize_logits_refuses_overlapping_out():
    a = {k: v for k, v in _good_penal().items() if k not in ("logits",)}
    wide = torch.zeros(4, 100)
    for x, out in ((wide[:3, :40], wide[:3, 20:60]), (wide[:3, :40], wide[1:, :40]), (wide[:3, 60:], wide[:3, 99:].as_strided((3, 40), (100, 1)))):
        with pytest.raises(ValueError, match="overlap"):
            ops.penalize_logits(x, out=out, **a)
    for x, out in ((wide[:3, :40], wide[:3, 50:90]), (wide[:3, 50:90], wide[:3, :40]), (wide[:3, :40], wide[:3, :40])):
        with pytest.raises(ValueError, match="CUDA"):
            ops.penalize_logits(x, out=out, **a)


def test_entry_points_refuse():
    lib = _lib.load()
    ARG, NO = _lib.VK_ERR_ARG, _lib.VK_ERR_UNSUPPORTED
    good = dict(q=fake, stride_q=512, dtype=0, k=fake, v=fake, lens=fake, off=fake, P=2, S=40, kb=40 * 128, ks=128, kp=fake, vp=fake,
                n_pages=6, page=16, pp=16 * 128, table=fake, max_pages=3, st=3, tails=fake, out=1 << 20, lse=None, B=4, H=8, HK=2,
                D=64, scale=0.125, ws=fake, ws_bytes=lib.vk_shared_attention_workspace_bytes(4, 8, 2, 64, 2, 40, 48), stream=None)
    assert good["ws_bytes"] > 0 and lib.vk_shared_attention_workspace_bytes(0, 8, 2, 64, 2, 40, 48) == 0
    assert lib.vk_shared_attention(*{**good, "B": 0}.values()) == _lib.VK_OK
    for change in (dict(q=None), dict(q=8), dict(k=None), dict(v=24), dict(lens=None), dict(off=None), dict(table=None), dict(tails=None),
                   dict(out=None), dict(ws=None), dict(ws_bytes=good["ws_bytes"] - 1), dict(B=-1), dict(P=0), dict(S=0), dict(H=7),
                   dict(HK=0), dict(page=24), dict(page=512), dict(page=4), dict(n_pages=0), dict(max_pages=-1), dict(st=2),
                   dict(stride_q=504), dict(stride_q=516), dict(ks=64), dict(ks=132), dict(kb=128), dict(pp=128), dict(scale=0.0),
                   dict(scale=float("nan")), dict(S=2 ** 31 - 20, kb=2 ** 40), dict(B=2 ** 30)):
        assert lib.vk_shared_attention(*{**good, **change}.values()) == ARG, change
    for change in (dict(D=96), dict(dtype=2), dict(dtype=-1)):
        assert lib.vk_shared_attention(*{**good, **change}.values()) == NO, change

    n = lib.vk_pages_workspace_bytes(3, 2, 4, 2)
    assert n > 0 and lib.vk_pages_workspace_bytes(3, 0, 4, 2) == 0
    pool = dict(table=fake, lens=fake, refs=fake, rows=3, max_pages=2, n_pages=4, page=16)
    ext = {**pool, "list": fake, "n": 2, "count": 1, "page_out": fake, "slot_out": fake, "ws": fake, "ws_bytes": n, "stream": None}
    fork = {**pool, "src": fake, "dst": fake, "n": 2, "k": fake, "v": fake, "layers": 1, "token_bytes": 256, "ws": fake, "ws_bytes": n,
            "stream": None}
    free = {k: v for k, v in pool.items() if k != "page"} | {"list": fake, "n": 2, "stream": None}
    comp = {k: v for k, v in pool.items() if k != "lens"} | {"k": fake, "v": fake, "layers": 1, "token_bytes": 256, "live": fake,
                                                             "ws": fake, "ws_bytes": n, "stream": None}
    every = [(lib.vk_pages_extend, ext), (lib.vk_pages_fork, fork), (lib.vk_pages_free, free), (lib.vk_pages_compact, comp)]
    for f, a in every:
        for change in (dict(table=None), dict(refs=None), dict(rows=0), dict(max_pages=0), dict(n_pages=0), dict(rows=2 ** 30, max_pages=4)):
            assert f(*{**a, **change}.values()) == ARG, (f, change)
        for change in (dict(lens=None), dict(page=12), dict(ws=None), dict(ws=8), dict(ws_bytes=15), dict(n=-1), dict(list=None),
                       dict(count=0), dict(count=33), dict(page_out=None), dict(src=None), dict(dst=None), dict(k=None), dict(v=8),
                       dict(layers=0), dict(token_bytes=24), dict(live=None)):
            if set(change) <= set(a):
                assert f(*{**a, **change}.values()) == ARG, (f, change)
    for f, a in every[:3]:
        assert f(*{**a, "n": 0}.values()) == _lib.VK_OK

    pen = dict(logits=fake, out=fake, dtype=2, ld=40, ld_out=40, B=3, V=40, history=fake, lens=fake, T=5, ldh=5, rep=fake, pres=fake,
               freq=fake, bias=fake, ldb=0, mask=fake, ldm=2, masks=2, index=fake, stream=None)
    assert lib.vk_penalize_logits(*{**pen, "B": 0}.values()) == _lib.VK_OK
    for change in (dict(logits=None), dict(out=None), dict(ld=39), dict(ld_out=39), dict(B=-1), dict(V=0), dict(lens=None), dict(T=-1),
                   dict(ldh=4), dict(ldb=39), dict(ldm=1), dict(masks=0), dict(index=None)):
        assert lib.vk_penalize_logits(*{**pen, **change}.values()) == ARG, change
    assert lib.vk_penalize_logits(*{**pen, "dtype": 3}.values()) == NO


def test_documented_names():
    for f in ("shared_prefix_attention", "KVPages", "pages_extend", "pages_fork", "pages_free", "pages_compact", "penalize_logits"):
        assert inspect.getdoc(getattr(ops, f))
