"""The operators over cached sequences refuse on the host what they cannot
do: shapes, types, devices, gradients, and the same through the C ABI."""
import ctypes

import pytest
import torch

from afterimage_b200 import _lib
from afterimage_b200.runtime import seq_ops as S

BF = torch.bfloat16


def _i(*v):
    return torch.tensor(v, dtype=torch.int64)


def _prompt(**kw):
    a = dict(q=torch.zeros(6, 4, 16, dtype=BF), k=torch.zeros(6, 2, 16, dtype=BF), v=torch.zeros(6, 2, 16, dtype=BF),
             cu_q=_i(0, 2, 6), scale=1.0)
    a.update(kw)
    return S.prompt_attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("cu_q"), a.pop("scale"), **a)


CACHE = torch.zeros(2, 2, 8, 16, dtype=BF)


@pytest.mark.parametrize("kw,text", [
    ({}, "CUDA"),
    (dict(q=torch.zeros(6, 4, 16)), "bf16"),
    (dict(q=torch.zeros(6, 4, 32, dtype=BF)[..., ::2]), "unit stride"),
    (dict(q=torch.zeros(6, 64, dtype=BF)), "q must be"),
    (dict(q=torch.zeros(6, 4, 16, dtype=BF, requires_grad=True)), "backward"),
    (dict(cu_q=torch.zeros(3, dtype=torch.int32)), "int64"),
    (dict(cu_q=_i(0, 2, 6, 0, 0, 0)[::2]), "contiguous"),
    (dict(k=torch.zeros(6, 2, 8, dtype=BF)), "one shape"),
    (dict(k=torch.zeros(5, 2, 16, dtype=BF), v=torch.zeros(5, 2, 16, dtype=BF)), "cu_k"),
    (dict(k=torch.zeros(6, 3, 16, dtype=BF), v=torch.zeros(6, 3, 16, dtype=BF)), "divide"),
    (dict(k=CACHE, v=CACHE), "len_k"),
    (dict(k=CACHE, v=CACHE, len_k=_i(2, 6), cu_k=_i(0, 2, 6)), "cu_k"),
    (dict(k=CACHE[:1], v=CACHE[:1], len_k=_i(2, 6)), "1 caches"),
    (dict(k=CACHE, v=CACHE, len_k=_i(2)), "len_k"),
    (dict(len_k=_i(2, 6)), "without len_k"),
    (dict(cu_k=_i(0, 6)), "cu_k"),
    (dict(out=torch.zeros(6, 4, 8, dtype=BF)), "q's shape"),
    (dict(out=torch.zeros(1, 4, 16, dtype=BF).expand(6, 4, 16)), "expanded"),
    (dict(q=torch.zeros(6, 4, 264, dtype=BF), k=torch.zeros(6, 2, 264, dtype=BF), v=torch.zeros(6, 2, 264, dtype=BF)),
     "head size"),
    (dict(k=torch.zeros(6, 2, 16, dtype=BF, device="meta")), "meta"),
])
def test_prompt_attention_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _prompt(**kw)


def _tree(**kw):
    a = dict(q=torch.zeros(2, 3, 4, 16, dtype=BF), k_cache=CACHE, v_cache=CACHE, pos=_i(1, 4),
             mask=torch.ones(3, 3, dtype=torch.bool), scale=1.0)
    a.update(kw)
    return S.tree_attention(**a)


@pytest.mark.parametrize("kw,text", [
    ({}, "CUDA"),
    (dict(q=torch.zeros(3, 4, 16, dtype=BF)), "q must be"),
    (dict(k_cache=CACHE.float()), "bf16"),
    (dict(k_cache=CACHE[:1]), "caches must be"),
    (dict(pos=_i(1)), "pos"),
    (dict(pos=torch.zeros(2, dtype=torch.int32)), "pos"),
    (dict(mask=torch.ones(3, 3)), "mask"),
    (dict(mask=torch.ones(2, 3, dtype=torch.bool)), "mask"),
    (dict(mask=torch.ones(3, 3, 3, dtype=torch.bool)), "mask"),
    (dict(mask=torch.ones(3, 9, dtype=torch.bool)), "drafted tokens"),
    (dict(q=torch.zeros(2, 3, 3, 16, dtype=BF)), "divide"),
    (dict(k_cache=CACHE.clone().requires_grad_()), "backward"),
])
def test_tree_attention_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _tree(**kw)


def _rope(**kw):
    a = dict(qkv=torch.zeros(5, 8 * 16, dtype=BF), nh=4, nkv=2, hd=16, cu=_i(0, 2, 5), start=_i(0, 3),
             inv_freq=torch.ones(8), k_cache=CACHE, v_cache=CACHE.clone())
    a.update(kw)
    return S.rope_cache_packed(**a)


@pytest.mark.parametrize("kw,text", [
    ({}, "CUDA"),
    (dict(qkv=torch.zeros(5, 100, dtype=BF)), "qkv must be"),
    (dict(hd=15), "head size"),
    (dict(start=_i(0)), "start"),
    (dict(depth=_i(0, 1)), "depth"),
    (dict(inv_freq=torch.ones(16)), "inv_freq"),
    (dict(inv_freq=torch.ones(8, dtype=torch.float64)), "inv_freq"),
    (dict(q_norm=torch.ones(16, dtype=BF)), "both"),
    (dict(q_norm=torch.ones(8, dtype=BF), k_norm=torch.ones(8, dtype=BF)), "norm weights"),
    (dict(v_cache=CACHE), "the same"),
    (dict(v_cache=CACHE[:, :1]), "caches must be"),
    (dict(k_cache=torch.zeros(1, 2, 8, 16, dtype=BF).expand(2, 2, 8, 16)), "expanded"),
    (dict(out=torch.zeros(5, 4, 8, dtype=BF)), "out"),
])
def test_rope_cache_packed_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        _rope(**kw)


@pytest.mark.parametrize("caches,pos,keep,text", [
    ([CACHE], _i(0, 1), torch.zeros(2, 3, dtype=torch.int64), "CUDA"),
    ([CACHE, CACHE], _i(0, 1), torch.zeros(2, 3, dtype=torch.int64), "twice"),
    ([CACHE, CACHE.float()], _i(0, 1), torch.zeros(2, 3, dtype=torch.int64), "bf16"),
    ([CACHE, CACHE[:, :, :4]], _i(0, 1), torch.zeros(2, 3, dtype=torch.int64), "one shape"),
    ([CACHE], _i(0), torch.zeros(2, 3, dtype=torch.int64), "pos"),
    ([CACHE], _i(0, 1), torch.zeros(3, dtype=torch.int64), "keep"),
    ([CACHE], _i(0, 1), torch.zeros(2, 3, dtype=torch.int32), "keep"),
    ([CACHE], _i(0, 1), torch.zeros(2, 257, dtype=torch.int64), "at most 256"),
    ([torch.zeros(1, 2, 8, 16, dtype=BF).expand(2, 2, 8, 16)], _i(0, 1), torch.zeros(2, 3, dtype=torch.int64),
     "expanded"),
])
def test_keep_cache_rows_refuses(caches, pos, keep, text):
    with pytest.raises(ValueError, match=text):
        S.keep_cache_rows(caches, pos, keep)


def test_keep_cache_rows_of_no_caches_does_nothing():
    S.keep_cache_rows([], _i(0), torch.zeros(1, 1, dtype=torch.int64))


def test_tree_mask():
    mask, depth = S.tree_mask([-1, 0, 0, 1, -1])
    assert depth.tolist() == [0, 1, 1, 2, 0]
    assert mask.tolist() == [[True, False, False, False, False], [True, True, False, False, False],
                             [True, False, True, False, False], [True, True, False, True, False],
                             [False, False, False, False, True]]
    assert S.tree_mask([])[0].shape == (0, 0)
    for bad in ([0], [-1, 1], [-2]):
        with pytest.raises(ValueError, match="parent"):
            S.tree_mask(bad)


def test_attention_descriptor_layout_matches_the_header(tmp_path):
    import pathlib
    import subprocess
    header = pathlib.Path(_lib.__file__).resolve().parent.parent / "include"
    fields = [f for f, _ in _lib.AttnDesc._fields_]
    src = tmp_path / "layout.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"afterimage_b200.h\"\nint main(void){"
                   "printf(\"%zu\\n\", sizeof(aib_attn_desc));"
                   + "".join('printf("%%zu\\n", offsetof(aib_attn_desc, %s));' % f for f in fields) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(header), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.AttnDesc)] + [getattr(_lib.AttnDesc, f).offset for f in fields]


def _desc(**kw):
    d = _lib.AttnDesc(q=0x1000, k=0x2000, v=0x3000, out=0x4000, tokens=4, batch=1, key_rows=8, nh=4, nkv=2, hd=16,
                      scale=1.0, cu_q=0x5000, cu_k=0x5000, pos=0x6000, mask=0x7000, mask_cols=4)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("entry", ["aib_prompt_attention_bf16", "aib_tree_attention_bf16"])
@pytest.mark.parametrize("kw,text", [
    (dict(nh=3), b"shape"), (dict(nkv=0), b"shape"), (dict(hd=257), b"shape"), (dict(tokens=-1), b"shape"),
    (dict(tokens=2 ** 31), b"32 bits"), (dict(scale=float("nan")), b"scale"), (dict(q=None), b"null"),
    (dict(v=None), b"null"), (dict(out=None), b"null"), (dict(sms=-1), b"sms"),
])
def test_attention_c_entries_refuse(entry, kw, text):
    L = _lib.load()
    d = _desc(**kw)
    assert getattr(L, entry)(ctypes.byref(d), None, 0, None, None) == _lib.AIB_EINVAL
    assert text in L.aib_last_error()


def test_attention_c_entries_refuse_what_only_one_takes():
    L = _lib.load()
    assert L.aib_prompt_attention_bf16(None, None, 0, None, None) == _lib.AIB_EINVAL
    assert L.aib_prompt_attention_bf16(ctypes.byref(_desc(cu_q=None)), None, 0, None, None) == _lib.AIB_EINVAL
    assert L.aib_prompt_attention_bf16(ctypes.byref(_desc(cu_k=None)), None, 0, None, None) == _lib.AIB_EINVAL
    assert b"cu_k" in L.aib_last_error()
    assert L.aib_tree_attention_bf16(ctypes.byref(_desc(pos=None)), None, 0, None, None) == _lib.AIB_EINVAL
    assert L.aib_tree_attention_bf16(ctypes.byref(_desc(mask=None)), None, 0, None, None) == _lib.AIB_EINVAL
    assert L.aib_tree_attention_bf16(ctypes.byref(_desc(mask_cols=9)), None, 0, None, None) == _lib.AIB_EINVAL
    assert b"columns" in L.aib_last_error()
    # nothing to do: no CUDA call
    for kw in (dict(tokens=0), dict(batch=0)):
        assert L.aib_prompt_attention_bf16(ctypes.byref(_desc(**kw)), None, 0, None, None) == _lib.AIB_OK
        assert L.aib_tree_attention_bf16(ctypes.byref(_desc(**kw)), None, 0, None, None) == _lib.AIB_OK


def test_cache_c_entries_refuse():
    L = _lib.load()
    st = (ctypes.c_int64 * 3)(256, 128, 16)
    def rope(n=4, hd=16, qn=None, kn=None, q=0x1000):
        return L.aib_rope_cache_packed_bf16(q, 128, n, 1, 4, 2, hd, 0x2000, 0x3000, None, qn, kn, 1e-6, 0x4000, 0x5000,
                                            0x6000, 0x7000, st, st, 8, None)
    assert rope(hd=15) == _lib.AIB_EINVAL
    assert rope(qn=0x100) == _lib.AIB_EINVAL and b"both" in L.aib_last_error()
    assert rope(q=None) == _lib.AIB_EINVAL and b"null" in L.aib_last_error()
    assert rope(n=0) == _lib.AIB_OK
    ptrs = (ctypes.c_void_p * 2)(0x1000, None)
    def keep(count=2, n=3, nkv=2):
        return L.aib_keep_cache_rows_bf16(ptrs, count, 1, nkv, 8, 16, st, 0x2000, 0x3000, n, None)
    assert keep() == _lib.AIB_EINVAL and b"null tensor 1" in L.aib_last_error()
    assert keep(n=257) == _lib.AIB_EINVAL and b"at most 256" in L.aib_last_error()
    assert keep(nkv=0) == _lib.AIB_EINVAL
    assert keep(n=0) == _lib.AIB_OK and keep(count=0) == _lib.AIB_OK


@pytest.mark.parametrize("entry,kw", [
    ("aib_tree_attention_bf16", {}),
    ("aib_prompt_attention_bf16", dict(mask=None, pos=None, mask_cols=0, cu_k=None, len_k=0x8000)),
])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_c_entries_refuse_a_workspace_that_is_null_small_or_not_on_16_bytes(entry, kw, hd):
    """On the host alone: with sms given, the shares join through the workspace (no cluster) on every machine."""
    L = _lib.load()
    d = _desc(hd=hd, key_rows=4096, sms=100, **kw)
    for name in ("q", "k", "v", "out"):
        setattr(d, name + "_token_stride", 4 * hd)
        setattr(d, name + "_head_stride", hd)
    for name in ("k", "v"):
        setattr(d, name + "_token_stride", hd)
        setattr(d, name + "_head_stride", 4096 * hd)
    need = L.aib_attention_workspace_floats(ctypes.byref(d))
    assert need > 0
    call = getattr(L, entry)
    for ptr, floats in ((None, need), (0x10000, need - 1)):
        assert call(ctypes.byref(d), ptr, floats, None, None) == _lib.AIB_EINVAL
        assert b"workspace of" in L.aib_last_error()
    for off in (4, 8, 12):
        assert call(ctypes.byref(d), 0x10000 + off, need, None, None) == _lib.AIB_EINVAL
        assert b"16" in L.aib_last_error()


@pytest.mark.parametrize("batch,tokens", [(1, 4), (8, 100), (3, 400), (16, 33), (40, 41), (2, 1000)])
def test_a_descriptor_with_the_fields_of_both_kinds_gets_a_workspace_for_either(batch, tokens):
    """The prompt entry does not look at the mask, nor the tree entry at cu_q: the size has to do for both. On the host
    alone: an address off 16 bytes is refused, and only after the size was found to do."""
    L = _lib.load()
    hd, rows = 128, 4096

    def desc(**kw):
        d = _desc(hd=hd, key_rows=rows, sms=100, batch=batch, tokens=tokens, cu_k=None, len_k=0x8000)
        d.q_batch_stride = d.out_batch_stride = tokens * 4 * hd
        d.k_batch_stride = d.v_batch_stride = 2 * rows * hd
        for name in ("q", "out"):
            setattr(d, name + "_token_stride", 4 * hd)
            setattr(d, name + "_head_stride", hd)
        for name in ("k", "v"):
            setattr(d, name + "_token_stride", hd)
            setattr(d, name + "_head_stride", rows * hd)
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    def floats(**kw):
        return L.aib_attention_workspace_floats(ctypes.byref(desc(**kw)))

    tree, prompt, both = floats(cu_q=None, len_k=None), floats(mask=None, pos=None), floats()
    assert both == max(tree, prompt)
    for entry, need in (("aib_tree_attention_bf16", tree), ("aib_prompt_attention_bf16", prompt)):
        if need:
            assert getattr(L, entry)(ctypes.byref(desc()), 0x10004, both, None, None) == _lib.AIB_EINVAL
            assert b"16-byte" in L.aib_last_error()


def _grad(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype, requires_grad=True)


@pytest.mark.parametrize("call", [
    lambda: _rope(k_cache=_grad(2, 2, 8, 16)),
    lambda: _rope(v_cache=_grad(2, 2, 8, 16)),
    lambda: _rope(inv_freq=_grad(8, dtype=torch.float32)),
    lambda: _rope(out=_grad(5, 4, 16)),
    lambda: _rope(q_norm=_grad(16), k_norm=torch.ones(16, dtype=BF)),
    lambda: S.keep_cache_rows([CACHE, _grad(2, 2, 8, 16)], _i(0, 1), torch.zeros(2, 3, dtype=torch.int64)),
    lambda: S.keep_cache_rows([_grad(2, 2, 8, 16)], _i(0, 1), torch.zeros(2, 3, dtype=torch.int64)),
    lambda: _prompt(out=_grad(6, 4, 16)),
    lambda: _tree(out=_grad(2, 3, 4, 16)),
], ids=["rope k", "rope v", "rope inv_freq", "rope out", "rope norms", "keep second", "keep first", "prompt out", "tree out"])
def test_tensors_that_need_a_gradient_are_refused(call):
    with pytest.raises(ValueError, match="backward"):
        call()
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # nothing but the device is wrong then
        call()


def test_a_torch_without_cuda_imports_the_operators(tmp_path):
    """CPU ranks use tree_mask; the operators themselves still ask for CUDA tensors."""
    import pathlib
    import subprocess
    import sys
    code = ("import torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n    delattr(torch._C, n)\n"
            "from afterimage_b200.runtime import seq_ops as S\n"
            "assert S.tree_mask([-1, 0])[1].tolist() == [0, 1]\n"
            "c = torch.zeros(1, 1, 4, 8, dtype=torch.bfloat16)\n"
            "i = torch.zeros(1, dtype=torch.int64)\n"
            "try:\n    S.keep_cache_rows([c], i, i[None])\n"
            "except ValueError as e:\n    assert 'CUDA' in str(e), e\n"
            "else:\n    raise AssertionError('not refused')\n")
    root = pathlib.Path(_lib.__file__).resolve().parent.parent
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
