"""Packed prompt passes, drafted trees and tree speculation of the
tensor-parallel decoder on a GPU: the kernels of seq_ops between the
projections, in every residency mode, against transformers and against the
same tokens one sequence at a time."""
import pytest
import torch

from bf16tol import FUSED_STEP_ATOL, check_logits
from test_streaming_engine_gpu import _store, _tiny
from test_tp_gpu import _check_greedy, _lib_status_clear, _ref_greedy

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def stored(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("packed")
    cfg, model = _tiny(tie=False, seed=31, layers=2)
    _, store, _ = _store(tmp, cfg, model, "p")
    return cfg, model.to("cuda"), store


def _ids(n, vocab, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).cuda()


def _cache(dec, n, batch=1):
    from afterimage_b200.runtime.tp_decoder import KVCache
    return KVCache(dec.n_layers, dec.nkv, dec.hd, n, dec.device, batch=batch)


def _ref(model, ids):
    with torch.no_grad():
        return model(input_ids=ids[None]).logits[0].float()


@pytest.mark.parametrize("resident,kw", [("decoded", {}), ("decoded", {"fused": False}), ("compressed", {}),
                                         ("compressed", {"overlap": True, "head_block_rows": 500}),
                                         ("streamed", {"slots": 2})])
def test_packed_prompts_and_trees_match_transformers(stored, resident, kw):
    from afterimage_b200.runtime.seq_ops import tree_mask
    from afterimage_b200.runtime.tp_decoder import load_tp_decoder
    cfg, model, store = stored
    dec = load_tp_decoder(store, cfg, 1, 0, None, "cuda", resident=resident, **kw)
    prompts = [_ids(n, cfg.vocab_size, n) for n in (11, 1, 60, 29)]
    more = [_ids(n, cfg.vocab_size, 90 + n) for n in (1, 8, 3, 17)]
    cache = _cache(dec, 80, batch=4)
    first, second = dec.forward_packed(prompts, cache), dec.forward_packed(more, cache)
    for b in range(4):
        check_logits(first[b], _ref(model, prompts[b])[-1], atol=FUSED_STEP_ATOL)
        check_logits(second[b], _ref(model, torch.cat((prompts[b], more[b])))[-1], atol=FUSED_STEP_ATOL)
    # a tree, and the path of it that is kept
    parents = [-1, 0, 0, 1, 2, 4, 2]
    mask, depth = tree_mask(parents, "cuda")
    toks = _ids(7, cfg.vocab_size, 5)
    one = _cache(dec, 80)
    dec.forward_packed([prompts[2]], one)
    got = dec.forward_tree(toks, mask, depth, one)
    for i in range(7):
        path = [i]
        while parents[path[0]] >= 0:
            path.insert(0, parents[path[0]])
        check_logits(got[i], _ref(model, torch.cat((prompts[2], toks[path])))[-1], atol=FUSED_STEP_ATOL)
    dec.keep_drafted(one, [0, 2, 4])
    nxt = _ids(1, cfg.vocab_size, 6)
    want = _ref(model, torch.cat((prompts[2], toks[[0, 2, 4]], nxt)))[-1]
    # the single-token step goes on from the cache that the operators wrote
    check_logits(dec.forward(nxt, one)[-1], want, atol=FUSED_STEP_ATOL)
    if resident != "decoded":
        _lib_status_clear()
    dec.close()


@pytest.mark.parametrize("branch", [(2, 2, 1), (1, 1, 1)])
@pytest.mark.parametrize("resident", ["decoded", "compressed"])
def test_tree_speculation_is_greedy_decoding(stored, resident, branch):
    from afterimage_b200.runtime.tp_decoder import TPDecoder, load_tp_decoder
    cfg, model, store = stored
    dec = load_tp_decoder(store, cfg, 1, 0, None, "cuda", resident=resident)
    ids = _ids(9, cfg.vocab_size, 3)[None]
    want, margins = _ref_greedy(model, ids, 10)
    sd = {k: v.clone().contiguous() for k, v in model.state_dict().items()}
    twin = TPDecoder(cfg, sd, device="cuda")
    other = TPDecoder(cfg, {k: v.clone() for k, v in _tiny(seed=77, layers=2)[1].to("cuda").state_dict().items()},
                      device="cuda")
    for draft, least in ((twin, 3), (other, 0)):
        stats = {}
        got = dec.generate_speculative_tree(ids, 10, draft, branch, stats=stats)
        assert got.shape == (1, 19)
        _check_greedy(got, want, margins, 9)
        assert stats["accepted_from_draft"] >= least, stats
    dec.close()


@pytest.mark.parametrize("resident", ["decoded", "compressed"])
def test_a_status_bit_raises_and_commits_nothing(stored, resident):
    from afterimage_b200 import _lib
    from afterimage_b200.runtime import _device
    from afterimage_b200.runtime.seq_ops import tree_mask
    from afterimage_b200.runtime.tp_decoder import load_tp_decoder
    cfg, model, store = stored
    dec = load_tp_decoder(store, cfg, 1, 0, None, "cuda", resident=resident)
    cache = _cache(dec, 40)
    ids = _ids(7, cfg.vocab_size, 8)
    mask, depth = tree_mask([-1, 0, 0], "cuda")
    word = _device.status_word(torch.device("cuda", torch.cuda.current_device()))
    word.fill_(_lib.STATUS_WAIT_TIMEOUT)  # as a wait that gives up leaves it
    with pytest.raises(RuntimeError, match="timed out"):
        dec.forward_packed([ids], cache)
    assert cache.lengths == [0]
    dec.forward_packed([ids], cache)  # the word was cleared
    word.fill_(_lib.STATUS_WAIT_TIMEOUT)
    with pytest.raises(RuntimeError, match="timed out"):
        dec.forward_tree(ids[:3], mask, depth, cache)
    assert cache.lengths == [7] and cache.drafted == 0
    check_logits(dec.forward_tree(ids[:3], mask, depth, cache)[0], _ref(model, torch.cat((ids, ids[:1])))[-1],
                 atol=FUSED_STEP_ATOL)
    dec.close()


@pytest.mark.parametrize("kw", [{}, {"decode_sms": 0}, {"decode_sms": 20}, {"decode_sms": 148}, {"decode_sms": 4096}],
                         ids=str)
def test_attention_beside_an_overlapped_decode_is_cut_for_every_sm(stored, kw):
    """Not for the SMs that the decode leaves: a long axis on those alone took longer than waiting for the others."""
    import ctypes

    from afterimage_b200 import _lib
    from afterimage_b200.runtime.tp_decoder import load_tp_decoder
    cfg, _, store = stored
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    dec = load_tp_decoder(store, cfg, 1, 0, None, "cuda", resident="compressed", overlap=True, **kw)
    assert dec.attention_sms == sms
    dec.close()
    # one kv head over 32768 rows: a share for (nearly) every SM
    d = _lib.AttnDesc(q=0x1000, k=0x2000, v=0x3000, out=0x4000, q_token_stride=512, q_head_stride=128,
                      out_token_stride=512, out_head_stride=128, k_token_stride=128, v_token_stride=128, tokens=1,
                      batch=1, key_rows=32768, nh=4, nkv=1, hd=128, scale=1.0, pos=0x6000, mask=0x7000, mask_cols=1,
                      sms=dec.attention_sms)
    assert _lib.load().aib_attention_workspace_floats(ctypes.byref(d)) == 64 * 128 * 130
    dec = load_tp_decoder(store, cfg, 1, 0, None, "cuda", resident="compressed")
    assert dec.attention_sms == 0  # nothing beside it: all SMs, and clusters
    dec.close()
