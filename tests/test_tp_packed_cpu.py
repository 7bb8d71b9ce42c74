"""Packed prompt passes, drafted trees and tree speculation of the
tensor-parallel decoder on CPU ranks (torch layer math): against the same
tokens one sequence at a time, and against greedy decoding."""
import pytest
import torch

from afterimage_b200.runtime.tp_decoder import KVCache, TPDecoder
from bf16tol import check_logits
from test_tp_cpu import _shard_weights, _tiny


def _dec(seed=3, arch="qwen3", tie=False):
    cfg, m = _tiny(seed, tie, arch)
    return cfg, m, TPDecoder(cfg, _shard_weights(m.state_dict(), 1, 0, tie), device="cpu")


def _cache(dec, n, batch=1):
    return KVCache(dec.n_layers, dec.nkv, dec.hd, n, dec.device, batch=batch)


def _ids(n, vocab, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("arch", ["qwen3", "llama"])
def test_packed_prompts_match_one_at_a_time(arch):
    cfg, _, dec = _dec(arch=arch)
    prompts = [_ids(n, cfg.vocab_size, n) for n in (7, 1, 19)]
    more = [_ids(n, cfg.vocab_size, 50 + n) for n in (2, 5, 1)]
    cache = _cache(dec, 40, batch=3)
    got = [dec.forward_packed(prompts, cache), dec.forward_packed(more, cache)]
    assert cache.lengths == [9, 6, 20]
    for b in range(3):
        one = _cache(dec, 40)
        for step, ids in enumerate((prompts[b], more[b])):
            # row for row the same products; oneDNN rounds a packed product differently (3 BF16 steps, as test_tp_cpu)
            check_logits(got[step][b], dec.forward(ids, one)[-1].float(), atol=2e-2)


def test_packed_prompts_refuse():
    cfg, _, dec = _dec()
    cache = _cache(dec, 8, batch=2)
    ids = _ids(5, cfg.vocab_size, 0)
    for bad, text in (([ids], "1 prompts"), ([ids, ids[:0]], "needs a token"), ([ids, _ids(9, 4, 0)], "cache of 8")):
        with pytest.raises(ValueError, match=text):
            dec.forward_packed(bad, cache)
    assert cache.lengths == [0, 0]


def test_a_tree_scores_each_node_like_its_own_path():
    from afterimage_b200.runtime.seq_ops import tree_mask
    cfg, _, dec = _dec()
    prompt = _ids(9, cfg.vocab_size, 1)
    parents = [-1, 0, 0, 1, 2, 4]
    toks = _ids(6, cfg.vocab_size, 2)
    mask, depth = tree_mask(parents)
    cache = _cache(dec, 32)
    dec.forward_packed([prompt], cache)
    whole = dec.forward_tree(toks, mask, depth, cache)
    # the same, the last three nodes in a call of their own
    cache2 = _cache(dec, 32)
    dec.forward_packed([prompt], cache2)
    parts = torch.cat((dec.forward_tree(toks[:3], mask[:3, :3], depth[:3], cache2),
                       dec.forward_tree(toks[3:], mask[3:], depth[3:], cache2)))
    assert cache.length == cache2.length == 9
    for i in range(6):
        path = [i]
        while parents[path[0]] >= 0:
            path.insert(0, parents[path[0]])
        one = _cache(dec, 32)
        ref = dec.forward(torch.cat((prompt, toks[path])), one)[-1].float()
        check_logits(whole[i], ref, atol=2e-2)
        check_logits(parts[i], ref, atol=2e-2)
    # the path 0, 2, 4 is kept: the next token sees exactly it
    dec.keep_drafted(cache, [0, 2, 4])
    assert cache.length == 12
    nxt = _ids(1, cfg.vocab_size, 7)
    one = _cache(dec, 32)
    ref = dec.forward(torch.cat((prompt, toks[[0, 2, 4]], nxt)), one)[-1].float()
    check_logits(dec.forward_packed([nxt], cache)[-1], ref, atol=2e-2)


def test_trees_refuse():
    from afterimage_b200.runtime.seq_ops import tree_mask
    cfg, _, dec = _dec()
    cache = _cache(dec, 8)
    dec.forward_packed([_ids(6, cfg.vocab_size, 0)], cache)
    mask, depth = tree_mask([-1, 0, 1])
    with pytest.raises(ValueError, match="cache of 8"):
        dec.forward_tree(_ids(3, 4, 0), mask, depth, cache)
    with pytest.raises(ValueError, match="T ids"):
        dec.forward_tree(_ids(2, 4, 0), mask, depth, cache)
    for path, text in (([1, 0], "ascend"), ([0, 0], "ascend"), ([-1], "ascend"), ([0, 2], "behind")):
        with pytest.raises(ValueError, match=text):
            dec.keep_drafted(cache, path)
    assert cache.length == 6


@pytest.mark.parametrize("branch", [(1,), (3, 2, 1), (2, 2), (1, 1, 1, 1)])
def test_tree_speculation_is_greedy_decoding(branch):
    """A draft that agrees often (the target itself, perturbed) and one that hardly does."""
    cfg, m, dec = _dec()
    ids = _ids(8, cfg.vocab_size, 4)
    want = dec.generate_greedy(ids, 12)
    sd = {k: v.clone() for k, v in m.state_dict().items()}
    g = torch.Generator().manual_seed(1)
    for k, v in sd.items():
        if v.dim() == 2:
            v += (0.004 * torch.randn(v.shape, generator=g)).to(v.dtype)
    near = TPDecoder(cfg, sd, device="cpu")
    far = _dec(seed=11)[2]
    for draft, least in ((dec, 12 * len(branch) // (len(branch) + 1) - len(branch)), (near, 1), (far, 0)):
        stats = {}
        got = dec.generate_speculative_tree(ids, 12, draft, branch, stats=stats)
        # greedy tokens may part where the two best logits are within a rounding of one another
        same = int((got == want).long().cumprod(-1).sum())
        assert same >= 8 + 6, (same, stats)
        assert stats["accepted_from_draft"] >= least and stats["sweeps"] >= 1
    assert dec.generate_speculative_tree(ids, 0, dec).shape == (1, 8)


def test_tree_speculation_refuses():
    cfg, _, dec = _dec()
    ids = _ids(4, cfg.vocab_size, 0)
    for branch in ((), (0,), (cfg.vocab_size + 1,)):
        with pytest.raises(ValueError, match="branch"):
            dec.generate_speculative_tree(ids, 4, dec, branch)


def _three(dec, vocab):
    """A cache of three sequences of different lengths, and a copy of what it holds."""
    cache = _cache(dec, 40, batch=3)
    dec.forward_packed([_ids(n, vocab, n) for n in (7, 4, 19)], cache)
    return cache, [c.clone() for c in cache.k + cache.v]


def _unchanged(cache, held, lengths):
    assert cache.lengths == lengths
    assert all(torch.equal(a, b) for a, b in zip(cache.k + cache.v, held))


@pytest.mark.parametrize("tokens", [1, 2, 5])
def test_a_forward_of_one_sequence_refuses_a_cache_of_several(tokens):
    cfg, _, dec = _dec()
    cache, held = _three(dec, cfg.vocab_size)
    with pytest.raises(ValueError, match="forward: a cache of one sequence"):
        dec.forward(_ids(tokens, cfg.vocab_size, 1), cache)
    _unchanged(cache, held, [7, 4, 19])


@pytest.mark.parametrize("path", [[], [0], [0, 1, 2], [0, 2], [3]])
def test_keeping_a_path_refuses_a_cache_of_several_sequences(path):
    cfg, _, dec = _dec()
    cache, held = _three(dec, cfg.vocab_size)
    with pytest.raises(ValueError, match="keep_drafted: a cache of one sequence"):
        dec.keep_drafted(cache, path)
    _unchanged(cache, held, [7, 4, 19])


def test_nodes_that_were_never_run_are_not_kept():
    from afterimage_b200.runtime.seq_ops import tree_mask
    cfg, _, dec = _dec()
    cache = _cache(dec, 40)
    dec.forward_packed([_ids(7, cfg.vocab_size, 0)], cache)
    mask, depth = tree_mask([-1, 0, 0, 1, 2])

    def refused(*paths):
        held, n = [c.clone() for c in cache.k + cache.v], cache.length
        for path in paths:
            with pytest.raises(ValueError, match="never run"):
                dec.keep_drafted(cache, path)
        _unchanged(cache, held, [n])

    refused([0], [0, 1, 2, 3, 4])           # no tree at all
    dec.forward_tree(_ids(3, cfg.vocab_size, 1), mask[:3, :3], depth[:3], cache)
    refused([3], [0, 1, 3])                 # a tree of three
    dec.forward_tree(_ids(2, cfg.vocab_size, 2), mask[3:], depth[3:], cache)
    refused([5], [0, 2, 5])                 # the same, with two more
    dec.keep_drafted(cache, [])             # keeps nothing, and the tree stands
    dec.keep_drafted(cache, [0, 2, 4])
    assert cache.length == 10
    refused([0], [1])                       # the tree is gone with its numbers
    cache.length = 7
    refused([0], [1])
    cache.length = 10
    for write in (lambda: dec.forward(_ids(1, cfg.vocab_size, 3), cache),
                  lambda: dec.forward(_ids(2, cfg.vocab_size, 3), cache),
                  lambda: dec.forward_packed([_ids(2, cfg.vocab_size, 3)], cache)):
        dec.forward_tree(_ids(5, cfg.vocab_size, 4), mask, depth, cache)
        n = cache.length
        write()
        refused([0], [1])                   # its rows are written over
        cache.length = n
        refused([0], [1])                   # and stay so when the tokens are cut again
    dec.forward_tree(_ids(2, cfg.vocab_size, 5), mask[:2, :2], depth[:2], cache)
    cache.length -= 1
    refused([0], [1])                       # its numbers count from another row now


@pytest.mark.parametrize("fails", ["forward_packed", "forward_tree"])
def test_a_pass_whose_kernels_gave_up_raises_and_commits_nothing(monkeypatch, fails):
    """A bounded wait that gives up leaves rows unwritten and sets the status word (stood in for here)."""
    from afterimage_b200.runtime import tp_decoder
    from afterimage_b200.runtime.seq_ops import tree_mask
    cfg, _, dec = _dec()
    cache = _cache(dec, 40)
    dec.forward_packed([_ids(7, cfg.vocab_size, 0)], cache)
    mask, depth = tree_mask([-1, 0, 0])

    def gave_up(dev):
        raise RuntimeError("a bounded shared-memory copy wait timed out")

    with monkeypatch.context() as m:
        m.setattr(tp_decoder._device, "check_status", gave_up)
        with pytest.raises(RuntimeError, match="timed out"):
            if fails == "forward_packed":
                dec.forward_packed([_ids(2, cfg.vocab_size, 1)], cache)
            else:
                dec.forward_tree(_ids(3, cfg.vocab_size, 1), mask, depth, cache)
    assert cache.lengths == [7] and cache.drafted == 0


@pytest.mark.parametrize("branch", [(2, 2, 1), (2, 2, 2, 2), (3,)])
def test_tokens_behind_moved_rows_are_greedy_too(branch):
    """24 tokens, each judged on its own prefix; the draft's second choice is the target's first, so that every sweep
    goes on from rows that keep_drafted moved together, in both caches."""
    from greedy_teacher import check_greedy_tokens, check_paths, record_kept, swap_best_two
    cfg, m, dec = _dec()
    draft = swap_best_two(_dec()[2])
    paths, drafts = record_kept(dec), record_kept(draft)
    got = dec.generate_speculative_tree(_ids(9, cfg.vocab_size, 6), 24, draft, branch)
    assert got.shape == (1, 33)
    check_greedy_tokens(m, got, 9, 2e-2)  # (the tolerance of the packed passes above)
    check_paths(paths, 24)
    if len(branch) > 1:
        assert any(p and p != list(range(len(p))) for p in drafts[:-1]), drafts
