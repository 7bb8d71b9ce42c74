"""Whether generated tokens are greedy decoding's, each judged on the prefix
that was actually generated: no early stop where two logits are close.

A decoder takes the largest of its logits, each of which is within a of the
reference's on the same prefix (a: what bf16tol.check_logits allows). The
token t that it takes and the reference's best one b then satisfy
    ref[t] >= got[t] - a >= got[b] - a >= ref[b] - 2 a.
"""
import torch

from bf16tol import bf16_ulp


def check_greedy_tokens(model, seq: torch.Tensor, n_prompt: int, atol: float) -> None:
    """seq [1, n]: every token behind the prompt within 2 a of the best logit of `model` (transformers) there."""
    with torch.no_grad():
        ref = model(input_ids=seq).logits[0, n_prompt - 1:-1].float()
    best = ref.max(-1).values
    a = torch.maximum(torch.full_like(best, atol), bf16_ulp(best))
    near = (ref >= (best - 2 * a)[:, None]).sum(-1)
    # the check says something: a token that has nothing to do with the prefix would pass once in a hundred times
    assert float(near.float().mean()) <= ref.shape[-1] / 100, near.tolist()
    took = ref.gather(1, seq[0, n_prompt:, None])[:, 0]
    assert bool((took >= best - 2 * a).all()), [(i, float(b - t)) for i, (b, t) in enumerate(zip(best, took))]


def swap_best_two(draft):
    """Makes a decoder rank its best token second: a tree then goes on from second children, and the rows that are kept
    lie apart."""
    def swapped(f):
        def call(*args):
            lg = f(*args).clone()
            top = lg.topk(2, -1)
            return lg.scatter_(-1, top.indices, top.values.flip(-1))
        return call
    draft.forward_packed, draft.forward_tree = swapped(draft.forward_packed), swapped(draft.forward_tree)
    return draft


def record_kept(dec) -> list:
    """The paths that `dec` keeps from now on."""
    paths, keep = [], dec.keep_drafted

    def call(cache, path):
        paths.append(list(path))
        keep(cache, path)
    dec.keep_drafted = call
    return paths


def check_paths(paths: list, tokens: int) -> None:
    """Several sweeps, and rows from places apart kept before the last of them."""
    assert len(paths) >= 2 and sum(map(len, paths)) >= tokens - 1, paths
    assert any(p != list(range(len(p))) for p in paths[:-1]), paths
