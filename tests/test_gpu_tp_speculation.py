"""Greedy decoding with a drafted tree on a GPU, over many sweeps whose kept
rows lie apart: every token judged on the prefix that was generated."""
import pytest
import torch

from bf16tol import FUSED_STEP_ATOL
from greedy_teacher import check_greedy_tokens, check_paths, record_kept, swap_best_two
from test_streaming_engine_gpu import _store, _tiny

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def stored(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("speculation")
    cfg, model = _tiny(tie=False, seed=31, layers=2)
    _, store, _ = _store(tmp, cfg, model, "s")
    return cfg, model.to("cuda"), store


@pytest.mark.parametrize("branch", [(2, 2, 1), (2, 2, 2, 2), (3,)])
@pytest.mark.parametrize("resident,kw", [("decoded", {}), ("compressed", {}), ("compressed", {"overlap": True}),
                                         ("streamed", {"slots": 2})])
def test_tokens_behind_moved_rows_are_greedy_too(stored, resident, kw, branch):
    from afterimage_b200.runtime.tp_decoder import TPDecoder, load_tp_decoder
    cfg, model, store = stored
    dec = load_tp_decoder(store, cfg, 1, 0, None, "cuda", resident=resident, **kw)
    sd = {k: v.clone().contiguous() for k, v in model.state_dict().items()}
    draft = swap_best_two(TPDecoder(cfg, sd, device="cuda"))
    paths, drafts = record_kept(dec), record_kept(draft)
    for seed in (3, 4):
        ids = torch.randint(0, cfg.vocab_size, (1, 9), generator=torch.Generator().manual_seed(seed)).cuda()
        paths.clear(), drafts.clear()
        got = dec.generate_speculative_tree(ids, 24, draft, branch)
        assert got.shape == (1, 33) and torch.equal(got[:, :9], ids)
        check_greedy_tokens(model, got, 9, FUSED_STEP_ATOL)
        check_paths(paths, 24)
        if len(branch) > 1:
            assert any(p and p != list(range(len(p))) for p in drafts[:-1]), drafts
    dec.close()
