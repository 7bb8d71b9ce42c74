"""The kernels over cached sequences against their plain 64-bit forms
(seq_ref.py, which derives the tolerances), at the sizes, masks, layouts and
values where such kernels go wrong."""
import pytest
import torch

import seq_ref as R

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
DEV = "cuda"


def _ops():
    from afterimage_b200.runtime import seq_ops
    return seq_ops


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _n(g, *shape, by=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * by).to(BF)


def _i(v):
    return torch.tensor(v, dtype=torch.int64, device=DEV)


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return _i(out)


HEADS = [(4, 4, 128), (8, 2, 128), (5, 1, 128), (10, 2, 64), (4, 2, 80), (3, 1, 16), (6, 2, 36), (2, 1, 256),
         (12, 1, 128), (7, 1, 8), (130, 1, 64)]
LENS = [[1], [2, 1, 3], [128], [129, 127], [0, 5, 0, 64, 0], [25, 26, 24], [300, 1, 77, 256], [513]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_packed_prompts(nh, nkv, hd, lens):
    g = _gen(nh * hd + len(lens))
    n = sum(lens)
    q, k, v = _n(g, n, nh, hd, by=1.5), _n(g, n, nkv, hd), _n(g, n, nkv, hd)
    cu = _cu(lens)
    got = _ops().prompt_attention(q, k, v, cu, hd ** -0.5)
    R.check(got, *R.prompt(q, k, v, cu, hd ** -0.5)[:2])


@pytest.mark.parametrize("lens", [[600], [300, 1, 77, 256], [129, 130, 0, 700], [26] * 20], ids=str)
@pytest.mark.parametrize("nh,nkv,hd", [(148, 148, 128), (100, 50, 64), (160, 32, 128), (120, 40, 80)])
def test_enough_heads_to_fill_every_sm(nh, nkv, hd, lens):
    """Two tiles to a block, the second partly or wholly empty."""
    g = _gen(nh * hd + len(lens))
    n = sum(lens)
    q, k, v = _n(g, n, nh, hd, by=1.5), _n(g, n, nkv, hd), _n(g, n, nkv, hd)
    k[lens[0] - 1] = 0
    v[lens[0] - 1, :, :9] = float("inf")  # the first sequence's last value
    got = _ops().prompt_attention(q, k, v, _cu(lens), hd ** -0.5)
    R.check(got, *R.prompt(q, k, v, _cu(lens), hd ** -0.5)[:2])


def test_many_sequences():
    """More sequences than a warp has lanes, empty ones among them."""
    g = _gen(70)
    lens = torch.randint(0, 90, (131,), device=DEV, generator=g).tolist()
    lens[5], lens[77], lens[130] = 0, 400, 300
    n = sum(lens)
    for nh, nkv, hd in ((8, 8, 64), (2, 1, 64)):
        q, k, v = _n(g, n, nh, hd, by=1.5), _n(g, n, nkv, hd), _n(g, n, nkv, hd)
        got = _ops().prompt_attention(q, k, v, _cu(lens), hd ** -0.5)
        R.check(got, *R.prompt(q, k, v, _cu(lens), hd ** -0.5)[:2])


@pytest.mark.parametrize("lens,ctx", [([1], [0]), ([64], [500]), ([130, 3], [1, 700]), ([7, 200, 31], [0, 129, 1000])])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (5, 1, 128), (4, 2, 64), (6, 2, 36)])
def test_prompts_over_caches(nh, nkv, hd, lens, ctx):
    g = _gen(sum(ctx) + nh)
    rows = max(a + c for a, c in zip(lens, ctx)) + 13
    q = _n(g, sum(lens), nh, hd, by=1.5)
    k, v = _n(g, len(lens), nkv, rows, hd), _n(g, len(lens), nkv, rows, hd)
    len_k = _i([a + c for a, c in zip(lens, ctx)])
    for b, L in enumerate(len_k.tolist()):  # what lies behind a sequence's keys is nobody's
        k[b, :, L:] = float("nan")
        v[b, :, L:] = float("inf")
    got = _ops().prompt_attention(q, k, v, _cu(lens), hd ** -0.5, len_k=len_k)
    R.check(got, *R.prompt(q, k, v, _cu(lens), hd ** -0.5, len_k=len_k)[:2])


def test_queries_before_their_first_key_are_zero():
    """More queries than keys: the first rows see nothing; also a sequence without keys."""
    g = _gen(1)
    q, k, v = _n(g, 300, 8, 128), _n(g, 140, 2, 128), _n(g, 140, 2, 128)
    cu_q, cu_k = _i([0, 290, 296, 300]), _i([0, 137, 137, 140])
    got = _ops().prompt_attention(q, k, v, cu_q, 0.1, cu_k=cu_k)
    want, size, _ = R.prompt(q, k, v, cu_q, 0.1, cu_k=cu_k)
    R.check(got, want, size)
    assert not got[:153].any() and not got[290:297].any()


@pytest.mark.parametrize("nh,nkv,hd", [(148, 148, 128), (148, 74, 64)])
def test_a_first_tile_that_sees_nothing_beside_a_second_that_does(nh, nkv, hd):
    g = _gen(62)
    for m, L in ((600, 200), (512, 130), (300, 44)):
        q, k, v = _n(g, m, nh, hd), _n(g, L, nkv, hd), _n(g, L, nkv, hd)
        for _ in range(4):
            out = torch.full_like(q, 5.0)
            _ops().prompt_attention(q, k, v, _cu([m]), 0.1, cu_k=_cu([L]), out=out)
            assert not out[:m - L].any()
        R.check(out, *R.prompt(q, k, v, _cu([m]), 0.1, cu_k=_cu([L]))[:2])


def test_rows_outside_every_sequence_stay():
    g = _gen(2)
    q, k, v = _n(g, 200, 8, 128), _n(g, 200, 2, 128), _n(g, 200, 2, 128)
    cu = _i([3, 80, 150])
    out = torch.full_like(q, 7.0)
    _ops().prompt_attention(q, k, v, cu, 0.1, out=out)
    want, size, rows = R.prompt(q, k, v, cu, 0.1)
    R.check(out[rows.to(DEV)], want[rows], size[rows])
    assert bool((out[~rows.to(DEV)] == 7.0).all())


def test_offsets_beyond_the_tensors_are_cut():
    """Lengths on the device that say more than the tensors hold."""
    g = _gen(3)
    q, k, v = _n(g, 50, 4, 64), _n(g, 50, 2, 64), _n(g, 50, 2, 64)
    got = _ops().prompt_attention(q, k, v, _i([0, 20, 10 ** 12]), 0.1)
    R.check(got, *R.prompt(q, k, v, _i([0, 20, 50]), 0.1)[:2])
    c, d = _n(g, 1, 2, 40, 64), _n(g, 1, 2, 40, 64)
    got = _ops().prompt_attention(q[:8], c, d, _i([0, 8]), 0.1, len_k=_i([10 ** 12]))
    R.check(got, *R.prompt(q[:8], c, d, _i([0, 8]), 0.1, len_k=_i([40]))[:2])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (5, 1, 64), (6, 2, 36)])
def test_values_that_a_row_does_not_see_do_not_reach_it(nh, nkv, hd, bad):
    """NaN and infinities in later tokens' keys and values, in the middle of a key tile."""
    g = _gen(4)
    q, k, v = _n(g, 200, nh, hd, by=1.5), _n(g, 200, nkv, hd), _n(g, 200, nkv, hd)
    v[70, :, 3] = bad
    v[150, 0] = bad
    k[199, 0] = float("nan")
    cu = _i([0, 60, 200])
    got = _ops().prompt_attention(q, k, v, cu, hd ** -0.5)
    want, size, _ = R.prompt(q, k, v, cu, hd ** -0.5)
    assert torch.isfinite(want[:70]).all() and not torch.isfinite(want[70:, 0]).all()
    # the last row sees the NaN key: its own outputs of that kv head are NaN
    R.check(got, want, size)


def test_strided_and_unaligned_prompts():
    """q, k, v as views of one projection's rows; an output with gaps; a view whose rows start off 16 bytes."""
    g = _gen(5)
    nh, nkv, hd, n = 8, 2, 128, 333
    cu = _cu([300, 33])
    for pad in (0, 8, 1):
        x = _n(g, n, (nh + 2 * nkv) * hd + pad)[:, pad:]
        q, k, v = (t.unflatten(-1, (-1, hd)) for t in x.split([nh * hd, nkv * hd, nkv * hd], -1))
        out = torch.full((n, nh + 1, hd + 8), 5.0, device=DEV, dtype=BF)
        got = _ops().prompt_attention(q, k, v, cu, 0.1, out=out[:, 1:, :hd])
        R.check(got, *R.prompt(q, k, v, cu, 0.1)[:2])
        assert bool((out[:, 0] == 5).all()) and bool((out[:, :, hd:] == 5).all())


def test_one_key_and_value_for_all_heads_by_an_expanded_tensor():
    g = _gen(6)
    q, k, v = _n(g, 90, 4, 64), _n(g, 90, 1, 64).expand(90, 4, 64), _n(g, 90, 1, 64).expand(90, 4, 64)
    R.check(_ops().prompt_attention(q, k, v, _i([0, 90]), 0.1), *R.prompt(q, k, v, _i([0, 90]), 0.1)[:2])


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (3, 1, 48), (8, 2, 128)])
def test_two_tiles_over_many_keys_with_values_that_are_not_finite(nh, nkv, hd):
    """One SM to count on, so that every block has two tiles; more key tiles than the ring holds, bad ones among them."""
    g = _gen(71)
    lens = [1500, 1, 130, 900]
    n = sum(lens)
    q, k, v = _n(g, n, nh, hd, by=1.5), _n(g, n, nkv, hd), _n(g, n, nkv, hd)
    for i, row in enumerate((130, 700, 1100, 1499, 1631, 2100, n - 1)):
        v[row, 0, i % hd] = (float("nan"), float("inf"), float("-inf"))[i % 3]
    cu = _cu(lens)
    want = R.prompt(q, k, v, cu, 0.1)[:2]
    for _ in range(3):
        R.check(_ops().prompt_attention(q, k, v, cu, 0.1, sms=1), *want)
    t = 200
    q, k, v = _n(g, 2, t, nh, hd, by=1.5), _n(g, 2, nkv, 1700, hd), _n(g, 2, nkv, 1700, hd)
    v[0, 0, 1350, 1] = float("nan")  # a column of the mask
    v[1, 0, 40, 2] = float("inf")
    mask = torch.rand(2, t, t, device=DEV, generator=g) < 0.2
    R.check(_ops().tree_attention(q, k, v, _i([1300, 1]), mask, 0.1, sms=1), *R.tree(q, k, v, [1300, 1], mask, 0.1))


@pytest.mark.parametrize("sms", [0, 90])
@pytest.mark.parametrize("nkv", [1, 3, 9, 18])
@pytest.mark.parametrize("hd", [40, 64, 72, 128])
def test_every_number_of_shares(hd, nkv, sms):
    """2, 4, 8 and 16 shares of the key axis in a cluster, others with a second kernel."""
    g = _gen(73 + hd)
    mask, _ = _ops().tree_mask([-1, 0, 1, 1, 0], DEV)
    for rows in (300, 900, 1900, 3000, 5000):
        q, k, v = _n(g, 1, 5, 4 * nkv, hd, by=1.5), _n(g, 1, nkv, rows, hd), _n(g, 1, nkv, rows, hd)
        for pos in (rows - 5, rows // 2, 0):
            R.check(_ops().tree_attention(q, k, v, _i([pos]), mask, hd ** -0.5, sms=sms),
                    *R.tree(q, k, v, [pos], mask, hd ** -0.5))
        R.check(_ops().prompt_attention(q[0], k, v, _cu([5]), hd ** -0.5, len_k=_i([rows]), sms=sms),
                *R.prompt(q[0], k, v, _cu([5]), hd ** -0.5, len_k=_i([rows]))[:2])


@pytest.mark.parametrize("sms", [0, 20, 100])
@pytest.mark.parametrize("hd", [64, 128])
def test_infinite_values_in_the_last_share(hd, sms):
    """A value that every row sees is infinite: so is the output, whichever way the shares of the key axis are joined."""
    g = _gen(72)
    q, k, v = _n(g, 1, 5, 8, hd), _n(g, 1, 2, 3000, hd), _n(g, 1, 2, 3000, hd)
    v[0, 0, 2890, 3] = float("inf")
    v[0, 1, 2700, 1] = float("-inf")
    v[0, 1, 10, 2] = float("inf")
    mask, _ = _ops().tree_mask([-1, 0, 1, 1, 0], DEV)
    want, size = R.tree(q, k, v, [2900], mask, 0.1)
    assert torch.isinf(want).sum() == 5 * 4 * 3
    R.check(_ops().tree_attention(q, k, v, _i([2900]), mask, 0.1, sms=sms), want, size)
    cu = _cu([5])
    R.check(_ops().prompt_attention(q[0], k, v, cu, 0.1, len_k=_i([2905]), sms=sms),
            *R.prompt(q[0], k, v, cu, 0.1, len_k=_i([2905]))[:2])


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30])
def test_scales_that_are_not_positive(scale):
    g = _gen(60)
    q, k, v = _n(g, 150, 4, 128), _n(g, 150, 2, 128), _n(g, 150, 2, 128)
    R.check(_ops().prompt_attention(q, k, v, _cu([100, 50]), scale), *R.prompt(q, k, v, _cu([100, 50]), scale)[:2])


def test_no_keys_at_all():
    q, k = torch.ones(5, 4, 64, dtype=BF, device=DEV), torch.ones(0, 2, 64, dtype=BF, device=DEV)
    out = torch.full_like(q, 3.0)
    _ops().prompt_attention(q, k, k, _cu([2, 3]), 0.1, cu_k=_cu([0, 0]), out=out)
    assert not out.any()


def test_the_output_may_be_the_queries():
    """A block has read its queries before it writes them, also where the key axis is shared out."""
    g = _gen(61)
    for n, nh, nkv in ((700, 4, 2), (300, 160, 32)):
        q, k, v = _n(g, n, nh, 128), _n(g, n, nkv, 128), _n(g, n, nkv, 128)
        want = _ops().prompt_attention(q, k, v, _cu([n - 30, 30]), 0.1)
        assert torch.equal(_ops().prompt_attention(q, k, v, _cu([n - 30, 30]), 0.1, out=q), want)


@pytest.mark.parametrize("sms", [1, 20, 33, 100, 1000])
def test_beside_other_kernels(sms):
    """Fewer SMs to count on: other shares and no clusters, the same result up to the order of sums."""
    g = _gen(63)
    q, k, v = _n(g, 1, 5, 32, 128), _n(g, 1, 8, 3000, 128), _n(g, 1, 8, 3000, 128)
    mask, _ = _ops().tree_mask([-1, 0, 1, 1, 0], DEV)
    R.check(_ops().tree_attention(q, k, v, _i([2900]), mask, 0.1, sms=sms), *R.tree(q, k, v, [2900], mask, 0.1))
    q, k, v = _n(g, 700, 10, 64), _n(g, 700, 5, 64), _n(g, 700, 5, 64)
    R.check(_ops().prompt_attention(q, k, v, _cu([600, 100]), 0.1, sms=sms),
            *R.prompt(q, k, v, _cu([600, 100]), 0.1)[:2])


def test_large_scores():
    """Scores of several hundred, rising along the keys: the running maximum has to follow, and early weights vanish."""
    g = _gen(7)
    q, k, v = _n(g, 700, 4, 128), _n(g, 700, 2, 128), _n(g, 700, 2, 128)
    q = q.abs()
    k = (k.abs() * torch.linspace(0.1, 3, 700, device=DEV)[:, None, None]).to(BF)
    cu = _i([0, 700])
    got = _ops().prompt_attention(q, k, v, cu, 1.0)
    want, size, _ = R.prompt(q, k, v, cu, 1.0)
    # a score of z carries an error of hd 2^-24 z = 8e-6 z or so: below 0.005 for z up to 600, which is the
    # relative error of a weight; the weights' errors add to at most twice that of mean|v|
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 0.01) * size
    assert bool(((got.double().cpu() - want).abs() <= tol).all())


TREE = [-1, 0, 0, 1, 1, 2, 3, 3, 5, 6, 8, 8]


@pytest.mark.parametrize("pos", [[0], [1], [127], [128], [1000], [300, 0, 511]], ids=str)
@pytest.mark.parametrize("t", [1, 2, 12])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (5, 1, 128), (4, 4, 64), (4, 2, 80), (6, 2, 36), (40, 8, 128)])
def test_trees(nh, nkv, hd, t, pos):
    g = _gen(t + sum(pos))
    rows = max(pos) + t + 5
    b = len(pos)
    q, k, v = _n(g, b, t, nh, hd, by=1.5), _n(g, b, nkv, rows, hd), _n(g, b, nkv, rows, hd)
    for i, p in enumerate(pos):
        k[i, :, p + t:] = float("nan")
        v[i, :, p + t:] = float("nan")
    mask, _ = _ops().tree_mask(TREE[:t], DEV)
    got = _ops().tree_attention(q, k, v, _i(pos), mask, hd ** -0.5)
    R.check(got, *R.tree(q, k, v, pos, mask, hd ** -0.5))


@pytest.mark.parametrize("t,cols,pos", [(70, 70, 900), (3, 200, 100), (257, 257, 130), (1, 300, 0)])
def test_wide_trees_and_random_masks(t, cols, pos):
    """More columns than queries, masks with empty rows, a mask of its own for each sequence, odd strides."""
    g = _gen(t)
    b, nh, nkv, hd = 2, 10, 2, 128
    q = _n(g, b, t, nh, hd, by=1.5)
    k, v = _n(g, b, nkv, pos + cols + 9, hd), _n(g, b, nkv, pos + cols + 9, hd)
    mask = torch.rand(b, t, cols, device=DEV, generator=g) < 0.3
    mask[:, 0] = False
    p = [pos, max(0, pos - 50)]
    want, size = R.tree(q, k, v, p, mask, 0.1)
    R.check(_ops().tree_attention(q, k, v, _i(p), mask, 0.1), want, size)
    odd = torch.zeros(b, t, 2 * cols + 1, dtype=torch.bool, device=DEV)[:, :, 1::2]
    odd.copy_(mask)
    R.check(_ops().tree_attention(q, k, v, _i(p), odd, 0.1), want, size)
    qt = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)  # heads outside the tokens
    out = torch.empty(t, b, nh, hd, device=DEV, dtype=BF).transpose(0, 1)
    R.check(_ops().tree_attention(qt, k, v, _i(p), mask, 0.1, out=out), want, size)


@pytest.mark.parametrize("nh,nkv,hd,t", [(40, 8, 128, 60), (16, 16, 64, 200), (16, 8, 128, 130)])
def test_a_batch_of_wide_trees(nh, nkv, hd, t):
    """Enough work for two tiles to a block."""
    g = _gen(t)
    b, rows = 20, 500
    pos = torch.randint(0, rows - t, (b,), device=DEV, generator=g)
    q, k, v = _n(g, b, t, nh, hd, by=1.5), _n(g, b, nkv, rows, hd), _n(g, b, nkv, rows, hd)
    mask = torch.rand(b, t, t, device=DEV, generator=g) < 0.2
    want, size = R.tree(q, k, v, pos.tolist(), mask, hd ** -0.5)
    R.check(_ops().tree_attention(q, k, v, pos, mask, hd ** -0.5), want, size)


def test_a_tree_row_that_sees_nothing_is_zero():
    g = _gen(8)
    q, k, v = _n(g, 1, 3, 4, 128), _n(g, 1, 2, 20, 128), _n(g, 1, 2, 20, 128)
    mask = torch.tensor([[0, 0, 0], [1, 0, 0], [0, 0, 0]], dtype=torch.bool, device=DEV)
    got = _ops().tree_attention(q, k, v, _i([0]), mask, 0.1)
    assert not got[0, 0].any() and not got[0, 2].any()
    R.check(got, *R.tree(q, k, v, [0], mask, 0.1))
    none = torch.zeros(1, 3, 0, dtype=torch.bool, device=DEV)  # no drafted tokens in the cache: the prefix alone
    R.check(_ops().tree_attention(q, k, v, _i([9]), none, 0.1), *R.tree(q, k, v, [9], none, 0.1))


@pytest.mark.parametrize("pos", [-2, -9, 18, 40])
def test_tree_positions_partly_or_wholly_outside_the_cache(pos):
    g = _gen(9)
    q, k, v = _n(g, 1, 4, 4, 64), _n(g, 1, 2, 20, 64), _n(g, 1, 2, 20, 64)
    mask = torch.ones(4, 4, dtype=torch.bool, device=DEV).tril()
    R.check(_ops().tree_attention(q, k, v, _i([pos]), mask, 0.1), *R.tree(q, k, v, [pos], mask, 0.1))


def test_a_sibling_with_nan_does_not_reach_the_others():
    g = _gen(10)
    q, k, v = _n(g, 1, 3, 8, 128), _n(g, 1, 2, 64, 128), _n(g, 1, 2, 64, 128)
    k[0, :, 31] = float("nan")
    v[0, :, 31] = float("inf")
    mask, _ = _ops().tree_mask([-1, 0, 0], DEV)
    got = _ops().tree_attention(q, k, v, _i([30]), mask, 0.1)
    want, size = R.tree(q, k, v, [30], mask, 0.1)
    assert torch.isfinite(want[0, [0, 2]]).all()
    R.check(got, want, size)


def test_the_cache_beyond_32_bit_offsets():
    """A cache of more than 2^31 elements, its last sequence read and written."""
    S = _ops()
    rows, nkv, hd = 70000, 8, 128
    b = 2 ** 31 // (rows * nkv * hd) + 2
    k = torch.empty(b, nkv, rows, hd, dtype=BF, device=DEV)
    v = torch.empty_like(k)
    g = _gen(11)
    k[-1], v[-1] = _n(g, nkv, rows, hd), _n(g, nkv, rows, hd)
    q = _n(g, b, 1, 8, hd)
    pos = _i([0] * (b - 1) + [2000])
    mask = torch.ones(1, 1, dtype=torch.bool, device=DEV)
    k[:-1, :, 0], v[:-1, :, 0] = 0, 1
    got = S.tree_attention(q, k, v, pos, mask, 0.1)
    assert bool((got[:-1] == 1).all())
    R.check(got[-1:], *R.tree(q[-1:], k[-1:, :, :2001], v[-1:, :, :2001], [2000], mask, 0.1))
    before = v[-1, :, 69999].clone()
    S.keep_cache_rows([k, v], _i([0] * (b - 1) + [69990]), _i([[-1, -1]] * (b - 1) + [[9, 0]]))
    assert torch.equal(v[-1, :, 69990], before)


@pytest.mark.parametrize("nh,nkv,hd", [(40, 8, 128), (4, 2, 64), (4, 2, 80), (2, 1, 18), (2, 2, 256), (1, 1, 2)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("tree", [False, True])
def test_rope_cache_packed(nh, nkv, hd, norm, tree):
    g = _gen(nh + hd)
    lens, start = [5, 0, 33, 1], [0, 4, 100000, 11]
    n, rows = sum(lens), 64
    start_d = _i(start)
    qkv = _n(g, n, (nh + 2 * nkv) * hd)
    depth = torch.randint(0, 9, (n,), device=DEV, generator=g) if tree else None
    w = [(1 + 0.2 * torch.randn(hd, device=DEV, generator=g)).to(BF) if norm else None for _ in range(2)]
    inv_freq = 1.0 / (1e4 ** (torch.arange(0, hd, 2, device=DEV, dtype=torch.float32) / hd))
    max_len = 100000 + rows if hd == 64 else rows  # elsewhere the third sequence lies behind its cache
    k, v = (torch.full((4, nkv, max_len, hd), 3.0, dtype=BF, device=DEV) for _ in range(2))
    got = _ops().rope_cache_packed(qkv, nh, nkv, hd, _cu(lens), start_d, inv_freq, k, v, depth=depth, q_norm=w[0],
                                   k_norm=w[1], eps=1e-6)
    q, qs, kk, ks, vv, seq, slot = R.rope(qkv, nh, nkv, hd, _cu(lens), start_d, inv_freq, depth, w[0], w[1])
    # one rounding (2^-8 of the value) and fp32 angles below pi, norms and sums: 2e-6 of the two terms
    assert bool(((got.double().cpu() - q).abs() <= 2.0 ** -8 * q.abs() + 2e-6 * qs).all())
    want_k, want_v = (torch.full((4, nkv, max_len, hd), 3.0, dtype=torch.float64) for _ in range(2))
    size = torch.zeros_like(want_k)
    for i in range(n):
        if slot[i] < max_len:
            want_k[seq[i], :, slot[i]], want_v[seq[i], :, slot[i]], size[seq[i], :, slot[i]] = kk[i], vv[i], ks[i]
    assert torch.equal(v.double().cpu(), want_v)
    assert bool(((k.double().cpu() - want_k).abs() <= 2.0 ** -8 * want_k.abs() + 2e-6 * size).all())


def test_rope_rows_outside_sequences_and_strided_caches():
    g = _gen(12)
    nh, nkv, hd = 4, 2, 128
    x = _n(g, 20, (nh + 2 * nkv) * hd + 24)
    qkv = x[:, 8:8 + (nh + 2 * nkv) * hd]
    cu, start = _i([2, 9, 15]), _i([-3, 4])
    inv_freq = 1.0 / (1e4 ** (torch.arange(0, hd, 2, device=DEV, dtype=torch.float32) / hd))
    kv = torch.full((2, 16, 2, nkv, hd), 3.0, dtype=BF, device=DEV)  # rows outside the heads, keys beside values
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    out = torch.full((20, nh, hd), 9.0, dtype=BF, device=DEV)
    _ops().rope_cache_packed(qkv, nh, nkv, hd, cu, start, inv_freq, k, v, out=out)
    q, qs, kk, ks, vv, seq, slot = R.rope(qkv, nh, nkv, hd, cu, start, inv_freq)
    assert bool((out[:2] == 9).all()) and bool((out[15:] == 9).all())
    assert bool(((out[2:15].double().cpu() - q[2:15]).abs() <= 2.0 ** -8 * q[2:15].abs() + 2e-6 * qs[2:15]).all())
    written = torch.zeros(2, 16, dtype=torch.bool)
    for i in range(2, 15):
        if slot[i] >= 0:
            written[seq[i], slot[i]] = True
            assert torch.equal(v[seq[i], :, slot[i]].double().cpu(), vv[i])
    assert bool((v.transpose(1, 2)[~written.to(DEV)] == 3).all())
    assert bool((k.transpose(1, 2)[~written.to(DEV)] == 3).all())


@pytest.mark.parametrize("nkv,hd,layers", [(8, 128, 40), (2, 64, 3), (3, 20, 2), (1, 1024, 1), (2, 128, 150)])
@pytest.mark.parametrize("n", [1, 5, 64, 256])
def test_keep_cache_rows(nkv, hd, layers, n):
    g = _gen(n + hd)
    b, rows = 2, 400
    caches = [_n(g, b, nkv, rows, hd) for _ in range(layers)]
    keep = torch.randint(-1, 300, (b, n), device=DEV, generator=g)  # any order, rows twice, rows behind the cache
    keep[0] = keep[0].sort().values
    pos = _i([3, 150])
    want = [c.clone() for c in caches]
    for c in want:
        old = c.clone()
        for i in range(b):
            for j in range(n):
                s, d = int(pos[i]) + int(keep[i, j]), int(pos[i]) + j
                if int(keep[i, j]) >= 0 and 0 <= s < rows and 0 <= d < rows:
                    c[i, :, d] = old[i, :, s]
        if layers > 3:
            break  # the first cache in full; the others against it below
    _ops().keep_cache_rows(caches, pos, keep)
    if layers <= 3:
        for got, w in zip(caches, want):
            assert torch.equal(got.view(torch.int16), w.view(torch.int16))
        return
    assert torch.equal(caches[0].view(torch.int16), want[0].view(torch.int16))
    place = torch.arange(n, device=DEV)
    src, dst = pos[:, None] + keep, pos[:, None] + place
    ok = (keep >= 0) & (src >= 0) & (src < rows) & (dst < rows)
    row = torch.arange(b, device=DEV)[:, None].expand(b, n)
    for got, w in zip(caches[1:], want[1:]):
        old = w.clone()
        w[row[ok], :, dst[ok]] = old[row[ok], :, src[ok]]
        assert torch.equal(got.view(torch.int16), w.view(torch.int16))


def test_keep_cache_rows_strided_and_odd():
    g = _gen(13)
    kv = _n(g, 2, 50, 2, 3, 17)  # rows outside heads, 34-byte rows
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    want = kv.clone()
    want[0, 5:8] = kv[0, [5, 9, 30]]
    want[1, 40] = kv[1, 49]
    _ops().keep_cache_rows([k, v], _i([5, 40]), _i([[0, 4, 25], [9, -1, -5]]))
    assert torch.equal(kv.view(torch.int16), want.view(torch.int16))


def _pass(S, g, lens, nh=8, nkv=2, hd=128, rows=256):
    """Rope and cache write, prompt attention over the caches, a drafted tree behind it, the kept path: the run of
    operators as a generation loop makes it. Returns everything that it writes."""
    b = len(lens)
    k, v = (torch.zeros(b, nkv, rows, hd, dtype=BF, device=DEV) for _ in range(2))
    inv_freq = 1.0 / (1e4 ** (torch.arange(0, hd, 2, device=DEV, dtype=torch.float32) / hd))
    x = _n(g, sum(lens), (nh + 2 * nkv) * hd)
    cu, zero, len_k = _cu(lens), _i([0] * b), _i(lens)
    mask, depth = S.tree_mask([-1, 0, 0, 1, 2], DEV)
    y = _n(g, 5 * b, (nh + 2 * nkv) * hd)
    tcu, keep = _i([5 * i for i in range(b + 1)]), _i([[0, 2, 4]] * b)

    def run():
        q = S.rope_cache_packed(x, nh, nkv, hd, cu, zero, inv_freq, k, v)
        a = S.prompt_attention(q, k, v, cu, hd ** -0.5, len_k=len_k)
        tq = S.rope_cache_packed(y, nh, nkv, hd, tcu, len_k, inv_freq, k, v, depth=depth.repeat(b))
        t = S.tree_attention(tq.view(b, 5, nh, hd), k, v, len_k, mask, hd ** -0.5)
        S.keep_cache_rows([k, v], len_k, keep)
        return q, a, tq, t, k.clone(), v.clone()

    return run, (x, y, k, v, cu, len_k, mask)


def test_the_operators_run_together():
    S, g = _ops(), _gen(14)
    lens = [100, 1, 37]
    run, (x, y, k, v, cu, len_k, mask) = _pass(S, g, lens)
    q, a, tq, t, kk, vv = run()
    # the tree's rows before the path was kept
    for b, L in enumerate(lens):
        y5 = y[5 * b:5 * b + 5].view(5, 12, 128)
        assert torch.equal(vv[b, :, L:L + 3], y5[[0, 2, 4], 10:].transpose(0, 1))
        vv[b, :, L:L + 5] = y5[:, 10:].transpose(0, 1)
        inv_freq = 1.0 / (1e4 ** (torch.arange(0, 128, 2, device=DEV, dtype=torch.float32) / 128))
        *_, ks, _, _, _ = R.rope(y[5 * b:5 * b + 5], 8, 2, 128, _i([0, 5]), _i([L]), inv_freq, _i([0, 1, 1, 2, 2]))
        want_k = R.rope(y[5 * b:5 * b + 5], 8, 2, 128, _i([0, 5]), _i([L]), inv_freq, _i([0, 1, 1, 2, 2]))[2]
        assert bool(((kk[b, :, L:L + 3].double().cpu() - want_k[[0, 2, 4]].transpose(0, 1)).abs()
                     <= 2.0 ** -8 * want_k[[0, 2, 4]].transpose(0, 1).abs() + 2e-6 * 10).all())
    R.check(a, *R.prompt(q, kk, vv, cu, 128 ** -0.5, len_k=len_k)[:2])
    # the tree read its own rows as they were written: again, from a cache that still has them
    k2, v2 = torch.zeros_like(kk), torch.zeros_like(vv)
    S.rope_cache_packed(x, 8, 2, 128, cu, _i([0] * 3), inv_freq, k2, v2)
    S.rope_cache_packed(y, 8, 2, 128, _i([0, 5, 10, 15]), len_k, inv_freq, k2, v2,
                        depth=_i([0, 1, 1, 2, 2] * 3))
    R.check(t, *R.tree(tq.view(3, 5, 8, 128), k2, v2, lens, mask, 128 ** -0.5))


def test_the_same_bits_each_time_on_any_stream_and_in_a_graph():
    S, g = _ops(), _gen(15)
    run, state = _pass(S, g, [70, 129, 2])
    first = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        held2 = run()
    for _ in range(2):
        for t in (*held, *held2):
            t.zero_()
        graph.replay()
        graph2.replay()
    for a, b, c in zip(first, held, held2):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_a_captured_step_follows_the_lengths_on_the_device():
    S, g = _ops(), _gen(16)
    q = _n(g, 1, 4, 8, 128)
    k, v = _n(g, 1, 2, 3000, 128), _n(g, 1, 2, 3000, 128)
    pos = _i([5])
    mask, _ = S.tree_mask([-1, 0, 1, 1], DEV)
    S.tree_attention(q, k, v, pos, mask, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = S.tree_attention(q, k, v, pos, mask, 0.1)
    for p in (0, 5, 900, 2996):
        pos.fill_(p)
        graph.replay()
        R.check(out, *R.tree(q, k, v, [p], mask, 0.1))


def test_two_streams_at_once():
    S, g = _ops(), _gen(17)
    q, k, v = _n(g, 1, 8, 8, 128), _n(g, 1, 2, 20000, 128), _n(g, 1, 2, 20000, 128)
    mask, _ = S.tree_mask([-1, 0, 0, 1, 1, 2, 2, 3], DEV)
    pos = [_i([19000]), _i([7000])]
    want = [S.tree_attention(q, k, v, p, mask, 0.1).clone() for p in pos]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(S.tree_attention(q, k, v, pos[i], mask, 0.1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    assert int(_status()) == 0


def _status():
    from afterimage_b200.runtime import _device
    return _device.status_word(torch.device("cuda", torch.cuda.current_device())).item()


def test_empty_calls():
    S = _ops()
    e = torch.zeros(0, 4, 64, dtype=BF, device=DEV)
    assert S.prompt_attention(e, e[:, :2], e[:, :2], _i([0]), 1.0).shape == (0, 4, 64)
    assert S.prompt_attention(e, e[:, :2], e[:, :2], _i([0, 0]), 1.0).shape == (0, 4, 64)
    q = torch.zeros(2, 0, 4, 64, dtype=BF, device=DEV)
    c = torch.zeros(2, 2, 8, 64, dtype=BF, device=DEV)
    assert S.tree_attention(q, c, c, _i([1, 1]), torch.zeros(0, 0, dtype=torch.bool, device=DEV), 1.0).shape == q.shape
    S.keep_cache_rows([c], _i([0, 0]), torch.zeros(2, 0, dtype=torch.int64, device=DEV))
