"""Digits of the sequence operators where the tolerances of test_gpu_sequence_ops.py leave room for their loss: small
and large gradients in float16, confident rows of the loss, long runs of one id, and what masked rows hold."""
import math

import pytest
import torch

import sequence_ref as ref
from dgnn_amd.operators import LinearCrossEntropyFuse, NodeEmbeddingFuse, PackedAttentionFuse

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = "cuda:0"


def ids_of(x):
    return str(x).replace("torch.", "")


def offsets(lens):
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    return off


# ------------------------------------------------------------------------------------ float16 attention
@pytest.mark.parametrize("size", [2.0 ** -18, 2.0 ** -13, 1.0, 2.0 ** 11], ids=["2^-18", "2^-13", "1", "2^11"])
@pytest.mark.parametrize("lq,lk,hq,hk,d,causal", [([4173], [4173], 1, 1, 64, False), ([2000, 31], [2000, 31], 2, 1, 32, True),
                                                  ([3, 1], [8192, 700], 2, 1, 128, False), ([60, 2, 33, 1], [60, 2, 33, 1], 4, 4, 64, False),
                                                  ([300, 40], [900, 1500], 4, 2, 128, True)], ids=str)
def test_float16_gradients_keep_their_digits(lq, lk, hq, hk, d, causal, size, monkeypatch):
    """The bounds without an allowance of the type's smallest step for every pair of a row and a key: p and ds may be off
    by half a step of their own size, whatever the size of the incoming gradient, and only the results by the
    type's smallest.  Values equal the keys, so that dq is about scale * grad however many keys there are."""
    gen = torch.Generator().manual_seed(7)
    q_off, k_off = offsets(lq), offsets(lk)
    k = torch.randn(k_off[-1], hk, d, generator=gen).half()
    q = (torch.randn(q_off[-1], hq, d, generator=gen) * 0.25).half()
    grad = (torch.randn(q_off[-1], hq, d, generator=gen) * size).half()
    small = ref.tiny(torch.float16)
    monkeypatch.setattr(ref, "tiny", lambda dtype: 0.0)
    scale = 0.5
    want = ref.attention(q, k, k, q_off, k_off, causal, scale, grad)
    ptr = [torch.tensor(o, dtype=torch.int32, device=DEV) for o in (q_off, k_off)]
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, k)]
    out = PackedAttentionFuse(*leaves, *ptr, causal=causal, scale=scale)
    got = torch.autograd.grad(out, leaves, grad.to(DEV))
    for name, x in zip(("dq", "dk", "dv"), got):
        assert want[name][0].abs().max() < 60000                  # the results themselves have room
        ref.check(x, (want[name][0], want[name][1] + small), name)


def test_float16_gradients_of_large_terms():
    """Terms past the type's end, 2^17, whose sums times the scale are inside it."""
    gen = torch.Generator().manual_seed(8)
    lens, d, scale = [2, 1, 37, 100], 128, 2.0 ** -6
    off = offsets(lens)
    q, k, v, grad = (torch.randn(off[-1], 2, d, generator=gen) for _ in range(4))
    q, k, v, grad = (t.half() for t in (q, k, v * 16, grad * 2 ** 11))
    want = ref.attention(q, k, v, off, off, False, scale, grad)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out = PackedAttentionFuse(*leaves, torch.tensor(off, dtype=torch.int32, device=DEV), scale=scale)
    for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, grad.to(DEV))):
        assert want[name][0].abs().max() < 60000
        ref.check(x, want[name], name)


def test_float16_weights_far_below_the_largest():
    """One key 26 powers of two above 262143 others, in tiles of rows that see all keys in one pass.  Weights are kept in
    steps of 2^-24 at 2^7 for the largest, so each of the others may be off by 2^-32 of it."""
    rows, keys, d = 128 * 257, 1 << 18, 16
    q = torch.zeros(rows, 1, d, dtype=torch.float16, device=DEV)
    k = torch.zeros(keys, 1, d, dtype=torch.float16, device=DEV)
    v = torch.ones(keys, 1, d, dtype=torch.float16, device=DEV)
    q[:, :, 0], k[0, 0, 0], v[0] = 1, 18.015625, 0
    ptr = [torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (rows, keys)]
    out = PackedAttentionFuse(q, k, v, *ptr, scale=1.0).double()
    want = (keys - 1) / (keys - 1 + math.exp(18.015625))
    assert (out - want).abs().max() <= keys * 2.0 ** -32 + 2 * ref.half_step(torch.float16) * want


# ------------------------------------------------------------------------------------ rows that see no key
@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("lq,lk,hq,hk", [([100, 7], [40, 7], 4, 2), ([20, 3, 40], [5, 3, 0], 4, 4), ([9, 1, 1], [5, 1000, 700], 1, 1),
                                         ([40, 1], [5, 900], 4, 2), ([700, 200], [100, 9000], 2, 1), ([2000], [1500], 1, 1)], ids=str)
def test_rows_that_see_no_key(lq, lk, hq, hk, dtype):
    """Causal sequences with more rows than keys: the first rows give zeros and take no gradient although the keys and
    values hold NaN and infinities, and nothing they hold themselves reaches the other rows or the keys."""
    gen = torch.Generator().manual_seed(11)
    d, q_off, k_off = 64, offsets(lq), offsets(lk)
    q, k, v, grad = (torch.randn(t, h, d, generator=gen).to(dtype) for t, h in
                     ((q_off[-1], hq), (k_off[-1], hk), (k_off[-1], hk), (q_off[-1], hq)))
    blind = torch.zeros(q_off[-1], dtype=torch.bool)
    for s in range(len(lq)):
        blind[q_off[s]:q_off[s] + max(0, lq[s] - lk[s])] = True
    ptr = [torch.tensor(o, dtype=torch.int32, device=DEV) for o in (q_off, k_off)]

    def step(q, k, v, grad):
        leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
        out = PackedAttentionFuse(*leaves, *ptr, causal=True)
        return [out.detach().cpu()] + [t.cpu() for t in torch.autograd.grad(out, leaves, grad.to(DEV))]

    clean = step(q, k, v, grad)
    for t in (clean[0], clean[1]):
        assert not t[blind].any() and t[~blind].any()
    for what in (float("nan"), float("inf")):
        bad_q, bad_grad = q.clone(), grad.clone()
        bad_q[blind], bad_grad[blind] = what, what
        for a, b in zip(step(bad_q, k, v, bad_grad), clean):
            assert torch.equal(a, b)
        bad_k, bad_v = k.clone(), v.clone()
        bad_k[::3], bad_v[::2] = what, what
        out, dq, _, _ = step(q, bad_k, bad_v, grad)
        assert not out[blind].any() and not dq[blind].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("d", [1, 7, 64, 127])
@pytest.mark.parametrize("tq,tk", [(0, 0), (5, 0), (300, 0), (0, 5), (0, 700)])
def test_attention_without_rows_or_keys(tq, tk, d, dtype):
    """Tensors of no rows at all, at head dims that are padded elsewhere: zeros, and gradients of zero."""
    leaves = [torch.randn(t, h, d, device=DEV).to(dtype).requires_grad_() for t, h in ((tq, 4), (tk, 2), (tk, 2))]
    for row_off, col_off in (([0, tq], [0, tk]), ([0], [0]), ([0, 0, tq], [0, tk, tk])):
        ptr = [torch.tensor(o, dtype=torch.int32, device=DEV) for o in (row_off, col_off)]
        out = PackedAttentionFuse(*leaves, *ptr, causal=len(row_off) == 3)
        assert out.shape == (tq, 4, d) and not out.any()
        for g, leaf in zip(torch.autograd.grad(out, leaves, torch.ones_like(out)), leaves):
            assert g.shape == leaf.shape and not g.any()


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("singles,rows,keys,hq,hk", [(40, 600, 700, 2, 2), (9, 700, 600, 8, 2), (120, 300, 300, 1, 1)])
def test_attention_of_prompts_and_single_tokens(singles, rows, keys, hq, hk, dtype):
    """One call with both: whichever way the whole batch is worked on, every sequence is right."""
    gen = torch.Generator().manual_seed(singles)
    lq, lk = [1] * singles, [keys - 7 * (i % 30) for i in range(singles)]
    lq.insert(singles // 2, rows), lk.insert(singles // 2, keys)
    d, q_off, k_off = 32, offsets(lq), offsets(lk)
    q, k, v, grad = (torch.randn(t, h, d, generator=gen).to(dtype) for t, h in
                     ((q_off[-1], hq), (k_off[-1], hk), (k_off[-1], hk), (q_off[-1], hq)))
    want = ref.attention(q, k, v, q_off, k_off, True, d ** -0.5, grad)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out = PackedAttentionFuse(*leaves, *(torch.tensor(o, dtype=torch.int32, device=DEV) for o in (q_off, k_off)), causal=True)
    ref.check(out, want["out"], "out")
    for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, grad.to(DEV))):
        ref.check(x, want[name], name)


# ------------------------------------------------------------------------------------ loss
@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("top", [50.0, 400.0, -272.0])
@pytest.mark.parametrize("n,classes,dim", [(60, 41, 64), (33, 41, 33), (20, 3000, 64), (100, 1000, 128), (120, 1000, 129),
                                           (520, 33000, 528)], ids=str)
def test_loss_of_confident_rows(n, classes, dim, top, dtype):
    """The label's logit leads all others by 14, with logits of hundreds: the loss is (classes - 1) exp(-14) and the gradient
    of the label's logit about as small.  Logits are exact (one product each), so what is left is the sum of exp(z - top):
    one term of 1, at most 25 additions it takes part in (16 of a block, 4 blocks, 1 of the other half, 4 waves), the others
    2 * 14 + 8 roundings each."""
    lead = 14.0
    gen = torch.Generator().manual_seed(n)
    at = torch.randint(0, classes, (dim,), generator=gen)
    weight = torch.full((classes, dim), top - lead)
    weight[at, torch.arange(dim)] = top
    x, w = torch.eye(n, dim).to(DEV, dtype).requires_grad_(), weight.to(DEV, dtype).requires_grad_()
    assert torch.equal(w.detach().cpu().float(), weight)
    label = at[:n].to(DEV)
    loss = LinearCrossEntropyFuse(x, w, label, reduction="none")
    one = math.exp(-lead)
    rest = (classes - 1) * one
    want = math.log1p(rest)
    assert loss.min() >= 0
    assert (loss.double() - want).abs().max() <= (25 + (2 * lead + 8) * rest + want) * ref.U
    dw, = torch.autograd.grad(loss.sum(), w)
    e, t0 = ref.half_step(dtype), ref.tiny(dtype)
    dz = torch.full((classes, n), one / (1 + rest), dtype=torch.float64, device=DEV)
    bound = dz * ((25 + 2 * lead + 16) * ref.U + 2 * e) + t0
    pick = (label, torch.arange(n, device=DEV))
    dz[pick] = -rest / (1 + rest)
    bound[pick] = 32 * ref.U + 2 * e * rest + t0
    ref.check(dw[:, :n], (dz, bound), "dw")
    assert not dw[:, n:].any()


def test_loss_backward_refuses_half_of_the_log_sum():
    from dgnn_amd._lib import DgnnError
    from dgnn_amd.native import fused_cross_entropy as ext
    x, w = torch.randn(8, 16, device=DEV), torch.randn(5, 16, device=DEV)
    label, grad = torch.arange(8, device=DEV) % 5, torch.ones((), device=DEV)
    _, lse = ext.linear_ce_forward(x, w, label, -100, 1)
    assert lse.shape == (2, 8)
    for bad in (lse[0], lse[:1], lse[:, :4].contiguous()):
        with pytest.raises(DgnnError, match="lse"):
            ext.linear_ce_backward(x, w, label, -100, 1, bad, grad)


# ------------------------------------------------------------------------------------ embedding
def piece(n):
    """Sorted positions that one float sum runs over at most."""
    r = 64
    while 16 * r * r < n:
        r *= 2
    return r


@pytest.mark.parametrize("n,rows,dim", [(1 << 20, 1, 16), (1 << 20, 2, 6), (1 << 20, 3, 3), (400003, 1, 64), (70001, 1, 100), (9000, 2, 5)])
def test_embedding_gradient_of_long_runs(n, rows, dim):
    """One id named by all positions but a few, gradients of one value: every rounding goes the same way.  A quarter of a
    piece is added up in float, four waves are joined, the piece and the result are rounded: the number of pieces has no part in it."""
    ids = torch.zeros(n, dtype=torch.int64, device=DEV)
    ids[::997] = rows - 1
    table = torch.zeros(rows, dim, device=DEV, requires_grad=True)
    grad = torch.full((n, dim), 0.1, device=DEV)
    got, = torch.autograd.grad(NodeEmbeddingFuse(ids, table), [table], grad)
    want = torch.bincount(ids, minlength=rows).double()[:, None].expand(rows, dim) * grad[0, 0].double()
    # (the short runs of the last row may lie inside a piece: one wave adds them up)
    depth = torch.full((rows, 1), piece(n) / 4 + 8, dtype=torch.float64, device=DEV)
    depth[rows - 1] = max(depth[rows - 1], piece(n)) if rows > 1 else depth[rows - 1]
    ref.check(got, (want, depth * ref.U * want), "grad_table")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids_of)
@pytest.mark.parametrize("n,rows,dim", [(70001, 7, 33), (300000, 40, 8), (8193, 3, 129), (8192, 5, 20), (1 << 20, 1000, 4)])
def test_embedding_gradient_of_whole_numbers(n, rows, dim, dtype):
    """Whole numbers whose sums are exact: no term is dropped or taken twice in runs of any length."""
    gen = torch.Generator(device=DEV).manual_seed(n)
    ids = (torch.rand(n, device=DEV, generator=gen, dtype=torch.float64) ** 4 * (rows + 1)).long() - 1
    grad = torch.randint(-8, 9, (n, dim), device=DEV, generator=gen).to(dtype)
    table = torch.zeros(rows, dim, device=DEV, dtype=dtype, requires_grad=True)
    got, = torch.autograd.grad(NodeEmbeddingFuse(ids, table), [table], grad)
    good = ids >= 0
    want = torch.zeros(rows, dim, device=DEV, dtype=torch.float64).index_add_(0, ids[good], grad[good].double())
    assert torch.equal(got, want.to(dtype))


# ------------------------------------------------------------------------------------ forward mode
@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no_grad"])
def test_forward_mode_is_refused(grad):
    """A tangent is not dropped: none of the operators has a forward-mode derivative, and all say so."""
    import torch.autograd.forward_ad as fwd
    ptr = torch.tensor([0, 8], dtype=torch.int32, device=DEV)
    x, w, table = torch.randn(8, 2, 16, device=DEV), torch.randn(5, 16, device=DEV), torch.randn(9, 16, device=DEV)
    ids, label = torch.arange(8, device=DEV), torch.arange(8, device=DEV) % 5
    flat = x[:, 0].contiguous()
    calls = [lambda d: PackedAttentionFuse(d(x), x, x, ptr), lambda d: PackedAttentionFuse(x, d(x), x, ptr),
             lambda d: PackedAttentionFuse(x, x, d(x), ptr), lambda d: NodeEmbeddingFuse(ids, d(table)),
             lambda d: LinearCrossEntropyFuse(d(flat), w, label), lambda d: LinearCrossEntropyFuse(flat, d(w), label)]
    with torch.set_grad_enabled(grad), fwd.dual_level():
        for call in calls:
            with pytest.raises(NotImplementedError):
                call(lambda t: fwd.make_dual(t, torch.ones_like(t)))
            assert not call(lambda t: t).requires_grad            # inside a level, without a tangent
