"""GPU parity of the sequence operators (node embedding, packed attention, linear cross entropy)
against plain float64 forms, at the sizes, layouts and masks where they can go wrong.  The
tolerances are sums of rounding errors (tests/sequence_ref.py)."""
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


# ------------------------------------------------------------------------------------ embedding
@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("n,rows,dim", [(1, 1, 1), (1, 300, 64), (7, 5, 3), (63, 1000, 41), (4096, 41, 100),
                                        (4097, 70000, 8), (5000, 257, 129), (20000, 3, 16), (300, 200000, 24),
                                        (70001, 2708, 33)])
def test_embedding(n, rows, dim, dtype):
    gen = torch.Generator().manual_seed(n * 7 + dim)
    ids = (torch.rand(n, generator=gen, dtype=torch.float64) ** 3 * (rows + 1)).long() - (torch.arange(n) % 5 == 3).long()
    ids[0] = rows - 1
    ids[n // 2:n // 2 + 1] = rows if n > 2 else rows - 1             # one behind the last row: names none
    table = torch.randn(rows, dim, generator=gen).to(dtype)
    grad = torch.randn(n, dim, generator=gen).to(dtype)
    scale = 1.7
    good = (ids >= 0) & (ids < rows)
    at = ids.clamp(0, rows - 1)
    want = (table[at].float() * torch.tensor(scale)) * good[:, None]
    gsum = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, at[good], grad[good].double()) * scale
    mass = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, at[good], grad[good].double().abs()) * scale
    most = int(torch.bincount(at[good], minlength=1).max()) if bool(good.any()) else 0
    bound = (most + 4) * ref.U * mass + ref.half_step(dtype) * gsum.abs() * (1 + 1e-6) + ref.tiny(dtype)
    results = []
    for wide in (torch.int64, torch.int32):
        t = table.to(DEV).requires_grad_()
        out = NodeEmbeddingFuse(ids.to(DEV, wide), t, scale)
        assert torch.equal(out.detach().cpu(), want.to(dtype))
        out.backward(grad.to(DEV))
        ref.check(t.grad, (gsum, bound), f"grad_table {wide}")
        results.append(t.grad.clone())
    assert torch.equal(results[0], results[1])                       # the same bits, whatever the id type


def test_embedding_shapes_empty_and_unaligned():
    table = torch.randn(50, 12, device=DEV)
    ids = torch.randint(0, 50, (3, 4, 5), device=DEV)
    t = table.clone().requires_grad_()
    out = NodeEmbeddingFuse(ids, t)
    assert out.shape == (3, 4, 5, 12) and torch.equal(out, table[ids])
    out.sum().backward()
    assert torch.equal(t.grad, torch.bincount(ids.flatten(), minlength=50).float()[:, None].expand(50, 12))
    for ids in (torch.empty(0, dtype=torch.int64, device=DEV), torch.full((9,), -1, device=DEV),
                torch.full((9,), 1 << 40, device=DEV)):
        t = table.clone().requires_grad_()
        out = NodeEmbeddingFuse(ids, t)
        assert out.shape == (ids.numel(), 12) and not out.any()
        out.sum().backward()
        assert not t.grad.any()
    # rows that start off 16 bytes: a view behind one element
    for dtype in DTYPES:
        flat = torch.randn(50 * 16 + 1, device=DEV).to(dtype)
        view = flat[1:].view(50, 16)
        ids = torch.randint(0, 50, (77,), device=DEV)
        assert torch.equal(NodeEmbeddingFuse(ids, view), view[ids])
        # a transposed table and ids with a stride are taken as values
        wide = torch.randn(16, 50, device=DEV).to(dtype)
        assert torch.equal(NodeEmbeddingFuse(ids[::2], wide.t()), wide.t()[ids[::2]])


# ------------------------------------------------------------------------------------ attention
def offsets(lens, front=0):
    off = [front]
    for n in lens:
        off.append(off[-1] + n)
    return off


def attention_case(lq, lk, hq, hk, d, causal, dtype, seed=0, front=0, back=0, scale=None, layout="split",
                   poison=False, grads=True):
    gen = torch.Generator().manual_seed(seed + 1000 * d + sum(lk))
    q_off, k_off = offsets(lq, front), offsets(lk, front)
    tq, tk = q_off[-1] + back, k_off[-1] + back
    same = lq is lk

    def make(t, h):
        return torch.randn(t, h, d, generator=gen).to(dtype)

    q, k, v, grad = make(tq, hq), make(tk, hk), make(tk, hk), make(tq, hq)
    scale = d ** -0.5 if scale is None else scale
    want = ref.attention(q, k, v, q_off, k_off, causal, scale, grad if grads else None)
    if poison:                                            # rows of no sequence hold anything
        for t, off in ((q, q_off), (k, k_off), (v, k_off), (grad, q_off)):
            t[:off[0]] = float("nan")
            t[off[-1]:] = float("inf")
    if layout == "packed" and same:                       # slices of one projection
        qkv = torch.cat([q, k, v], 1).to(DEV)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    elif layout == "heads":                               # head major
        q, k, v = (t.transpose(0, 1).contiguous().to(DEV).transpose(0, 1) for t in (q, k, v))
    elif layout == "last":                                # the last dimension has a stride
        q, k, v = (t.permute(2, 0, 1).contiguous().to(DEV).permute(1, 2, 0) for t in (q, k, v))
    elif layout == "offset":                              # rows off 16 bytes
        q, k, v = (torch.cat([torch.zeros(1, dtype=dtype), t.flatten()]).to(DEV)[1:].view(t.shape) for t in (q, k, v))
    else:
        q, k, v = (t.to(DEV) for t in (q, k, v))
    row_ptr = torch.tensor(q_off, dtype=torch.int32, device=DEV)
    col_ptr = None if same else torch.tensor(k_off, dtype=torch.int32, device=DEV)
    leaves = [t.detach().requires_grad_(grads) for t in (q, k, v)]
    out = PackedAttentionFuse(*leaves, row_ptr, col_ptr, causal=causal, scale=scale)
    assert out.dtype == dtype and out.is_contiguous()
    ref.check(out, want["out"], "out")
    if grads:
        got = torch.autograd.grad(out, leaves, grad.to(DEV))
        again = torch.autograd.grad(PackedAttentionFuse(*leaves, row_ptr, col_ptr, causal=causal, scale=scale), leaves,
                                    grad.to(DEV))
        for name, x, y in zip(("dq", "dk", "dv"), got, again):
            ref.check(x, want[name], name)
            assert torch.equal(x, y), f"{name} differs from run to run"


SELF = [[1], [2], [31], [64, 1], [65, 0, 33], [0, 0, 1, 0], [5, 0, 128, 127, 129, 1], [300, 7]]


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("lens", SELF, ids=str)
def test_attention_lengths(lens, causal, dtype):
    attention_case(lens, lens, 4, 2, 64, causal, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("d", [1, 3, 8, 16, 24, 32, 33, 41, 63, 64, 72, 96, 100, 120, 127, 128])
def test_attention_head_dims(d, dtype):
    attention_case([70, 1, 33], [70, 1, 33], 2, 1, d, d % 2 == 0, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 3), (3, 1), (6, 2), (8, 1), (40, 1), (10, 2), (16, 8)])
def test_attention_heads(hq, hk, dtype):
    lens = [45, 20, 131]
    attention_case(lens, lens, hq, hk, 32, True, dtype)
    attention_case(lens, lens, hq, hk, 32, False, dtype, seed=1)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
def test_attention_queries_and_keys_of_different_lengths(causal, dtype):
    """Single queries, rows that see nothing (more queries than keys), sequences without either."""
    for lq, lk in (([1] * 6, [1, 2, 64, 65, 300, 1000]), ([9, 40, 0, 5, 1], [3, 1, 17, 0, 129]),
                   ([150, 3], [20, 500]), ([1], [2500]), ([200], [1])):
        attention_case(lq, lk, 8, 2, 64, causal, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("layout", ["packed", "heads", "last", "offset"])
@pytest.mark.parametrize("d", [64, 41])
def test_attention_layouts(layout, d, dtype):
    lens = [70, 1, 200]
    attention_case(lens, lens, 4, 2, d, True, dtype, layout=layout)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("layout", ["heads", "last", "offset"])
@pytest.mark.parametrize("d", [32, 64, 108])
def test_attention_layouts_of_split_keys(layout, d, dtype):
    """The same where the keys are split: single queries and few tiles of rows."""
    attention_case([1, 2, 0], [600, 257, 300], 4, 2, d, True, dtype, layout=layout)
    attention_case([100, 40], [2100, 900], 4, 2, d, True, dtype, layout=layout)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
def test_attention_rows_of_no_sequence(causal, dtype):
    """Padding in front and behind: never read (it holds NaN and infinities), zeros come back."""
    lens = [33, 0, 90]
    attention_case(lens, lens, 4, 4, 64, causal, dtype, front=37, back=150, poison=True)
    attention_case([3, 1], [70, 5], 4, 1, 128, causal, dtype, front=2, back=3, poison=True)
    attention_case([], [], 2, 1, 32, causal, dtype, back=5, poison=True)         # no sequence at all


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
def test_attention_scales(dtype):
    lens = [100, 29]
    for scale in (0.0, -0.2, 0.5):
        attention_case(lens, lens, 2, 2, 32, True, dtype, scale=scale)


def test_attention_broadcast_inputs_and_gradients():
    """Expanded keys, values and gradients (strides of zero): values as if they had been copied."""
    for dtype in DTYPES:
        ptr = torch.tensor([0, 40, 70], dtype=torch.int32, device=DEV)
        q = torch.randn(70, 4, 64, device=DEV).to(dtype).requires_grad_()
        one = torch.randn(70, 1, 64, device=DEV).to(dtype).requires_grad_()          # one key head for all
        row = torch.randn(1, 4, 64, device=DEV).to(dtype).requires_grad_()           # one value row for all
        out = PackedAttentionFuse(q, one.expand(70, 4, 64), row.expand(70, 4, 64), ptr, causal=True)
        got = torch.autograd.grad(out.sum(), [q, one, row])
        q2, k2, v2 = (t.detach().clone().requires_grad_() for t in (q, one.expand(70, 4, 64), row.expand(70, 4, 64)))
        out2 = PackedAttentionFuse(q2, k2.contiguous(), v2.contiguous(), ptr, causal=True)
        want = torch.autograd.grad(out2, [q2, k2, v2], torch.ones_like(out2))
        assert torch.equal(out, out2) and torch.equal(got[0], want[0])
        assert torch.equal(got[1], want[1].sum(1, keepdim=True)) and torch.equal(got[2], want[2].sum(0, keepdim=True))


def test_second_derivatives_are_refused():
    ptr = torch.tensor([0, 8], dtype=torch.int32, device=DEV)
    q = torch.randn(8, 1, 16, device=DEV, requires_grad=True)
    out = PackedAttentionFuse(q, q, q, ptr)
    for loss in (out.sum(), out.pow(2).sum()):            # the gradient of out constant, and with a graph of its own
        g, = torch.autograd.grad(loss, [q], create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), [q])


def test_attention_nan_stays_in_its_sequence():
    for dtype in DTYPES:
        q, k, v = (torch.randn(200, 2, 64, device=DEV).to(dtype) for _ in range(3))
        ptr = torch.tensor([0, 70, 131, 200], dtype=torch.int32, device=DEV)
        clean = PackedAttentionFuse(q, k, v, ptr)
        for t in (q, k, v):
            bad = [x.clone() for x in (q, k, v)]
            bad[[x is t for x in (q, k, v)].index(True)][70:131] = float("nan")
            leaves = [x.requires_grad_() for x in bad]
            out = PackedAttentionFuse(*leaves, ptr)
            assert torch.equal(out[:70], clean[:70]) and torch.equal(out[131:], clean[131:])
            assert torch.isnan(out[70:131]).all()
            for g in torch.autograd.grad(out, leaves, torch.ones_like(out)):
                assert torch.isfinite(g[:70]).all() and torch.isfinite(g[131:]).all()
    # a key or value far in the future of a causal row is not seen by it
    q, k, v = (torch.randn(400, 2, 64, device=DEV) for _ in range(3))
    ptr = torch.tensor([0, 400], dtype=torch.int32, device=DEV)
    clean = PackedAttentionFuse(q, k, v, ptr, causal=True)
    k[399], v[399] = float("inf"), float("nan")
    assert torch.equal(PackedAttentionFuse(q, k, v, ptr, causal=True)[:256], clean[:256])


def test_attention_large_scores_and_long_rows():
    """Scores of +-300 (the running maximum moves), 5000 keys."""
    for dtype in DTYPES:
        gen = torch.Generator().manual_seed(3)
        q, k, v = (torch.randn(600, 1, 64, generator=gen) for _ in range(3))
        q, k, v = (t.to(dtype) for t in (q * 6, k * 6, v))
        ptr = torch.tensor([0, 600], dtype=torch.int32, device=DEV)
        want = ref.attention(q, k, v, [0, 600], [0, 600], True, 1.0)
        ref.check(PackedAttentionFuse(q.to(DEV), k.to(DEV), v.to(DEV), ptr, causal=True, scale=1.0), want["out"], "out")
    attention_case([40], [5000], 4, 1, 128, True, torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("hq,hk,d", [(1, 1, 32), (6, 2, 64), (4, 1, 128)])
def test_attention_long_rows_split_backward(hq, hk, d, causal, dtype):
    """Long sequences, few key tiles: the queries of a key tile are split and joined."""
    attention_case([1100, 0, 901], [1100, 0, 901], hq, hk, d, causal, dtype, back=5, poison=True)
    attention_case([1500], [333], hq, hk, d, causal, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("hq,hk,d", [(1, 1, 32), (8, 2, 64), (16, 1, 128), (6, 2, 41)])
def test_attention_few_rows_long_keys(hq, hk, d, causal, dtype):
    """Rows split over chunks of the keys: ragged keys, some sequences with many rows, with none, without
    keys, padding in front and behind."""
    attention_case([1] * 7, [300, 1, 700, 0, 257, 256, 1500], hq, hk, d, causal, dtype, front=3, back=2, poison=True)
    attention_case([2, 0, 70, 1, 3], [1000, 600, 900, 0, 513], hq, hk, d, causal, dtype)
    attention_case([1], [4000], hq, hk, d, causal, dtype)


@pytest.mark.parametrize("scale", [None, -0.3, 0.0], ids=["scale", "negative", "zero"])
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("hq,hk,d", [(4, 1, 128), (6, 3, 100), (3, 3, 64), (8, 2, 33), (4, 4, 20)])
def test_attention_four_rows_of_floats(hq, hk, d, causal, scale):
    """The split forward of at most four rows a sequence on average: fewer rows, more rows, none, ragged keys."""
    lq, lk = [1, 1, 0, 1, 1, 1, 1], [300, 31, 257, 0, 2049, 1, 1000]
    attention_case(lq, lk, hq, hk, d, causal, torch.float32, front=1, back=3, poison=True, scale=scale, grads=False)
    if hq == hk:
        attention_case([9, 0, 1, 2], [700, 512, 640, 5], hq, hk, d, causal, torch.float32, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("rows,keys", [(128, 128), (64, 64), (32, 32), (1, 256), (1, 512)])
def test_attention_equal_lengths(rows, keys, dtype):
    """Spare tile slots at a fixed period, which are dealt out in an order of their own."""
    attention_case([rows] * 71, [keys] * 71, 2, 1, 32, rows == 64, dtype, back=5)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("hq,hk,d", [(1, 1, 32), (6, 2, 64), (4, 1, 128), (3, 3, 41)])
def test_attention_few_tiles_long_keys(hq, hk, d, causal, dtype):
    """Tiles of rows whose keys are split and joined: ragged, no rows, fewer keys than rows, no keys."""
    attention_case([140, 0, 300, 7, 90], [3000, 700, 1501, 5000, 40], hq, hk, d, causal, dtype, front=2, back=70, poison=True)
    attention_case([1200, 33], [1200, 0], hq, hk, d, causal, dtype)
    attention_case([70], [4097], hq, hk, d, causal, dtype, scale=-0.2, grads=False)


def test_attention_many_small_graphs():
    lens = [(i * 7) % 40 for i in range(700)]
    attention_case(lens, lens, 1, 1, 32, False, torch.float32)
    attention_case(lens, lens, 1, 1, 32, True, torch.bfloat16)


# ------------------------------------------------------------------------------------ cross entropy
def ce_case(n, classes, dim, dtype, reduction="mean", ignored=0.2, wide=True, seed=0, spread=2.0):
    gen = torch.Generator().manual_seed(seed + n + classes)
    feat = torch.randn(n, dim, generator=gen).to(dtype)
    weight = (torch.randn(classes, dim, generator=gen) * spread / math.sqrt(dim)).to(dtype)
    label = torch.randint(0, classes, (n,), generator=gen)
    drop = torch.rand(n, generator=gen) < ignored
    label[drop] = -100
    if n > 3 and ignored:
        label[1], label[2] = classes, -7                   # outside: no label either
    label = label if wide else label.int()
    grad = torch.rand(n, generator=gen) + 0.5 if reduction == "none" else torch.tensor(1.5)
    want = ref.linear_ce(feat, weight, label, -100, reduction, grad)
    clean = feat.clone()
    feat[(label < 0) | (label >= classes)] = float("nan")  # rows without a label are never read
    x, w = feat.to(DEV).requires_grad_(), weight.to(DEV).requires_grad_()
    loss = LinearCrossEntropyFuse(x, w, label.to(DEV), reduction=reduction)
    assert loss.dtype == torch.float32 and clean.shape == feat.shape
    ref.check(loss, want["loss"], "loss")
    got = torch.autograd.grad(loss, [x, w], grad.to(DEV))
    again = torch.autograd.grad(LinearCrossEntropyFuse(x, w, label.to(DEV), reduction=reduction), [x, w], grad.to(DEV))
    for name, a, b in zip(("dx", "dw"), got, again):
        ref.check(a, want[name], name)
        assert torch.equal(a, b), f"{name} differs from run to run"


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("n,classes,dim", [(1, 1, 1), (1, 1000, 64), (3, 2, 5), (64, 41, 64), (129, 127, 128),
                                           (130, 129, 33), (257, 1000, 100), (500, 4099, 24), (33, 20011, 65),
                                           (2500, 47, 16), (600, 130, 500)])
def test_cross_entropy(n, classes, dim, dtype):
    ce_case(n, classes, dim, dtype)
    ce_case(n, classes, dim, dtype, reduction="none", wide=False, seed=1)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
def test_cross_entropy_reductions_and_masks(dtype):
    for reduction in ("none", "mean", "sum"):
        for ignored in (0.0, 0.9, 1.0):
            ce_case(300, 200, 40, dtype, reduction=reduction, ignored=ignored)
    ce_case(200, 300, 64, dtype, spread=60.0)              # logits of some hundred


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("n,classes,dim", [(4100, 4300, 72), (8200, 8210, 520), (5000, 20000, 264), (900, 70000, 136)])
def test_cross_entropy_large_tiles_and_pieces(n, classes, dim, dtype):
    """Enough tiles for the wide shapes, several pieces of the classes, split sums (reference in
    float64 on the GPU)."""
    gen = torch.Generator(device=DEV).manual_seed(n)
    feat = torch.randn(n, dim, generator=gen, device=DEV).to(dtype)
    weight = (torch.randn(classes, dim, generator=gen, device=DEV) * 2 / math.sqrt(dim)).to(dtype)
    label = torch.randint(-classes // 20, classes, (n,), generator=gen, device=DEV)
    grad = torch.tensor(1.5, device=DEV)
    with torch.device(DEV):
        want = ref.linear_ce(feat, weight, label, -100, "mean", grad)
    x, w = feat.requires_grad_(), weight.requires_grad_()
    loss = LinearCrossEntropyFuse(x, w, label)
    ref.check(loss, want["loss"], "loss")
    for name, got in zip(("dx", "dw"), torch.autograd.grad(loss, [x, w], grad)):
        ref.check(got, want[name], name)


def test_cross_entropy_only_one_gradient_and_no_rows():
    feat, weight = torch.randn(40, 16, device=DEV), torch.randn(30, 16, device=DEV)
    label = torch.randint(0, 30, (40,), device=DEV)
    full = [t.clone().requires_grad_() for t in (feat, weight)]
    LinearCrossEntropyFuse(*full, label).backward()
    x = feat.clone().requires_grad_()
    LinearCrossEntropyFuse(x, weight, label).backward()
    w = weight.clone().requires_grad_()
    LinearCrossEntropyFuse(feat, w, label).backward()
    assert torch.equal(x.grad, full[0].grad) and torch.equal(w.grad, full[1].grad)
    for reduction in ("none", "mean", "sum"):
        x, w = feat[:0].clone().requires_grad_(), weight.clone().requires_grad_()
        loss = LinearCrossEntropyFuse(x, w, label[:0], reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and not loss.any()
        loss.sum().backward()
        assert not w.grad.any() and x.grad.shape == (0, 16)


# ------------------------------------------------------------------------------------ beyond 32 bits
def test_offsets_past_32_bits():
    """Tables, caches and weights of more than 2^31 elements: the last rows are where they should be."""
    rows, dim = 34_000_000, 64
    table = torch.zeros(rows, dim, dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([0, 1, 33_554_431, 33_554_432, rows - 1], device=DEV)
    table[at] = torch.randn(5, dim, device=DEV).bfloat16()
    assert torch.equal(NodeEmbeddingFuse(at, table), table[at])
    x = torch.randn(40, dim, device=DEV).bfloat16()
    label = at.repeat(8)
    w = table.requires_grad_()
    loss = LinearCrossEntropyFuse(x, w, label, reduction="none")
    z = x.double() @ table.detach()[at].double().t()
    total = torch.exp(z).sum(1) + (rows - 5)                      # every other row scores 0
    want = torch.log(total) - z.gather(1, torch.arange(5, device=DEV).repeat(8).unsqueeze(1))[:, 0]
    assert (loss.double() - want).abs().max() < 1e-4              # 2^-24 times a sum of 266 k tile terms at most
    g, = torch.autograd.grad(loss.sum(), w)
    dw = (torch.softmax(torch.cat([z, torch.log(torch.full_like(total, rows - 5.0)).unsqueeze(1)], 1), 1)[:, :5]
          - torch.eye(5, device=DEV, dtype=torch.float64).repeat(8, 1)).t() @ x.double()
    mass = x.double().abs().sum(0)                                # |dz| <= 1, one rounding of dz and one of dw
    assert ((g[at].double() - dw).abs() <= 2 ** -8 * (mass + dw.abs())).all()
    del g, w, loss
    t = table.detach().requires_grad_()
    go = torch.randn(5, dim, device=DEV).bfloat16()
    g, = torch.autograd.grad(NodeEmbeddingFuse(at, t), [t], go)
    assert torch.equal(g[at], go) and int((g != 0).any(1).sum()) == 5
    del g, t, table
    # a cache of 1.1 M tokens, 16 heads of 128: one query for each of three sequences, and a prompt at its end
    tk, h, d = 1_100_000, 16, 128
    k, v = (torch.randn(tk, h, d, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    ptr = torch.tensor([0, 300, tk - 700, tk], dtype=torch.int32, device=DEV)
    for lq, causal in (([1, 1, 1], False), ([0, 0, 200], True)):
        off = offsets(lq)
        q = torch.randn(off[-1], h, d, device=DEV, dtype=torch.bfloat16)
        out = PackedAttentionFuse(q, k, v, torch.tensor(off, dtype=torch.int32, device=DEV), ptr, causal=causal)
        for s in (0, 2):
            if lq[s] == 0:
                continue
            a, b = [0, 300, tk - 700, tk][s:s + 2]
            n = b - a
            want = ref.attention(q[off[s]:off[s + 1]].cpu(), k[a:b].cpu(), v[a:b].cpu(), [0, lq[s]], [0, n], causal, d ** -0.5)
            ref.check(out[off[s]:off[s + 1]], want["out"], f"sequence {s}")


# ------------------------------------------------------------------------------------ together
def model(params, ids, ptr, label, heads, kv_heads, dim):
    """Nodes -> embedding -> one attention layer with a residual -> scores against all nodes (tied table)."""
    x = NodeEmbeddingFuse(ids, params["table"], math.sqrt(params["table"].size(1)))
    qkv = (x @ params["qkv"]).view(-1, heads + 2 * kv_heads, dim)
    o = PackedAttentionFuse(qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], ptr, causal=True)
    x = x + o.flatten(1) @ params["out"]
    return LinearCrossEntropyFuse(x, params["table"], label)


def model64(params, ids, off, label, heads, kv_heads, dim):
    table = params["table"]
    good = ids >= 0
    x = table[ids.clamp(min=0)] * good[:, None] * math.sqrt(table.size(1))
    qkv = (x @ params["qkv"]).view(-1, heads + 2 * kv_heads, dim)
    outs = []
    for a, b in zip(off[:-1], off[1:]):
        q, k, v = (t.transpose(0, 1) for t in (qkv[a:b, :heads], qkv[a:b, heads:heads + kv_heads], qkv[a:b, heads + kv_heads:]))
        k, v = (t.repeat_interleave(heads // kv_heads, 0) for t in (k, v))
        z = q @ k.transpose(1, 2) * dim ** -0.5
        z = z.masked_fill(torch.ones(b - a, b - a).triu(1).bool(), float("-inf"))
        outs.append((torch.softmax(z, -1) @ v).transpose(0, 1))
    x = x + torch.cat(outs + [torch.zeros(len(ids) - off[-1], heads, dim, dtype=x.dtype)]).flatten(1) @ params["out"]
    kept = label >= 0
    return torch.nn.functional.cross_entropy(x[kept] @ table.t(), label[kept])


def test_a_training_step_of_the_three_together():
    """Value and gradients of embedding + attention + loss on tied weights against float64 autograd:
    float32 throughout, so a relative 1e-4 of each gradient's own norm covers sums of at most 400 terms
    through four chained products (4 * 400 * 2^-24 = 1e-4)."""
    heads, kv_heads, dim, width, nodes = 4, 2, 16, 48, 300
    lens = [50, 1, 133, 0, 64]
    off = offsets(lens)
    n = off[-1] + 9
    gen = torch.Generator().manual_seed(0)
    p64 = dict(table=torch.randn(nodes, width, generator=gen).double() * 0.2,
               qkv=torch.randn(width, (heads + 2 * kv_heads) * dim, generator=gen).double() / math.sqrt(width),
               out=torch.randn(heads * dim, width, generator=gen).double() / 8)
    p64 = {k: v.float().double().requires_grad_() for k, v in p64.items()}
    ids = torch.randint(0, nodes, (n,), generator=gen)
    label = torch.randint(0, nodes, (n,), generator=gen)
    ids[off[-1]:], label[off[-1]:] = -1, -100
    label[::7] = -100
    want = model64(p64, ids, off, label, heads, kv_heads, dim)
    want.backward()
    params = {k: v.detach().float().to(DEV).requires_grad_() for k, v in p64.items()}
    ptr = torch.tensor(off, dtype=torch.int32, device=DEV)
    loss = model(params, ids.to(DEV), ptr, label.to(DEV), heads, kv_heads, dim)
    loss.backward()
    assert abs(loss.item() - want.item()) <= 1e-4 * abs(want.item())
    for name in params:
        a, b = params[name].grad.cpu().double(), p64[name].grad
        assert (a - b).norm() <= 1e-4 * b.norm(), name


def test_replayed_from_a_graph():
    """Forward and backward of the three captured once and replayed with new inputs in between."""
    heads, kv_heads, dim, width, nodes = 2, 1, 32, 64, 500
    off = offsets([90, 3, 200])
    gen = torch.Generator(device=DEV).manual_seed(5)
    params = dict(table=torch.randn(nodes, width, device=DEV, generator=gen),
                  qkv=torch.randn(width, (heads + 2 * kv_heads) * dim, device=DEV, generator=gen) / 8,
                  out=torch.randn(heads * dim, width, device=DEV, generator=gen) / 8)
    params = {k: v.to(torch.bfloat16).requires_grad_() for k, v in params.items()}
    ids = torch.randint(0, nodes, (off[-1],), device=DEV, generator=gen)
    label = torch.randint(0, nodes, (off[-1],), device=DEV, generator=gen)
    ptr = torch.tensor(off, dtype=torch.int32, device=DEV)

    def step():
        loss = model(params, ids, ptr, label, heads, kv_heads, dim)
        return [loss.detach()] + list(torch.autograd.grad(loss, list(params.values())))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i in range(4):
        ids.copy_(torch.randint(0, nodes, ids.shape, device=DEV, generator=gen))
        label.copy_(torch.randint(-20, nodes, ids.shape, device=DEV, generator=gen))
        ptr.copy_(torch.tensor(offsets([90 - 20 * i, 3 + i, 150]), dtype=torch.int32))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(static, want):
            assert torch.equal(a, b)


def test_on_a_side_stream():
    """Calls run on the caller's current stream: inputs made there, with the default stream busy elsewhere."""
    lens = [100, 50]
    ptr = torch.tensor(offsets(lens), dtype=torch.int32, device=DEV)
    q = torch.randn(150, 2, 64, device=DEV)
    label = torch.randint(0, 77, (150,), device=DEV)
    w = torch.randn(77, 128, device=DEV)
    table = torch.randn(20, 64, device=DEV)
    ids = torch.randint(0, 20, (150,), device=DEV)
    torch.cuda.synchronize()

    def work(x):
        y = PackedAttentionFuse(x, x, x, ptr)
        return y, LinearCrossEntropyFuse(y.flatten(1), w, label, reduction="none"), NodeEmbeddingFuse(ids, table * x[0, 0, 0])

    want = work(q * 2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = work(q * 2)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_two_graphs_replayed_at_the_same_time():
    """Two captured calls of each kind, replayed on two streams: neither finds the other's workspace."""
    gen = torch.Generator(device=DEV).manual_seed(9)
    ptr = torch.tensor(offsets([400, 700, 0, 900]), dtype=torch.int32, device=DEV)
    rows, nodes = 2000, 5000

    def inputs():
        x = torch.randn(rows, 6, 64, device=DEV, generator=gen).to(torch.bfloat16)
        w = (torch.randn(nodes, 128, device=DEV, generator=gen) / 8).to(torch.bfloat16)
        ids = torch.randint(0, nodes, (20000,), device=DEV, generator=gen)
        return [x.requires_grad_(), w.requires_grad_(), ids, torch.randint(-9, nodes, (rows,), device=DEV, generator=gen)]

    def step(x, w, ids, label):
        y = PackedAttentionFuse(x[:, :2], x[:, 2:4], x[:, 4:], ptr, causal=True)
        one = PackedAttentionFuse(x[:4, :2], x[:, 2:4], x[:, 4:], torch.arange(5, dtype=torch.int32, device=DEV), ptr)
        loss = LinearCrossEntropyFuse(y.flatten(1), w, label) + NodeEmbeddingFuse(ids, w, 0.5).float().mean() + one.float().mean()
        return [loss.detach()] + list(torch.autograd.grad(loss, [x, w]))

    both, graphs, static, want = [inputs(), inputs()], [], [], []
    for args in both:
        want.append([t.clone() for t in step(*args)])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*args)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            static.append(step(*args))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for got, ref_ in zip(static, want):
            for a, b in zip(got, ref_):
                assert torch.equal(a, b)
