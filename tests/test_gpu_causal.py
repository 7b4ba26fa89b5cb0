"""Rotary positions, attention over packed sequences and over a paged cache, on the GPU, against 64-bit definitions with
element-wise bounds (tests/causal_reference.py)."""
import math

import pytest
import torch

import causal_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
name = lambda t: str(t).split(".")[-1]  # noqa: E731


def rand(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


# ------------------------------------------------------------------------------------------------------------- packed
SHAPES = [(4, 4, 16), (4, 2, 64), (3, 1, 80), (8, 2, 128), (6, 2, 96), (12, 1, 32), (1, 1, 8), (5, 5, 72)]
LENGTHS = [
    ([1], None), ([0, 1, 0, 2], None), ([31, 32, 33], None), ([127, 128, 129, 65], None), ([300, 7, 511], None),
    ([5, 40, 0, 3], [70, 40, 9, 200]),             # new tokens of longer sequences; one of none
    ([50, 130, 9], [20, 129, 0]),                  # rows that see no key at all
]


# Few 128-row tiles are worked on 32 rows at a time, many 128: short sequences behind the tested ones make them many
MANY = [5] * 400


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("more", [[], MANY], ids=["few", "many"])
def test_packed_attention_and_gradient(dtype, shape, lengths, more):
    import transformer as M
    H, Hk, D = shape
    n, m = lengths[0], lengths[1] or lengths[0]
    rows, keys = sum(n), sum(m)
    g = gen(hash((H, Hk, D, sum(n), sum(m))) & 0xffff)
    pack = M.PackedSequences(n + more, DEV, None if lengths[1] is None else m + more)
    for causal in (True, False):
        q, k, v, do = (rand(g, r + sum(more), h, D, dtype=dtype) for r, h in ((rows, H), (keys, Hk), (keys, Hk), (rows, H)))
        for x in (q, k, v):
            x.requires_grad_()
        out = M.packed_attention(q, k, v, pack, causal=causal)
        want = ref.packed(q.detach()[:rows], k.detach()[:keys], v.detach()[:keys], n, m, causal, 1 / math.sqrt(D), do[:rows])
        grads = torch.autograd.grad(out, (q, k, v), do)
        for what, got, w, size in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads), want, (rows, rows, keys, keys)):
            ref.within(got[:size], w, f"{what} causal={causal}")
            assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", TYPES, ids=name)
def test_packed_attention_long(dtype):
    """More than one part on the key side, many tiles, scores far from zero and a scale of its own."""
    import transformer as M
    g, n, (H, Hk, D) = gen(5), [2500, 17, 1100], (8, 1, 64)
    q, do = rand(g, sum(n), H, D, dtype=dtype), rand(g, sum(n), H, D, dtype=dtype)
    k, v = (3 * rand(g, sum(n), Hk, D, dtype=dtype) for _ in range(2))
    k[::97] *= 4                                   # maxima that move late in a row
    for x in (q, k, v):
        x.requires_grad_()
    pack = M.PackedSequences(n, DEV)
    out = M.packed_attention(q, k, v, pack, scale=0.2)
    grads = torch.autograd.grad(out, (q, k, v), do)
    for what, got, w in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads), ref.packed(q.detach(), k.detach(), v.detach(), n, n, True, 0.2, do)):
        ref.within(got, w, what)
    again = torch.autograd.grad(M.packed_attention(q, k, v, pack, scale=0.2), (q, k, v), do)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "the same bits on every run"


@pytest.mark.parametrize("dtype", TYPES, ids=name)
def test_packed_attention_views_and_rows_behind(dtype):
    """Parts of one projection, transposed heads, a misaligned slice and a shared (expanded) key; what lies behind the
    last sequence, NaN here, reaches nothing, and has no gradient."""
    import transformer as M
    g, n, (H, Hk, D) = gen(6), [40, 150], (4, 2, 32)
    rows = sum(n) + 9
    qkv = rand(g, rows, (H + 2 * Hk) * D, dtype=dtype)
    qkv[sum(n):] = math.nan
    do = rand(g, rows, H, D, dtype=dtype)
    do[sum(n):] = math.nan
    pack = M.PackedSequences(n, DEV)
    odd = torch.empty(rows * Hk * D + 1, dtype=dtype, device=DEV)[1:].view(rows, Hk, D).copy_(qkv[:, (H + Hk) * D:].reshape(rows, Hk, D))
    views = {
        "projection": [x.unflatten(1, (-1, D)) for x in qkv.split([H * D, Hk * D, Hk * D], 1)],
        "transposed": [x.unflatten(1, (-1, D)).transpose(0, 1).contiguous().transpose(0, 1) for x in qkv.split([H * D, Hk * D, Hk * D], 1)],
        "misaligned": [qkv[:, :H * D].unflatten(1, (-1, D)), odd, odd],
        "inner stride": [x.unflatten(1, (-1, D)).transpose(1, 2).contiguous().transpose(1, 2) for x in qkv.split([H * D, Hk * D, Hk * D], 1)],
    }
    for what, (q, k, v) in views.items():
        q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
        out = M.packed_attention(q, k, v, pack)
        grads = torch.autograd.grad(out, (q, k, v), do.transpose(0, 1).contiguous().transpose(0, 1) if what == "transposed" else do)
        live = [x.detach()[:sum(n)] for x in (q, k, v)]
        for name_, got, w in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads), ref.packed(*live, n, n, True, 1 / math.sqrt(D), do[:sum(n)])):
            ref.within(got[:sum(n)], w, f"{what} {name_}")
            assert (got[sum(n):] == 0).all(), f"{what} {name_} behind the last sequence"
    # heads so far apart that 64 rows of a group pass 31 bits: copied
    far = torch.empty(12, 1 << 22, dtype=dtype, device=DEV)[:, :rows * 8].view(12, rows, 8).transpose(0, 1)
    q, k = rand(g, rows, 12, 8, dtype=dtype), rand(g, rows, 1, 8, dtype=dtype)
    far.copy_(q)
    a, b = (M.packed_attention(x, k, k, pack) for x in (far, q))
    assert torch.equal(a[:sum(n)], b[:sum(n)])
    # one key head broadcast to two: the gradient of the shared one is the sum
    one = rand(g, rows, 1, D, dtype=dtype)
    q = views["projection"][0].detach()
    leaf = one.clone().requires_grad_()
    out = M.packed_attention(q, leaf.expand(rows, 2, D), leaf.expand(rows, 2, D), pack)
    (got,) = torch.autograd.grad(out, leaf, do)
    a = ref.packed(q[:sum(n)], one[:sum(n)].expand(-1, 2, -1), one[:sum(n)].expand(-1, 2, -1), n, n, True, 1 / math.sqrt(D), do[:sum(n)])
    value, bound = (a[2][i] + a[3][i] for i in range(2))
    # autograd adds dk to dv and then the two heads, in the inputs' type: three more roundings of the parts' sizes
    parts = (a[2][0].abs() + a[3][0].abs()).sum(1, keepdim=True)
    ref.within(got[:sum(n)], (value.sum(1, keepdim=True), bound.sum(1, keepdim=True) + 4 * ref.U[dtype] * parts), "shared head")


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("shape", [(4, 4, 16), (4, 1, 64), (8, 2, 128), (3, 1, 96)], ids=str)
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("more", [[], MANY], ids=["few", "many"])
def test_packed_attention_hidden_values(dtype, shape, what, more):
    """An infinity or NaN in K and V of token 150 reaches no row before it; one in Q and dO of rows before 70 reaches the
    gradient of no key that they do not see.  The neighbours in the tile are the plain result."""
    import transformer as M
    H, Hk, D = shape
    g, n = gen(17), [20, 237, 33] + more
    pack = M.PackedSequences(n, DEV)
    q, k, v, do = (rand(g, sum(n), h, D, dtype=dtype) for h in (H, Hk, Hk, H))
    at, last = 20 + 150, 20 + 150
    kb, vb = k.clone(), v.clone()
    vb[at, :, 3] = what
    for keys in (kb, kb.clone()):
        if keys is not kb:
            keys[at + 1] = what                    # and in K of the next
        leaves = [x.detach().requires_grad_() for x in (q, keys, vb)]
        out = M.packed_attention(*leaves, pack)
        dq = torch.autograd.grad(out, leaves[0], do)[0]
        want = ref.packed(q[20:last], k[20:last], v[20:last], [150], [150], True, 1 / math.sqrt(D), do[20:last])
        ref.within(out[20:last].detach(), want[0], "out before")
        ref.within(dq[20:last], want[1], "dq before")
        assert not torch.isfinite(out[at, :, 3]).any()
        for part in (slice(0, 20), slice(257, 290)):
            m = part.stop - part.start
            want = ref.packed(q[part], k[part], v[part], [m], [m], True, 1 / math.sqrt(D), do[part])
            ref.within(out[part].detach(), want[0], "other sequences")
            ref.within(dq[part], want[1], "other sequences")
    for dirty in ("q", "do"):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        d = do.clone()
        if dirty == "q":
            with torch.no_grad():
                leaves[0][20 + 60:20 + 70] = what
        else:
            d[20 + 60:20 + 70] = what
        dk, dv = torch.autograd.grad(M.packed_attention(*leaves, pack), leaves[1:], d)
        want = ref.packed(q[20:257], k[20:257], v[20:257], [237], [237], True, 1 / math.sqrt(D), do[20:257])
        for got, w, which in ((dk, want[2], "dk"), (dv, want[3], "dv")):
            ref.within(got[20 + 70:257], [x[70:] for x in w], f"{dirty} {which} behind")


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("shape", [(4, 4, 16), (4, 1, 64), (8, 2, 128)], ids=str)
def test_paged_attention_hidden_values(dtype, shape):
    """The same for new tokens over a cache: a NaN in V of a later one of the chunk reaches no earlier one."""
    import transformer as M
    H, Hk, D = shape
    g, page = gen(18), 16
    for n, c in ((4, 700), (90, 333), (200, 200)):
        keys, values, table = cache_of(g, [c, 40], page, Hk, D, dtype)
        q = rand(g, n + 1, H, D, dtype=dtype)
        bad = values.clone()
        at = c - 2
        bad[table[0, at // page].long(), at % page, :, 1] = math.nan
        got = M.paged_attention(q, keys, bad, M.PagedBatch(table, [c, 40], [n, 1]))
        check_paged(q[:n - 2], keys, values, table[:1], [c - 2], [n - 2], True, 1 / math.sqrt(D), got[:n - 2])
        check_paged(q[n:], keys, values, table[1:], [40], [1], True, 1 / math.sqrt(D), got[n:])
        assert torch.isnan(got[n - 2:n, :, 1]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("more", [[], MANY], ids=["few", "many"])
def test_packed_attention_of_one_key(dtype, shape, more):
    """A row that sees a single key returns its value, and its scores have no gradient: zeros, not small numbers."""
    import transformer as M
    H, Hk, D = shape
    g, n, m = gen(9), [1, 1, 1, 2, 1], [1, 1, 1, 1, 1]
    pack = M.PackedSequences(n + more, DEV, m + more)
    q, k, v, do = (rand(g, r + sum(more), h, D, dtype=dtype).requires_grad_() for r, h in ((6, H), (5, Hk), (5, Hk), (6, H)))
    out = M.packed_attention(q, k, v, pack)
    of = [0, 1, 2, None, 3, 4]                     # the first of two rows over one key sees none
    for r, j in enumerate(of):
        want = torch.zeros(H, D, dtype=dtype, device=DEV) if j is None else v[j].repeat_interleave(H // Hk, 0)
        # one weight p: p v, 1 / p and their product are rounded in fp32, half a step each; a 16-bit v then comes out itself
        assert ((out[r] - want).abs() <= (3.1 * 2.0 ** -24 if dtype == torch.float32 else 0.0) * want.abs()).all(), r
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    assert (dq[:6] == 0).all() and (dk[:5] == 0).all()
    for r, j in enumerate(of):
        if j is not None:
            ref.within(dv[j], [x(do[r].detach().double().view(Hk, H // Hk, D)) for x in
                               (lambda y: y.sum(1), lambda y: 4 * ref.U[dtype] * y.abs().sum(1))], f"dv {j}")


@pytest.mark.parametrize("dtype", TYPES[1:], ids=name)
@pytest.mark.parametrize("dim", [32, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("copies", [3, 30], ids=["few", "many"])
def test_packed_attention_gradient_of_few_keys(dtype, dim, causal, copies):
    """Rows of few keys: rounding the slopes dS and weights P adds nothing to what rounding the results costs.  What is left is
    O's weights in D: of n like keys 1 / n of the variance that rounded slopes have (that of the result's own rounding), so
    at most sqrt(1 + 1 / 2) = 1.23 times the result's own error; with rounded slopes it is sqrt(2) or more."""
    import transformer as M
    n = [2, 3, 128, 5, 9, 17, 40, 64, 100] * copies
    g = gen(17)
    q, k, v, do = (rand(g, sum(n), h, dim, dtype=dtype) for h in (8, 2, 2, 8))
    leaves = [x.requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(M.packed_attention(*leaves, M.PackedSequences(n, DEV), causal=causal), leaves, do)
    want = ref.packed(*(x.detach() for x in leaves), n, n, causal, 1 / math.sqrt(dim), do)
    for got, (value, _) in zip(grads, want[1:]):
        assert float((got.double() - value).norm()) <= 1.3 * float((value.to(dtype).double() - value).norm())


@pytest.mark.parametrize("dtype", TYPES, ids=name)
def test_packed_attention_gradient_against_differences(dtype):
    import transformer as M
    g, n, (H, Hk, D) = gen(7), [70, 33], (4, 2, 32)
    q, k, v, do, dq_, dk_, dv_ = (rand(g, sum(n), h, D, dtype=dtype) for h in (H, Hk, Hk, H, H, Hk, Hk))
    leaves = [x.requires_grad_() for x in (q, k, v)]
    pack = M.PackedSequences(n, DEV)
    grads = torch.autograd.grad(M.packed_attention(*leaves, pack), leaves, do)
    along = sum(float((a.double() * b.double()).sum()) for a, b in zip(grads, (dq_, dk_, dv_)))
    e = 1e-4

    def loss(sign):
        moved = [x.detach().double() + sign * e * y.double() for x, y in zip(leaves, (dq_, dk_, dv_))]
        return float((ref.packed(*moved, n, n, True, 1 / math.sqrt(D))[0][0] * do.double()).sum())

    difference = (loss(1) - loss(-1)) / (2 * e)
    # the three gradients' own bounds along the direction, and the difference's cut-off term (third derivatives ~ 1e2)
    bounds = ref.packed(q.detach(), k.detach(), v.detach(), n, n, True, 1 / math.sqrt(D), do)[1:]
    slack = sum(float((b[1] * y.double().abs()).sum()) for b, y in zip(bounds, (dq_, dk_, dv_)))
    size = sum(float((b[0].abs() * y.double().abs()).sum()) for b, y in zip(bounds, (dq_, dk_, dv_)))
    assert abs(along - difference) <= slack + 1e-6 * size, (along, difference, slack)


def test_layouts_are_freed_with_their_batch():
    """A batch's layout, plans and device lists go when it goes, without the cycle collector; a graph of it that still
    waits for its backward pass keeps what it needs."""
    import gc
    import weakref
    import transformer as M
    g = gen(14)
    gc.collect()
    gc.disable()
    try:
        q = rand(g, 50, 2, 32).requires_grad_()
        pack = M.PackedSequences([20, 30], DEV)
        out = M.packed_attention(q, q, q, pack)
        gone = weakref.ref(pack)
        del pack
        assert gone() is None
        out.sum().backward()
        assert torch.isfinite(q.grad).all()
        first = M.packed_attention(q, q, q, M.PackedSequences([50], DEV))
        (one,) = torch.autograd.grad(first.sum(), q, create_graph=True)
        with pytest.raises(RuntimeError):
            one.sum().backward()                   # once differentiable
    finally:
        gc.enable()


def test_packed_attention_captured():
    """Forward and backward in a graph, replayed with new inputs between eager work, on a stream of their own."""
    import transformer as M
    n, (H, Hk, D) = [300, 45, 129], (8, 1, 64)
    pack = M.PackedSequences(n, DEV)
    g = gen(8)
    q, k, v, do = (rand(g, sum(n), h, D, dtype=torch.bfloat16) for h in (H, Hk, Hk, H))
    leaves = [x.requires_grad_() for x in (q, k, v)]

    def both():
        out = M.packed_attention(*leaves, pack)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for turn in range(3):
        with torch.no_grad():
            for x in (q, k, v, do):
                x.copy_(rand(g, *x.shape, dtype=x.dtype))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        for a, b in zip(got, both()):
            assert torch.equal(a, b), turn


# -------------------------------------------------------------------------------------------------------------- paged
def cache_of(g, context, page, Hk, D, dtype, spare=3):
    need = [-(-c // page) for c in context]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    table = torch.zeros(len(context), max(1, max(need)), dtype=torch.int32)
    for i, m in enumerate(need):
        table[i, :m] = torch.tensor(order[:m], dtype=torch.int32)
        order = order[m:]
    keys, values = (rand(g, pages, page, Hk, D, dtype=dtype) for _ in range(2))
    return keys, values, table.to(DEV)


def rows_of(pool, table, c):
    return pool[table.long()].flatten(0, 1)[:c]


def check_paged(q, keys, values, table, context, new, causal, scale, got):
    H, Hk = q.shape[1], keys.shape[2]
    r = 0
    for i, (n, c) in enumerate(zip(new, context)):
        k, v = rows_of(keys, table[i], c), rows_of(values, table[i], c)
        for h in range(H):
            (w,) = ref.head(q[r:r + n, h], k[:, h // (H // Hk)], v[:, h // (H // Hk)], c - n, causal, scale, q.dtype)
            # parts and waves add their sums: a few more fp32 roundings of the sum of sizes, inside (m + 4) STEP
            ref.within(got[r:r + n, h], w, f"sequence {i} head {h}")
        r += n


CONTEXTS = [
    ([1], [1]), ([1, 1, 1], [1, 17, 777]), ([1, 0, 1], [5000, 40, 0 + 1]), ([3, 1, 16], [64, 1000, 16]),
    ([40, 5, 200], [40, 3000, 517]), ([129, 1], [1300, 1025]),
]


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("shape", [(4, 4, 16), (8, 1, 64), (8, 2, 128), (6, 2, 96), (3, 1, 40), (40, 1, 32)], ids=str)
@pytest.mark.parametrize("case", CONTEXTS, ids=str)
def test_paged_attention(dtype, shape, case):
    import transformer as M
    (H, Hk, D), (new, context) = shape, case
    for page, causal in ((16, True), (64, True), (32, False)):
        g = gen(page + sum(context))
        keys, values, table = cache_of(g, context, page, Hk, D, dtype)
        for i, c in enumerate(context):            # what lies behind a sequence's end is stale, NaN here
            if c % page:
                keys[table[i, c // page].long(), c % page:] = math.nan
                values[table[i, c // page].long(), c % page:] = math.nan
        q = rand(g, sum(new), H, D, dtype=dtype)
        got = M.paged_attention(q, keys, values, M.PagedBatch(table, context, new), causal=causal)
        check_paged(q, keys, values, table, context, new, causal, 1 / math.sqrt(D), got)


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("shape", [(8, 8, 16), (16, 8, 8), (6, 6, 24), (10, 5, 32), (3, 3, 40)], ids=str)
def test_paged_attention_of_narrow_heads(dtype, shape):
    """Heads that share 128 bytes of the cache are worked on in an order of their own: every (part, head) once."""
    import transformer as M
    H, Hk, D = shape
    g, context, new = gen(19), [3000, 1, 700], [1, 1, 1]
    keys, values, table = cache_of(g, context, 16, Hk, D, dtype)
    q = rand(g, 3, H, D, dtype=dtype)
    got = M.paged_attention(q, keys, values, M.PagedBatch(table, context, new))
    check_paged(q, keys, values, table, context, new, True, 1 / math.sqrt(D), got)


@pytest.mark.parametrize("dtype", TYPES, ids=name)
def test_paged_attention_absent_pages(dtype):
    """A page number outside the pool: its keys are not there; a sequence of such pages gives zeros."""
    import transformer as M
    g, (H, Hk, D), page = gen(11), (4, 2, 64), 16
    for new in ([1, 1, 1], [100, 30, 2]):
        context = [300, 200, 100]
        keys, values, table = cache_of(g, context, page, Hk, D, dtype)
        bad = table.clone()
        bad[0, 3], bad[0, 7], bad[1, 0] = -1, keys.shape[0], 2 ** 31 - 1
        bad[2] = -5
        q = rand(g, sum(new), H, D, dtype=dtype)
        got = M.paged_attention(q, keys, values, M.PagedBatch(bad, context, new))
        r = 0
        for i, (n, c) in enumerate(zip(new, context)):
            k, v = rows_of(keys, table[i], c), rows_of(values, table[i], c)
            there = ((bad[i] >= 0) & (bad[i] < keys.shape[0])).repeat_interleave(page)[:c]
            for t in range(n):
                seen = there & (torch.arange(c, device=DEV) <= c - n + t)
                for h in range(H):
                    if not bool(seen.any()):
                        assert (got[r + t, h] == 0).all()
                        continue
                    (w,) = ref.head(q[r + t:r + t + 1, h], k[seen][:, h // 2], v[seen][:, h // 2], 0, False, 1 / math.sqrt(D), dtype)
                    ref.within(got[r + t:r + t + 1, h], w, f"sequence {i} token {t} head {h}")
            r += n


def test_paged_lengths_on_the_device():
    """Lengths rewritten on the device: beyond the table's pages there are no keys and nothing is written, below the number
    of new tokens the first of them see nothing, negative ones are empty."""
    import transformer as M
    g, (H, Hk, D), page, dtype = gen(15), (4, 2, 64), 16, torch.bfloat16
    for n in (3, 100):
        context = [120, 120, 120]
        keys, values, table = cache_of(g, context, page, Hk, D, dtype)           # 8 pages: 128 tokens each
        batch = M.PagedBatch(table, context, [n] * 3, max_length=128)
        batch.lengths.copy_(torch.tensor([128 + 2, 2, -7], dtype=torch.int32))
        q, k, v = (rand(g, 3 * n, h, D, dtype=dtype) for h in (H, Hk, Hk))
        got = M.paged_attention(q, keys, values, batch)
        ka, va = rows_of(keys, table[0], 128), rows_of(values, table[0], 128)
        for h in range(H):
            (w,) = ref.head(q[:n, h], ka[:, h // 2], va[:, h // 2], 130 - n, True, 1 / math.sqrt(D), dtype)
            ref.within(got[:n, h], w, "beyond the table")
            (w,) = ref.head(q[2 * n - 2:2 * n, h], rows_of(keys, table[1], 2)[:, h // 2], rows_of(values, table[1], 2)[:, h // 2], 0, True,
                            1 / math.sqrt(D), dtype)
            ref.within(got[2 * n - 2:2 * n, h], w, "short")
        assert (got[n:2 * n - 2] == 0).all() and (got[2 * n:] == 0).all()
        freq, _ = M.rotary_frequencies(D, device=DEV)
        before = keys.clone()
        M.append_rotary(q, k, v, keys, values, batch, freq)
        same = torch.ones(keys.shape[:2], dtype=torch.bool, device=DEV)
        for row, positions in ((0, range(130 - n, 128)), (1, range(2))):
            for p in positions:
                at = (table[row, p // page].long(), p % page)
                same[at] = False
                source = p - (130 - n) if row == 0 else n + (n - 2) + p
                assert torch.equal(values[at], v[source])
        assert torch.equal(keys[same], before[same])


def test_paged_attention_pool_beyond_32_bits():
    """A pool of more than 2^31 elements, the sequence in its last pages."""
    import transformer as M
    g, (H, Hk, D), page = gen(12), (4, 2, 128), 64
    pages = (1 << 31) // (page * Hk * D) + 40
    keys = torch.empty(pages, page, Hk, D, dtype=torch.bfloat16, device=DEV)
    values = torch.empty_like(keys)
    keys[-20:] = rand(g, 20, page, Hk, D, dtype=torch.bfloat16)
    values[-20:] = rand(g, 20, page, Hk, D, dtype=torch.bfloat16)
    table = torch.arange(pages - 1, pages - 21, -1, device=DEV, dtype=torch.int32)[None]
    for new in ([1], [300]):
        q = rand(g, new[0], H, D, dtype=torch.bfloat16)
        got = M.paged_attention(q, keys, values, M.PagedBatch(table, [1270], new))
        check_paged(q, keys, values, table, [1270], new, True, 1 / math.sqrt(D), got)
    k = rand(g, 5, Hk, D, dtype=torch.bfloat16)
    freq, _ = M.rotary_frequencies(D, device=DEV)
    M.append_rotary(q[:5], k, k, keys, values, M.PagedBatch(table, [1275], [5]), freq)
    assert torch.equal(rows_of(values, table[0], 1275)[1270:], k)


def test_paged_step_captured():
    """A decoding step in a graph: lengths grow on the device between replays; two graphs over one cache."""
    import transformer as M
    g, (H, Hk, D), page = gen(13), (8, 2, 64), 16
    context = [600, 33, 1200]
    keys, values, table = cache_of(g, [c + 40 for c in context], page, Hk, D, torch.bfloat16)
    freq, _ = M.rotary_frequencies(D, device=DEV)
    batch = M.PagedBatch(table, context, [1, 1, 1], max_length=1240)
    q, k, v = (rand(g, 3, h, D, dtype=torch.bfloat16) for h in (H, Hk, Hk))

    def step(b):
        return M.paged_attention(M.append_rotary(q, k, v, keys, values, b, freq), keys, values, b)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(batch)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(batch))
    for turn in range(6):
        for x in (q, k, v):
            x.copy_(rand(g, *x.shape, dtype=x.dtype))
        batch.lengths.add_(1)
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        got = outs[turn % 2].clone()
        fresh = M.PagedBatch(table, [c + turn + 1 for c in context], [1, 1, 1], max_length=1240)
        assert torch.equal(got, step(fresh)), turn


# ------------------------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims", [(16, 16), (128, 128), (96, 48), (80, 20), (6, 2), (64, 0), (33, 10), (256, 256), (128, 24)], ids=str)
def test_rotary(dtype, interleaved, dims):
    import transformer as M
    D, R = dims
    for rows, H, Hk, first in ((1, 3, 1, 0), (37, 5, 2, 1000000), (2500, 4, 4, -7)):
        g = gen(D + R + rows)
        qk = rand(g, rows, (H + Hk) * D, dtype=dtype)
        q, k = (x.unflatten(1, (-1, D)).detach().requires_grad_() for x in qk.split([H * D, Hk * D], 1))
        freq = (10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))).to(DEV)
        pos = torch.arange(rows, device=DEV, dtype=torch.int32) + first
        out = M.apply_rotary(q, k, pos, freq, interleaved=interleaved, multiplier=1.25)
        do = [rand(g, *x.shape, dtype=dtype) for x in out]
        grads = torch.autograd.grad(out, (q, k), do)
        for x, y, d, e in zip((q, k), out, do, grads):
            ref.within(y.detach(), ref.turned(x.detach(), pos, freq, interleaved, 1.25), "turned")
            ref.within(e, ref.turned(d, pos, freq, interleaved, 1.25, -1.0), "gradient")
            assert torch.equal(y[..., R:], x[..., R:])
        alone, none = M.apply_rotary(q.detach().transpose(1, 2).contiguous().transpose(1, 2), None, pos, freq, interleaved=interleaved, multiplier=1.25)
        assert none is None and torch.equal(alone, out[0])


def test_rotary_frequencies():
    import transformer as M
    plain, one = M.rotary_frequencies(64, device="cpu")
    assert one == 1.0 and plain[0] == 1.0 and abs(float(plain[-1]) - 10000.0 ** (-62 / 64)) < 1e-18
    assert torch.allclose(M.rotary_frequencies(64, scaling="linear", factor=4.0, device="cpu")[0], plain / 4, rtol=1e-15)
    base, _ = M.rotary_frequencies(64, scaling="base", factor=4.0, device="cpu")
    assert base[0] == 1.0 and abs(float(base[-1] / plain[-1]) - 0.25) < 1e-12
    ramp, m = M.rotary_frequencies(64, scaling="ramp", factor=8.0, original_length=2048, device="cpu")
    turns = 2048 * plain / (2 * math.pi)
    assert torch.equal(ramp[turns >= 32], plain[turns >= 32]) and torch.allclose(ramp[turns <= 1], plain[turns <= 1] / 8)
    assert abs(m - (1 + 0.1 * math.log(8))) < 1e-15 and (ramp <= plain).all() and (ramp >= plain / 8).all()


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("dims", [(128, 128, True), (96, 48, False), (40, 20, True), (36, 10, False), (16, 16, False)], ids=str)
def test_append_rotary(dtype, dims):
    import transformer as M
    (D, R, interleaved), H, Hk, page = dims, 6, 2, 16
    g = gen(D + R)
    for new, context in (([1, 1, 1], [40, 1, 16]), ([50, 0, 33, 1], [50, 20, 90, 17])):
        keys, values, table = cache_of(g, context, page, Hk, D, dtype)
        before = keys.clone(), values.clone()
        rows = sum(new) + 3
        q, k, v = (rand(g, rows, h, D, dtype=dtype) for h in (H, Hk, Hk))
        freq = (10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)).to(DEV)
        out = M.append_rotary(q, k, v, keys, values, M.PagedBatch(table, context, new), freq, interleaved=interleaved, multiplier=0.5)
        assert (out[sum(new):] == 0).all()
        written = torch.zeros(keys.shape[:2], dtype=torch.bool, device=DEV)
        r = 0
        for i, (n, c) in enumerate(zip(new, context)):
            pos = torch.arange(c - n, c, device=DEV, dtype=torch.int32)
            at = (table[i].long()[pos.long() // page], pos.long() % page)
            ref.within(out[r:r + n], ref.turned(q[r:r + n], pos, freq, interleaved, 0.5), "q")
            ref.within(keys[at], ref.turned(k[r:r + n], pos, freq, interleaved, 0.5), "k")
            assert torch.equal(values[at], v[r:r + n])
            written[at] = True
            r += n
        for pool, old in zip((keys, values), before):
            assert torch.equal(pool[~written], old[~written]), "only the new tokens' places are written"
        bad = table.clone()
        bad[:, 0] = torch.tensor([-1, 10 ** 6, -2, 2 ** 31 - 1][:len(new)], dtype=torch.int32, device=DEV)
        for pool, old in zip((keys, values), before):
            pool.copy_(old)
        M.append_rotary(q, k, v, keys, values, M.PagedBatch(bad, context, new), freq)
        absent = torch.cat([table[i, :1].long() for i in range(len(new))])
        assert torch.equal(keys[absent], before[0][absent]) and torch.equal(values[absent], before[1][absent])


# ----------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", TYPES, ids=name)
def test_model_trains_and_serves(dtype):
    """The module over packed sequences against itself over the cache: a prompt in chunks, then token by token."""
    import transformer as M
    torch.manual_seed(3)
    E, H, Hk = 128, 4, 2
    net = M.GroupedQueryAttention(E, H, Hk, rotary_dim=16, scaling="ramp", factor=4.0, original_length=64, dtype=dtype).to(DEV)
    lengths = [90, 7, 41]
    g = gen(21)
    x = rand(g, sum(lengths), E)
    pack = M.PackedSequences(lengths, DEV)
    with torch.no_grad():
        whole = net(x, pack)
    cache = net.new_cache(12, page_size=16)
    ids = [cache.add() for _ in lengths]
    start, left, parts = [0, 90, 97], list(lengths), [[] for _ in lengths]
    for chunk in ([40, 3, 1], [49, 0, 39], [1, 1, 1], [0, 1, 0], [0, 1, 0], [0, 1, 0]):
        batch = cache.extend(ids, chunk)
        new = torch.cat([x[s:s + n] for s, n in zip(start, chunk)])
        y = net.step(new, cache, batch).split(chunk)
        for i, n in enumerate(chunk):
            parts[i].append(y[i])
            start[i] += n
    served = torch.cat([torch.cat(p) for p in parts])
    # the same rotation and scores: outputs differ by the weights' rounding (twice a step of the type) through fc_out
    size = float(whole.abs().max())
    assert float((served - whole).abs().max()) <= (8 * ref.U[dtype] if dtype != torch.float32 else 2e-5) * max(1.0, size) * 2
    assert cache.free_pages == 12 - 6 - 1 - 3
    cache.remove(ids[0])
    assert cache.free_pages == 12 - 1 - 3
    # and the gradients of a training step exist and follow the loss along them
    loss = (net(x, pack) ** 2).sum()
    loss.backward()
    grads = [p.grad for p in net.parameters()]
    assert all(p is not None and bool(torch.isfinite(p).all()) for p in grads)


def test_other_stream():
    """Operators enqueue on the current stream: work on a side stream sees what that stream wrote."""
    import transformer as M
    g, n = gen(31), [500, 300]
    pack = M.PackedSequences(n, DEV)
    q, k, v = (rand(g, sum(n), h, 64, dtype=torch.bfloat16) for h in (8, 2, 2))
    want = M.packed_attention(q * 2, k, v, pack)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = M.packed_attention(q * 2, k, v, pack)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_batch_dropped_while_another_stream_reads_it():
    """A batch that goes while a launch on a side stream still waits: its lists are not handed to the next ones."""
    import transformer as M
    g, n = gen(32), [700, 10, 300]
    q, k, v = (rand(g, sum(n), h, 64, dtype=torch.bfloat16) for h in (4, 2, 2))
    want = M.packed_attention(q, k, v, M.PackedSequences(n, DEV))
    keys, values, table = cache_of(g, [90, 40], 16, 2, 64, torch.bfloat16)
    one = M.paged_attention(q[:2], keys, values, M.PagedBatch(table, [90, 40], [1, 1]))
    big = torch.empty(1 << 26, device=DEV)
    side = torch.cuda.Stream()
    for _ in range(3):
        pack, batch = M.PackedSequences(n, DEV), M.PagedBatch(table.clone(), [90, 40], [1, 1])
        lists = pack._work.query_tiles(2, True)
        held = {t.data_ptr() for t in (lists, batch.lengths, batch.starts, batch.table)}
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(20):
                big.zero_()                                    # the launches below wait for these
            got, two = M.packed_attention(q, k, v, pack), M.paged_attention(q[:2], keys, values, batch)
        del pack, batch, lists
        new = [torch.full((m,), 1, dtype=torch.int32, device=DEV) for m in (2, 3, 64, 96, 128) for _ in range(4)]
        waiting = not side.query()
        assert not waiting or not held & {t.data_ptr() for t in new}
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(two, one)


def test_saved_tensors_laid_out_anew():
    """Hooks on saved tensors may hand back the same values with other strides."""
    import transformer as M
    g, n, T = gen(33), [70, 0, 200], 290
    for dtype in (torch.bfloat16, torch.float32):
        qkv = rand(g, T, 8, 64, dtype=dtype).requires_grad_()
        do = rand(g, T, 4, 64, dtype=dtype)
        pack = M.PackedSequences(n, DEV)

        def run():
            return torch.autograd.grad(M.packed_attention(*qkv.split([4, 2, 2], 1), pack), qkv, do)[0]
        want = run()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu().contiguous(), lambda t: t.to(DEV)):
            got = run()
        assert torch.equal(got, want)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.transpose(0, -1).contiguous().transpose(0, -1)):
            got = run()
        assert torch.equal(got, want)


def test_arguments_go_by_value():
    """A scale held in a tensor is read at every call; what the host has checked cannot be replaced."""
    import transformer as M
    from s2g.lib import S2GError
    g = gen(34)
    q = rand(g, 20, 2, 32)
    pack = M.PackedSequences([20], DEV)
    keys, values, table = cache_of(g, [40], 16, 2, 32, torch.float32)
    batch = M.PagedBatch(table, [40], [20])
    scale = torch.tensor(0.5)
    first = M.packed_attention(q, q, q, pack, scale=scale), M.paged_attention(q, keys, values, batch, scale=scale)
    scale.fill_(0.125)
    again = M.packed_attention(q, q, q, pack, scale=scale), M.paged_attention(q, keys, values, batch, scale=scale)
    want = M.packed_attention(q, q, q, pack, scale=0.125), M.paged_attention(q, keys, values, batch, scale=0.125)
    for f, a, w in zip(first, again, want):
        assert torch.equal(a, w) and not torch.equal(f, w)
    for name in ("table", "rows", "max_length"):
        with pytest.raises(S2GError):
            setattr(batch, name, getattr(batch, name))
    with pytest.raises(S2GError):
        pack.rows = 10


@pytest.mark.parametrize("queries,keys", [([0, 0], [3, 0]), ([5, 0], [0, 0]), ([0], [0])])
def test_packed_attention_without_queries_or_keys(queries, keys):
    import transformer as M
    pack = M.PackedSequences(queries, DEV, keys)
    for spare in (0, 2):
        q, k, v = (torch.full((r + spare, h, 32), math.nan, device=DEV, requires_grad=True)
                   for r, h in ((sum(queries), 4), (sum(keys), 2), (sum(keys), 2)))
        out = M.packed_attention(q, k, v, pack)
        out.sum().backward()
        assert all(bool((x == 0).all()) for x in (out, q.grad, k.grad, v.grad))


def test_module_without_tokens():
    import transformer as M
    net = M.GroupedQueryAttention(64, 4, 2).to(DEV)
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    y = net(x, M.PackedSequences([0, 0], DEV))
    assert y.shape == (0, 64)
    y.sum().backward()
    assert x.grad.shape == x.shape and all(bool((p.grad == 0).all()) for p in net.parameters())
    cache = net.new_cache(2, page_size=16)
    assert net.step(x.detach(), cache, cache.extend([cache.add()], [0])).shape == (0, 64)


def test_refusals_on_gpu_tensors():
    import transformer as M
    from s2g.lib import S2GError
    pack = M.PackedSequences([4], DEV)
    x = lambda r, h, d, t=torch.float32: torch.zeros(r, h, d, dtype=t, device=DEV)  # noqa: E731
    for bad in ((x(4, 3, 32), x(4, 2, 32), x(4, 2, 32)), (x(4, 2, 12), x(4, 2, 12), x(4, 2, 12)), (x(4, 2, 136),) * 3,
                (x(3, 2, 32), x(4, 2, 32), x(4, 2, 32)), (x(4, 2, 32), x(3, 2, 32), x(3, 2, 32)), (x(4, 2, 32), x(4, 2, 32), x(4, 2, 64)),
                (x(4, 2, 32), x(4, 2, 32, torch.bfloat16), x(4, 2, 32)), (x(4, 2, 32, torch.float64),) * 3):
        with pytest.raises(S2GError):
            M.packed_attention(*bad, pack)
    ok = x(4, 2, 32)
    for scale in (0.0, -1.0, math.nan, math.inf, 1e31, 1e-31):
        with pytest.raises(S2GError):
            M.packed_attention(ok, ok, ok, pack, scale=scale)
    table = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    pool = torch.zeros(4, 16, 2, 32, device=DEV)
    batch = M.PagedBatch(table, [10], [4])
    freq, _ = M.rotary_frequencies(32, device=DEV)
    M.paged_attention(ok, pool, pool.clone(), batch)
    for keys in (torch.zeros(4, 12, 2, 32, device=DEV), torch.zeros(4, 16, 2, 40, device=DEV), torch.zeros(4, 16, 3, 32, device=DEV),
                 pool.bfloat16(), pool[..., ::2], torch.zeros(0, 16, 2, 32, device=DEV)):
        with pytest.raises(S2GError):
            M.paged_attention(ok, keys, keys.clone(), batch)
        with pytest.raises(S2GError):
            M.append_rotary(ok, ok, ok, keys, keys.clone(), batch, freq)
    with pytest.raises(S2GError):
        M.paged_attention(ok, pool, pool, M.PagedBatch(table, [40], [4]))           # beyond the table
    with pytest.raises(S2GError):
        M.paged_attention(ok[:3], pool, pool, batch)
    with pytest.raises(S2GError):
        M.paged_attention(ok.clone().requires_grad_(), pool, pool, batch)
    pos = torch.arange(4, dtype=torch.int32, device=DEV)
    for args in ((ok, ok, pos.long(), freq), (ok, ok, pos[:3], freq), (ok, ok, pos, freq.float()), (ok, x(3, 2, 32), pos, freq),
                 (x(4, 2, 16), None, pos, freq), (x(4, 1, 300), None, pos, freq)):
        with pytest.raises(S2GError):
            M.apply_rotary(*args)


def test_positions_and_frequencies_dropped_while_another_stream_reads_them():
    """The same for the positions of a batch and the frequencies of a module, which the rotation reads: forward without a graph,
    and the gradient's launch, which outlives the graph that held them."""
    import transformer as M
    g, n = gen(35), [700, 10, 300]
    q, k = (rand(g, sum(n), h, 64, dtype=torch.bfloat16).requires_grad_() for h in (4, 2))
    d = [rand(g, sum(n), h, 64, dtype=torch.bfloat16) for h in (4, 2)]
    freq, _ = M.rotary_frequencies(64, device=DEV)
    keys, values, table = cache_of(g, [90, 40], 16, 2, 64, torch.bfloat16)
    new = [x.detach()[:2] for x in (q, k, k)]

    def turned(pack, freq, batch):
        out = M.apply_rotary(q, k, pack.positions, freq)
        return [*(x.detach() for x in out), *torch.autograd.grad(out, (q, k), d),
                *M.apply_rotary(q.detach(), k.detach(), pack.positions, freq),
                M.append_rotary(*new, keys, values, batch, freq)]

    want = turned(M.PackedSequences(n, DEV), freq, M.PagedBatch(table, [90, 40], [1, 1]))
    big = torch.empty(1 << 26, device=DEV)
    side = torch.cuda.Stream()
    for _ in range(3):
        pack, mine, batch = M.PackedSequences(n, DEV), freq.clone(), M.PagedBatch(table.clone(), [90, 40], [1, 1])
        held = {pack.starts.data_ptr(), mine.data_ptr()}                # positions lie behind the starts
        rows = sum(n) + len(n) + 1
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(20):
                big.zero_()                                            # the launches below wait for these
            got = turned(pack, mine, batch)
        del pack, mine, batch
        fresh = [torch.full((m,), 7, dtype=t, device=DEV) for m, t in ((rows, torch.int32), (32, torch.float64)) for _ in range(4)]
        waiting = not side.query()
        assert not waiting or not held & {t.data_ptr() for t in fresh}
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tangents_are_refused_on_gpu_tensors():
    import transformer as M
    from s2g.lib import S2GError
    from torch.autograd import forward_ad
    g = gen(36)
    x, pack = rand(g, 20, 2, 32), M.PackedSequences([20], DEV)
    keys, values, table = cache_of(g, [40], 16, 2, 32, torch.float32)
    batch, (freq, _) = M.PagedBatch(table, [40], [20]), M.rotary_frequencies(32, device=DEV)
    leaf = x.clone().requires_grad_()
    out, want = M.packed_attention(leaf, x, x, pack), M.packed_attention(x, x, x, pack)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: M.apply_rotary(dual, None, pack.positions, freq), lambda: M.packed_attention(x, dual, x, pack),
                     lambda: M.append_rotary(x, dual, x, keys, values, batch, freq), lambda: M.paged_attention(dual, keys, values, batch),
                     lambda: torch.autograd.grad(out, leaf, dual)):
            with pytest.raises(S2GError, match="tangent"):
                call()
        assert torch.equal(M.packed_attention(x, x, x, pack), want)


def test_inference_mode_before_training():
    """A module, a batch and a cache first used under inference_mode train and are written to afterwards."""
    import transformer as M
    torch.manual_seed(4)
    net = M.GroupedQueryAttention(64, 4, 2, dtype=torch.bfloat16).to(DEV)
    x = rand(gen(37), 30, 64)
    with torch.inference_mode():
        pack = M.PackedSequences([20, 10], DEV)
        first = net(x, pack)
        cache = net.new_cache(4, page_size=16)
        batch = cache.extend([cache.add()], [20])
        net.step(x[:20], cache, batch)
    y = net(x, pack)
    assert torch.equal(y, first)
    y.square().mean().backward()
    assert all(bool(torch.isfinite(p.grad).all()) for p in net.parameters())
    batch.lengths.add_(0)
    cache.keys[0].zero_()
    assert not any(t.is_inference() for t in (pack.positions, pack.starts, batch.lengths, batch.starts, batch.table))


def test_first_use_inside_a_capture_is_refused():
    """A batch, or a module's copy of the frequencies, that would be made inside a capture raises; the capture goes on."""
    import transformer as M
    from s2g.lib import S2GError
    g = gen(38)
    q, pack = rand(g, 30, 2, 32), M.PackedSequences([30], DEV)
    leaf = q.clone().requires_grad_()
    warm = M.PackedSequences([30], DEV)
    M.packed_attention(leaf, q, q, warm)                   # forward only
    net, x = M.GroupedQueryAttention(64, 2).to(DEV), rand(g, 30, 64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: M.packed_attention(q, q, q, pack), lambda: M.PackedSequences([30], DEV), lambda: M.PagedBatch([[0]], [3], [1]),
                     lambda: net._turns(x.device), lambda: torch.autograd.grad(M.packed_attention(leaf, q, q, warm), leaf, q)):
            with pytest.raises(S2GError, match="capture"):
                call()
        held = M.packed_attention(q, q, q, warm)
    want = M.packed_attention(q, q, q, pack)
    for _ in range(2):
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
    net(x, pack)


@pytest.mark.parametrize("dtype", TYPES, ids=name)
def test_rotary_without_tokens_or_with_one_feature_in_any_layout(dtype):
    import transformer as M
    freq, _ = M.rotary_frequencies(32, device=DEV)
    q = torch.empty(0, 32, 4, dtype=dtype, device=DEV).transpose(1, 2).requires_grad_()
    out, _ = M.apply_rotary(q, None, torch.zeros(0, dtype=torch.int32, device=DEV), freq)
    out.sum().backward()
    assert out.shape == q.grad.shape == (0, 4, 32)
    wide = rand(gen(39), 7, 3, 5, dtype=dtype)
    one = wide.as_strided((7, 3, 1), (15, 5, 3))
    out, _ = M.apply_rotary(one, None, torch.zeros(7, dtype=torch.int32, device=DEV), freq[:0])
    assert torch.equal(out, wide[:, :, :1])


def test_tokens_too_wide_are_refused():
    import transformer as M
    from s2g.lib import S2GError
    g, t = gen(40), torch.float16
    q, k = rand(g, 1, 32768, 128, dtype=t), rand(g, 1, 256, 128, dtype=t)
    pack = M.PackedSequences([1], DEV)
    for args in ((q, k, k), (q.transpose(1, 2).contiguous().transpose(1, 2), k, k), (q, q, q), (q[:, :1].expand(1, 32768, 128), k, k)):
        with pytest.raises(S2GError, match="2\\^22"):
            M.packed_attention(*args, pack)
    with pytest.raises(S2GError, match="2\\^22"):
        M.paged_attention(q, k.expand(16, 256, 128)[None].contiguous(), k.expand(16, 256, 128)[None].contiguous(), M.PagedBatch([[0]], [1], [1]))
    pool = k.expand(16, 256, 128)[None].contiguous()
    got = M.paged_attention(q[:, :1].expand(1, 32768, 128), pool, pool, M.PagedBatch([[0]], [1], [1]))        # a broadcast one can be fetched
    assert torch.equal(got, k.repeat_interleave(128, 1))                                                     # (one key: its value)


@pytest.mark.parametrize("dim", [16, 40, 64, 128])
@pytest.mark.parametrize("queries", [2048, 100], ids=["many", "few"])
def test_packed_attention_small_weights_in_the_gradient(dim, queries):
    """fp16 weights below 2^-14, here 1 / 90000 each, reach dV with all their bits.  dO is one, so dV = queries / 90000.
    Off by half a step of the weight, all of them alike (2^-11), and half a step of the result (2^-11, and its floor); L is off by
    at most 2^-19 (half a step at 16, as much for the logarithm), 2^x by 2^-21, sums of like weights of 11 bits are exact."""
    import transformer as M
    g, m, dt = gen(41), 90000, torch.float16
    q, do = torch.zeros(queries, 1, dim, dtype=dt, device=DEV), torch.ones(queries, 1, dim, dtype=dt, device=DEV)
    k, v = (rand(g, m, 1, dim, dtype=dt).requires_grad_() for _ in range(2))
    out = M.packed_attention(q, k, v, M.PackedSequences([queries], DEV, [m]), causal=False)
    (dv,) = torch.autograd.grad(out, v, do)
    want = queries / m
    assert float((dv.double() - want).abs().max()) <= want * (2.0 ** -10 + 2.0 ** -17) + 2.0 ** -25


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("shape", [(4, 4, 16), (4, 2, 32), (3, 1, 64), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("more", [[], MANY], ids=["few", "many"])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention_of_a_key_that_no_row_weighs(dtype, shape, more, causal):
    """A key that is minus infinity in a feature in which all queries are positive: every score of it is minus infinity, every
    weight zero.  The rest is attention without that key; its own gradients are zeros, whatever stands behind the last row."""
    import transformer as M
    H, Hk, D = shape
    g, n, at = gen(42), [237, 40, 3] + more, 5
    q, k, v, do = (rand(g, sum(n), h, D, dtype=dtype) for h in (H, Hk, Hk, H))
    q[..., 1] = q[..., 1].abs() + 1
    bad = k.clone()
    bad[at, :, 1] = -math.inf
    leaves = [x.clone().requires_grad_() for x in (q, bad, v)]
    out = M.packed_attention(*leaves, M.PackedSequences(n, DEV), causal=causal)
    dk, dv = torch.autograd.grad(out, leaves[1:], do)
    assert (dk[at] == 0).all() and (dv[at] == 0).all()
    # rows before it see the keys up to themselves, rows from it on all of theirs but it
    rest = lambda x: torch.cat([x[:at], x[at + 1:237]])  # noqa: E731
    if causal:
        want = ref.packed(q[:237], *(torch.cat([x[:at], rest(x)]) for x in (k, v)), [at, 237 - at], [at, 236], True, 1 / math.sqrt(D), do[:237])
        want[2:] = [[torch.cat([x[:at] + x[at:2 * at], x[2 * at:]]) for x in w] for w in want[2:]]
    else:
        want = ref.packed(q[:237], rest(k), rest(v), [237], [236], False, 1 / math.sqrt(D), do[:237])
    ref.within(out[:237].detach(), want[0], "out")
    ref.within(rest(dk), want[2], "dk")
    ref.within(rest(dv), want[3], "dv")


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("shape", [(4, 2, 32), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("more", [[], MANY], ids=["few", "many"])
def test_rows_of_no_weight_give_zeros(dtype, shape, more):
    """Scores that are all minus infinity: zeros, as of a row that sees no key, and no gradient of k and v."""
    import transformer as M
    H, Hk, D = shape
    g, n = gen(43), [5, 150, 40] + more
    q, k, v, do = (rand(g, sum(n), h, D, dtype=dtype) for h in (H, Hk, Hk, H))
    q[..., 1] = q[..., 1].abs() + 1
    k[5:155, :, 1] = -math.inf
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = M.packed_attention(*leaves, M.PackedSequences(n, DEV))
    dk, dv = torch.autograd.grad(out, leaves[1:], do)
    assert all(bool((x[5:155] == 0).all()) for x in (out, dk, dv))
    assert all(bool(torch.isfinite(x).all()) and bool((x[155:] != 0).any()) for x in (out, dk, dv))
    keys, values, table = cache_of(g, [150, 90], 16, Hk, D, dtype)
    keys[table[0].long(), :, :, 1] = -math.inf
    for new in ([1, 1], [100, 2]):
        got = M.paged_attention(q.detach()[:sum(new)], keys, values, M.PagedBatch(table, [150, 90], new))
        assert (got[:new[0]] == 0).all()
        check_paged(q.detach()[new[0]:sum(new)], keys, values, table[1:], [90], new[1:], True, 1 / math.sqrt(D), got[new[0]:])


@pytest.mark.parametrize("dtype", TYPES[1:], ids=name)
@pytest.mark.parametrize("shape", [(4, 4, 16), (8, 2, 64), (16, 4, 128), (6, 2, 96)], ids=str)
def test_paged_attention_of_single_tokens_keeps_its_weights(dtype, shape):
    """Single tokens: rounding the weights adds nothing to what rounding the result costs.  Their second half leaves 2^-16 (bf16) of
    a weight, 2^-7 of a half step; with weights of one half the error is sqrt(2) of the result's own."""
    import transformer as M
    H, Hk, D = shape
    g, context = gen(44), [700, 33, 2900, 5100]
    keys, values, table = cache_of(g, context, 32, Hk, D, dtype)
    for new in ([1] * 4, [3, 1, 2, 4]):
        q = rand(g, sum(new), H, D, dtype=dtype)
        got = M.paged_attention(q, keys, values, M.PagedBatch(table, context, new))
        r, off, own = 0, 0.0, 0.0
        for i, (n, c) in enumerate(zip(new, context)):
            k, v = rows_of(keys, table[i], c), rows_of(values, table[i], c)
            for h in range(H):
                ((value, _),) = ref.head(q[r:r + n, h], k[:, h // (H // Hk)], v[:, h // (H // Hk)], c - n, True, 1 / math.sqrt(D), dtype)
                off += float((got[r:r + n, h].double() - value).square().sum())
                own += float((value.to(dtype).double() - value).square().sum())
            r += n
        assert off <= 1.02 ** 2 * own, math.sqrt(off / own)


def test_module_training_captured():
    """A training pass of the module in a graph: positions and frequencies of another stream, replayed between eager passes; the
    batch may go after the graph."""
    import transformer as M
    torch.manual_seed(5)
    g = gen(45)
    net = M.GroupedQueryAttention(64, 4, 2, rotary_dim=8, interleaved=True, dtype=torch.bfloat16).to(DEV)
    pack = M.PackedSequences([70, 3, 200], DEV)
    x, do = rand(g, 273, 64), rand(g, 273, 64)
    params = list(net.parameters())

    def both():
        y = net(x, pack)
        return [y.detach(), *torch.autograd.grad(y, params, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for turn in range(3):
        x.copy_(rand(g, 273, 64))
        do.copy_(rand(g, 273, 64))
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in held]
        for a, b in zip(got, both()):
            assert torch.equal(a, b), turn
    del graph, held, pack
    torch.cuda.synchronize()
    assert torch.isfinite(net(x, M.PackedSequences([273], DEV))).all()


def test_captured_decoding_over_pages_reserved_ahead():
    """All the tokens to come reserved by one extension, a batch of one token a sequence over its table, lengths advanced in place."""
    import transformer as M
    torch.manual_seed(6)
    g, steps, prompts = gen(46), 40, [20, 5]
    net = M.GroupedQueryAttention(64, 4, 2, dtype=torch.bfloat16).to(DEV)
    cache, plain = net.new_cache(16, page_size=16), net.new_cache(16, page_size=16)
    ids, twins = [cache.add() for _ in prompts], [plain.add() for _ in prompts]
    x = rand(g, sum(prompts), 64)
    net.step(x, cache, cache.extend(ids, prompts))
    net.step(x, plain, plain.extend(twins, prompts))
    ahead = cache.extend(ids, [steps] * 2)
    batch = M.PagedBatch(ahead.table, [p + 1 for p in prompts], [1, 1], max_length=max(prompts) + steps)
    token = rand(g, 2, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        net.step(token, cache, batch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = net.step(token, cache, batch)
    # two roundings of attention, a mean of values, half a step each, through fc_out's weights
    through, largest = float(net.fc_out.weight.detach().abs().sum(1).max()), 0.0
    for i in range(steps):
        token.copy_(rand(g, 2, 64))
        with torch.no_grad():
            largest = max(largest, *(float(net._project(z)[2].abs().max()) for z in (x, token)))
        graph.replay()
        want = net.step(token, plain, plain.extend(twins, [1, 1]))
        assert float((y - want).abs().max()) <= 2 * 2.0 ** -8 * 1.01 * through * largest, i
        batch.lengths.add_(1)


def test_first_calls_of_two_threads():
    """Two threads that use one batch for the first time, each on a stream of its own."""
    import threading
    import transformer as M
    g, n = gen(47), [500, 30, 77]
    q, k, v, do = (rand(g, sum(n), h, 64, dtype=torch.bfloat16) for h in (4, 2, 2, 4))

    def both(pack):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = M.packed_attention(*leaves, pack)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]
    want = both(M.PackedSequences(n, DEV))
    for _ in range(5):
        pack, got, streams = M.PackedSequences(n, DEV), {}, [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()

        def run(i):
            with torch.cuda.stream(streams[i]):
                got[i] = both(pack)
        threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(2) for a, b in zip(got[i], want))


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("shape", [(3, 3, 128), (4, 2, 96), (9, 3, 72), (4, 2, 64)], ids=str)
def test_packed_attention_gradient_of_keys_of_little_weight(dtype, shape):
    """Scores far apart, weights down to 2^-60 and below: a key that no row weighs much has a small gradient, not a wrong one."""
    import transformer as M
    H, Hk, D = shape
    g, n = gen(48), [126, 216, 5, 40]
    q, k, v, do = (rand(g, sum(n), h, D, dtype=dtype) for h in (H, Hk, Hk, H))
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = M.packed_attention(*leaves, M.PackedSequences(n, DEV), scale=1.0)
    got = (out.detach(), *torch.autograd.grad(out, leaves, do))
    for x, w, what in zip(got, ref.packed(*(x.detach() for x in leaves), n, n, True, 1.0, do), ("out", "dq", "dk", "dv")):
        ref.within(x, w, what)


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("more", [[], MANY], ids=["few", "many"])
def test_packed_attention_statistics_in_32_bits(dtype, dim, more):
    """One row over each set of keys and dO of ones, so dV is the row's weights.  Scores are whole eighths and exact; the row's
    statistics and 2^x are off by 2^-17 at |score| < 64 (half steps of score log2(e), of the maximum and of L), what the weights'
    second half leaves of them by 2^-16, the result by half a step."""
    import transformer as M
    g, H = gen(49), 2
    m = torch.randint(2, 128, (60,), generator=g, device=DEV).tolist()
    n, keys = [1] * 60 + more, m + more
    q = torch.randint(-2, 3, (sum(n), H, dim), generator=g, device=DEV) / 2
    k = torch.randint(-2, 3, (sum(keys), H, dim), generator=g, device=DEV) / 4 * (2 if dim < 64 else 1)
    q, k = q.to(dtype), k.to(dtype)
    v = rand(g, sum(keys), H, dim, dtype=dtype).requires_grad_()
    (dv,) = torch.autograd.grad(M.packed_attention(q, k, v, M.PackedSequences(n, DEV, keys), scale=1.0), v, torch.ones_like(q))
    at = 0
    for i, c in enumerate(m):
        s = torch.einsum("hd,khd->kh", q[i].double().cpu(), k[at:at + c].double().cpu())
        assert float(s.abs().max()) < 64
        p = torch.softmax(s, 0)[..., None].to(DEV)
        bound = p * (ref.U[dtype] * 1.01 + 2.0 ** -15) + ref.FLOOR[dtype]
        over = ((dv[at:at + c].double() - p).abs() - bound).max()
        assert float(over) <= 0, (i, float(over))
        at += c


@pytest.mark.parametrize("dtype", TYPES, ids=name)
@pytest.mark.parametrize("shape", [(4, 4, 16), (8, 2, 64), (6, 2, 96), (16, 4, 128)], ids=str)
@pytest.mark.parametrize("what", [math.inf, -math.inf])
def test_paged_attention_of_an_infinite_value(dtype, shape, what):
    """An infinity in V of a key that the rows see, and weigh: infinite in its feature, with its sign; the rest as ever."""
    import transformer as M
    H, Hk, D = shape
    g, context = gen(50), [700, 90]
    keys, values, table = cache_of(g, context, 16, Hk, D, dtype)
    bad, at = values.clone(), 333
    bad[table[0, at // 16].long(), at % 16, :, 3] = what
    rest = torch.arange(D, device=DEV) != 3
    for new in ([1, 1], [2, 5], [100, 1]):
        q = rand(g, sum(new), H, D, dtype=dtype)
        got = M.paged_attention(q, keys, bad, M.PagedBatch(table, context, new))
        want = M.paged_attention(q, keys, values, M.PagedBatch(table, context, new))
        assert (got[:new[0], :, 3] == what).all()
        got[:new[0], :, 3] = want[:new[0], :, 3]
        check_paged(q, keys, values, table, context, new, True, 1 / math.sqrt(D), got)
