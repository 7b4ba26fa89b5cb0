"""Refusals and layouts of the causal-transformer operators that need no GPU: C entry points reject bad arguments before
any launch, the bindings' structures match the header, batches and caches refuse what cannot be."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SIZES = {"int": 4, "float": 4, "long": 8}


def fields(text):
    """(name, type) of every member of a C structure's body."""
    out = []
    for line in re.sub(r"/\*.*?\*/", "", text, flags=re.S).split(";"):
        line = line.split()
        if line:
            out += [(n.strip().split("[")[0], line[0]) for n in " ".join(line[1:]).split(",")]
    return out


@pytest.mark.parametrize("name", ["S2GPacked", "S2GPaged", "S2GRotary"])
def test_structures_match_the_header(name):
    from s2g import lib
    body = {}
    for path in ("include/s2g.h", "sequence-to-graph-gan_amd/csrc/causal_lib.hip"):
        text = open(os.path.join(ROOT, path)).read()
        body[path] = fields(re.search(r"struct %s \{(.*?)\}" % name, text, re.S).group(1))
    a, b = body.values()
    assert a == b, "the library's own copy"
    cls = getattr(lib, name)
    assert [f for f, _ in a] == [f for f, _ in cls._fields_]
    for (f, t), (_, c) in zip(a, cls._fields_):
        assert ctypes.sizeof(c) == SIZES[t], f


def packed(**change):
    from s2g.lib import S2GPacked
    d = dict(type=1, heads=4, kv_heads=2, dim=64, causal=1, scale=0.125, q_ld=256, q_hd=64, k_ld=128, k_hd=64, v_ld=128, v_hd=64,
             do_ld=256, do_hd=64, q_rows=10, k_rows=10)
    d.update(change)
    return ctypes.byref(S2GPacked(**d))


def paged(**change):
    from s2g.lib import S2GPaged
    d = dict(type=1, sequences=2, heads=4, kv_heads=2, dim=64, causal=1, page_size=16, pages=8, table_cols=4, max_new=1, max_length=64,
             part_keys=512, parts=1, by_rows=0, scale=0.125, q_rows=2, q_ld=256, q_hd=64, page_ld=2048, token_ld=128, head_ld=64)
    d.update(change)
    return ctypes.byref(S2GPaged(**d))


def rotary(**change):
    from s2g.lib import S2GRotary
    d = dict(type=1, heads=4, kv_heads=2, dim=64, rotary=64, interleaved=0, backward=0, multiplier=1.0, rows=10, q_ld=256, q_hd=64,
             k_ld=128, k_hd=64, v_ld=128, v_hd=64)
    d.update(change)
    return ctypes.byref(S2GRotary(**d))


BAD_HEADS = [dict(type=3), dict(type=-1), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(dim=0), dict(dim=136), dict(dim=12),
             dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(heads=258, kv_heads=2), dict(q_ld=257),
             dict(q_hd=1 << 22), dict(q_rows=1 << 30)]


def test_c_entry_points_refuse():
    """Every pointer is a placeholder that is never read: all of these are turned down on the host."""
    from s2g import lib
    l, p = lib.load(), 4096
    for change in BAD_HEADS + [dict(k_ld=4), dict(v_hd=2), dict(do_ld=-8), dict(k_rows=-1)]:
        assert l.s2g_packed_attention_fwd(p, p, p, p, None, None, p, 1, packed(**change), None) == -1, change
        assert l.s2g_packed_attention_bwd(p, p, p, p, p, p, p, p, p, p, p, None, p, 1, p, 1, None, 0, packed(**change), None) == -1, change
        assert l.s2g_packed_attention_bwd_workspace(packed(**change), 2) == -1, change
    wide = dict(heads=256, kv_heads=2, type=0)              # 128 heads of a group, too far apart for 31 bits
    assert l.s2g_packed_attention_fwd(p, p, p, p, None, None, p, 1, packed(**wide, q_hd=(1 << 22) - 4, q_ld=64), None) == -1
    assert l.s2g_packed_attention_bwd_workspace(packed(**wide, do_hd=(1 << 22) - 4, do_ld=64), 1) == -1
    for i in (0, 1, 2, 3, 6):
        args = [p, p, p, p, None, None, p]
        args[i] = None
        assert l.s2g_packed_attention_fwd(*args, 1, packed(), None) == -1, i
    assert l.s2g_packed_attention_fwd(p + 2, p, p, p, None, None, p, 1, packed(), None) == -1
    assert l.s2g_packed_attention_fwd(p, p, p, p, None, None, p, 0, packed(), None) == -1
    assert l.s2g_packed_attention_fwd(p, p, p, p, None, None, p, 1, None, None) == -1
    assert l.s2g_packed_attention_bwd(p, p, p, p, p, p, p, p, p, p, p, None, p, 1, p, 1, p, 1, packed(), None) == -1      # cut tiles, no workspace
    assert l.s2g_packed_attention_bwd(p, p, p, p, p, p, p, p, p, p, p, p, p, 1, p, 1, None, 1, packed(), None) == -1
    assert l.s2g_packed_attention_bwd(p, p, p, p, None, p, p, p, p, p, p, p, p, 1, p, 1, None, 0, packed(), None) == -1       # bf16, no rest
    assert l.s2g_packed_attention_bwd_workspace(packed(), 3) == 3 * 256 * 2 * 64 and l.s2g_packed_attention_bwd_workspace(packed(), -1) == -1
    for change in BAD_HEADS + [dict(sequences=0), dict(sequences=65536), dict(page_size=8), dict(page_size=24), dict(page_size=1 << 17),
                               dict(pages=0), dict(table_cols=0), dict(table_cols=1 << 26), dict(max_new=0), dict(max_new=3),
                               dict(part_keys=0), dict(part_keys=100), dict(parts=0), dict(parts=5000), dict(max_length=600), dict(token_ld=3),
                               dict(head_ld=1), dict(page_ld=5), dict(page_ld=1 << 35), dict(page_size=65536, token_ld=1 << 15)]:
        assert l.s2g_paged_attention(p, p, p, p, p, p, p, p, paged(**change), None) == -1, change
        assert l.s2g_paged_attention_workspace(paged(**change)) == -1, change
    for i in range(7):
        args = [p] * 8
        args[i] = None
        assert l.s2g_paged_attention(*args, paged(), None) == -1, i
    assert l.s2g_paged_attention(p, p, p, p, p, p, p, None, paged(parts=2), None) == -1
    assert l.s2g_paged_attention_workspace(paged(parts=2)) == 2 * 4 * 2 * 66 and l.s2g_paged_attention_workspace(paged()) == 0
    for change in (dict(type=5), dict(rows=0), dict(rows=1 << 31), dict(heads=-1), dict(heads=0, kv_heads=0), dict(dim=0), dict(dim=257),
                   dict(rotary=63), dict(rotary=66), dict(rotary=-2), dict(multiplier=float("inf")), dict(multiplier=float("nan"))):
        assert l.s2g_rotary(p, p, p, p, p, p, rotary(**change), None) == -1, change
        assert l.s2g_rotary_append(p, p, p, p, p, p, p, p, p, p, rotary(**change), paged(), None) == -1, change
    for i in range(6):
        args = [p] * 6
        args[i] = None
        assert l.s2g_rotary(*args, rotary(), None) == -1, i
    for i in range(10):
        args = [p] * 10
        args[i] = None
        assert l.s2g_rotary_append(*args, rotary(), paged(), None) == -1, i
    for change in (dict(sequences=0), dict(page_size=15), dict(pages=0), dict(table_cols=0), dict(max_new=0), dict(max_new=11)):
        assert l.s2g_rotary_append(*[p] * 10, rotary(), paged(**change), None) == -1, change


def test_cpu_tensors_are_refused():
    import transformer as M
    from s2g.lib import S2GError
    x = torch.zeros(4, 2, 32)
    freq, _ = M.rotary_frequencies(32, device="cpu")
    with pytest.raises(S2GError):
        M.apply_rotary(x, x, torch.zeros(4, dtype=torch.int32), freq)
    with pytest.raises(S2GError):
        M.packed_attention(x, x, x, None)
    with pytest.raises(S2GError):
        M.paged_attention(x, x[None], x[None], None)
    with pytest.raises(S2GError):
        M.append_rotary(x, x, x, x[None], x[None], None, freq)
    with pytest.raises(S2GError):
        M.PackedSequences([3], "cpu")
    for bad in ([], [-1], [1 << 30]):
        with pytest.raises(S2GError):
            M.PackedSequences(bad, "cuda:0")
    with pytest.raises(S2GError):
        M.PackedSequences([1, 2], "cuda:0", [1])
    for lengths, new in (([], []), ([1], [2]), ([1, 2], [1]), ([3], [-1]), ([1 << 30], [1])):
        with pytest.raises(S2GError):
            M.PagedBatch(torch.zeros(1, 1, dtype=torch.int32), lengths, new)
    with pytest.raises(S2GError):
        M.PagedBatch(torch.zeros(2, 1, dtype=torch.int32), [1], [1])
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=4, base=0.0), dict(rotary_dim=4, factor=0.0), dict(rotary_dim=4, scaling="other")):
        with pytest.raises(S2GError):
            M.rotary_frequencies(**bad, device="cpu")
    for bad in ((5, 2, None), (8, 3, 2), (8, 4, 3), (8, 4, 0), (24, 2, 1), (272, 2, 2), (64, 2, 2, 34), (2064, 258, 2), (16, 2, 1, 4, False, 1e4, None, 1.0, 64, torch.float64)):
        with pytest.raises(S2GError):
            M.GroupedQueryAttention(*bad)


def test_cache_bookkeeping():
    """Pages are reserved on the host; the batch itself needs a GPU, so it is looked at before it is made."""
    from s2g import causal
    from s2g.lib import S2GError
    made = []
    whole, causal.PagedBatch = causal.PagedBatch, lambda table, lengths, new, device=None: made.append((table, lengths, new))
    try:
        cache = causal.PagedKVCache(6, 16, 2, 32, device="cpu")
        a, b = cache.add(), cache.add()
        cache.extend([a, b], [17, 0])
        assert cache.free_pages == 4 and cache.length(a) == 17 and made[-1][0].shape == (2, 2)
        cache.extend([b, a], [16, 15])
        assert cache.free_pages == 3 and made[-1][1] == [16, 32]
        cache.extend([a], [1])
        assert cache.free_pages == 2
        with pytest.raises(S2GError):
            cache.extend([a, b], [16, 32])
        assert cache.free_pages == 2 and cache.length(a) == 33 and cache.length(b) == 16
        pages = set(made[-1][0].flatten().tolist())
        cache.remove(a)
        assert cache.free_pages == 5
        c = cache.add()
        cache.extend([c], [80])
        assert cache.free_pages == 0 and pages <= set(made[-1][0].flatten().tolist())
        for bad in (([a], [1]), ([b, b], [1, 1]), ([b], [1, 2]), ([b], [-1]), ([], [])):
            with pytest.raises(S2GError):
                cache.extend(*bad)
        for bad in ((0, 16, 2, 32), (4, 8, 2, 32), (4, 24, 2, 32), (4, 16, 2, 12), (4, 16, 0, 32)):
            with pytest.raises(S2GError):
                causal.PagedKVCache(*bad, device="cpu")
        with pytest.raises(S2GError):
            causal.PagedKVCache(4, 16, 2, 32, dtype=torch.float64, device="cpu")
    finally:
        causal.PagedBatch = whole


def test_cache_refusals_change_nothing():
    """A batch that cannot be made leaves the cache as it was; pages a sequence does not own yet are no pages."""
    from s2g import causal
    from s2g.lib import S2GError

    def refuse(*args, **kw):
        raise S2GError("refused")
    whole, causal.PagedBatch = causal.PagedBatch, refuse
    try:
        cache = causal.PagedKVCache(6, 16, 2, 32, device="cpu")
        a, b = cache.add(), cache.add()
        with pytest.raises(S2GError):
            cache.extend([a, b], [17, 3])
        assert cache.free_pages == 6 and cache.length(a) == 0
        causal.PagedBatch = lambda table, lengths, new, device=None: table
        table = cache.extend([a, b], [33, 3])
        assert (table[1, 1:] == -1).all() and len({*table[0].tolist(), int(table[1, 0])}) == 4 and cache.free_pages == 2
        assert (cache.extend([a], [0])[0] == table[0]).all() and cache.extend([cache.add()], [0]).tolist() == [[-1]]
    finally:
        causal.PagedBatch = whole


def test_key_tiles_cover_every_row_once():
    """The key side's work list: every row that sees a tile is in exactly one of its entries, slots are consecutive."""
    import numpy as np
    from s2g import causal
    old, causal._on_device = causal._on_device, lambda values, device: torch.from_numpy(np.array(values, dtype=np.int32))
    try:
        for q, k in (([5000, 1, 130], None), ([3], [900]), ([700, 0, 40], [100, 300, 2048]), ([1] * 200, None)):
            pack = causal._WorkLists(np.array(q), np.array(k or q), "cpu")
            for group, heads, is_causal in ((1, 1, True), (8, 2, True), (3, 1, False)):
                tiles, cut, slots = pack.key_tiles(group, is_causal, heads)
                spans, used = {}, []
                for qs, ql, ks, kl, t, lo, hi, slot in tiles.tolist():
                    assert lo % 128 == 0 and (hi % 128 == 0 or hi == ql * group)
                    spans.setdefault((ks, kl, t), []).append((lo, hi))
                    used += [slot] if slot >= 0 else []
                assert sorted(used) == list(range(slots))
                assert len(spans) == sum(-(-m // 128) for m in pack.k_len)
                named = sorted(x for e in cut.tolist() for x in range(e[7], e[7] + e[5]))
                assert named == list(range(slots))
                for (ks, kl, t), parts in spans.items():
                    i = [j for j in range(len(pack.k_len)) if pack.k_start[j] == ks and pack.k_len[j] == kl][0]
                    rows = int(pack.q_len[i]) * group
                    first = max(0, t * 128 - (kl - int(pack.q_len[i]))) * group if is_causal else 0
                    parts.sort()
                    assert parts[0][0] <= first or first >= rows
                    assert all(a[1] == b[0] for a, b in zip(parts, parts[1:])) and (parts[-1][1] == rows or first >= rows)
    finally:
        causal._on_device = old


class Watched(torch.Tensor):
    """Says on which streams it has been recorded."""

    def record_stream(self, stream):
        self.streams.append(stream)


def watched(x):
    x = x.as_subclass(Watched)
    x.streams = []
    return x


def test_rotary_holds_positions_and_frequencies(monkeypatch):
    """What a launch reads of a batch (or of a module) that may go before the launch is done is kept from the allocator on the
    launch's stream, in the gradient too."""
    from s2g import causal
    monkeypatch.setattr(causal, "_launch", lambda *args: None)
    monkeypatch.setattr(causal, "_stream", lambda device: "the current one", raising=False)
    q, k = torch.randn(6, 2, 8, requires_grad=True), torch.randn(6, 1, 8, requires_grad=True)
    positions, frequencies = watched(torch.arange(6, dtype=torch.int32)), watched(torch.rand(4, dtype=torch.float64))
    causal._turn(q.detach(), None, positions, frequencies, False, 1.0, False)
    assert positions.streams == frequencies.streams == ["the current one"]
    out = causal.RotaryFn.apply(q, k, positions, frequencies, True, 1.0)
    assert positions.streams == frequencies.streams == ["the current one"] * 2
    torch.autograd.grad(out, (q, k), [torch.ones_like(x) for x in out])
    assert positions.streams == frequencies.streams == ["the current one"] * 3


def test_tangents_are_refused(monkeypatch):
    """The operators have no forward-mode derivative: a tensor that carries a tangent is turned down, whatever the gradient mode,
    where it would come back without it; so is one that reaches a gradient."""
    import transformer as M
    from s2g import causal
    from s2g.lib import S2GError
    from torch.autograd import forward_ad
    monkeypatch.setattr(causal, "_launch", lambda *args: None)
    monkeypatch.setattr(causal, "_check", lambda *args, **tensors: None)
    monkeypatch.setattr(causal, "_stream", lambda device: None)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, stream: None)
    x = torch.randn(4, 2, 32)
    pool, positions = torch.zeros(2, 16, 2, 32), torch.arange(4, dtype=torch.int32)
    freq, _ = M.rotary_frequencies(32, device="cpu")
    batch, pack = object.__new__(M.PagedBatch), object.__new__(M.PackedSequences)
    out = M.apply_rotary(x.clone().requires_grad_(), None, positions, freq)[0]
    with forward_ad.dual_level():
        dual, dual_pool = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(pool, torch.ones_like(pool))
        turns = forward_ad.make_dual(freq, torch.ones_like(freq))
        calls = [lambda: M.apply_rotary(x, None, positions, turns), lambda: M.append_rotary(x, x, x, pool, pool, batch, turns),
                 lambda: M.apply_rotary(dual, None, positions, freq), lambda: M.apply_rotary(x, dual, positions, freq),
                 lambda: M.packed_attention(dual, x, x, pack), lambda: M.packed_attention(x, x, dual, pack),
                 lambda: M.append_rotary(dual, x, x, pool, pool, batch, freq), lambda: M.append_rotary(x, x, x, pool, dual_pool, batch, freq),
                 lambda: M.paged_attention(dual, pool, pool, batch), lambda: M.paged_attention(x, dual_pool, pool, batch),
                 lambda: torch.autograd.grad(out, out.grad_fn.next_functions[0][0].variable, dual, retain_graph=True)]
        for call in calls:
            for mode in (torch.no_grad, torch.enable_grad):
                with mode(), pytest.raises(S2GError, match="tangent"):
                    call()
        M.apply_rotary(x, None, positions, freq)           # without one: as ever, inside a level too


def test_what_a_module_and_a_batch_keep_is_no_inference_tensor(monkeypatch):
    """Made while torch.inference_mode() is on, they are used by training steps later: autograd could not save them."""
    import transformer as M
    from s2g import causal
    monkeypatch.setattr(causal, "_no_capture", lambda *args: None)
    net = M.GroupedQueryAttention(64, 4, 2)
    with torch.inference_mode():
        made = [causal._on_device([1, 2, 3], "cpu"), net._turns(torch.device("meta")), M.rotary_frequencies(8, device="cpu")[0],
                *M.GroupedQueryAttention(64, 4, 2)._frequencies.values()]
        cache = causal.PagedKVCache(2, 16, 2, 32, device="cpu")
    assert not any(x.is_inference() for x in made + [cache.keys, cache.values])
    positions, q = made[0], torch.randn(3, 2, 8, requires_grad=True)
    (q * positions[:, None, None]).sum().backward()        # saved for it
    assert q.grad is not None


def test_layouts_are_refused_inside_a_capture(monkeypatch):
    """Asked of the stream that the call is on, not of the one that the batch was made on, which is not being captured."""
    import contextlib
    import numpy as np
    import transformer as M
    from s2g import causal
    from s2g.lib import S2GError
    current, made = ["the captured stream"], []

    @contextlib.contextmanager
    def stream(to):
        before, current[0] = current[0], to
        try:
            yield
        finally:
            current[0] = before
    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[0] == "the captured stream")
    monkeypatch.setattr(torch, "from_numpy", lambda x: made.append(x) or torch.zeros(x.shape, dtype=torch.int32))
    lists = causal._WorkLists(np.array([300]), np.array([300]), "cpu", "the batch's stream")
    for make in (lambda: lists.query_tiles(2, True), lambda: lists.key_tiles(2, True, 1)):
        with pytest.raises(S2GError, match="capture"):
            make()
    net = M.GroupedQueryAttention(64, 4, 2)
    with pytest.raises(S2GError, match="capture"):
        net._turns(torch.device("meta"))
    assert not made and not lists.kept
    current[0] = "another stream"
    kept = lists.query_tiles(2, True), lists.key_tiles(2, True, 1), net._turns(torch.device("meta"))
    current[0] = "the captured stream"
    assert kept[0] is lists.query_tiles(2, True) and kept[1] is lists.key_tiles(2, True, 1) and kept[2] is net._turns(torch.device("meta"))


@pytest.mark.parametrize("q", [torch.empty(0, 32, 4).transpose(1, 2), torch.ones(3, 2, 5)[:, :, ::5], torch.ones(3, 4, 4).transpose(1, 2)], ids=["empty", "narrow", "dense copy"])
def test_turn_of_layouts_that_count_as_contiguous(q, monkeypatch):
    """No tokens, or one feature: contiguous() hands such a tensor back with whatever last stride it has."""
    from s2g import causal
    launched = []
    monkeypatch.setattr(causal, "_launch", lambda device, name, *args: launched.append(name))
    monkeypatch.setattr(causal, "_hold", lambda *args: None)
    if q.shape[0] == 3 and q.shape[2] == 1:
        q = q.as_strided(q.shape, (10, 5, 5))
    assert q.stride(2) != 1
    positions = torch.zeros(q.shape[0], dtype=torch.int32)
    out, none = causal._turn(q, None, positions, torch.zeros(q.shape[2] // 2, dtype=torch.float64), False, 1.0, False)
    assert out.shape == q.shape and out.stride(2) == 1 and none is None and len(launched) == (q.shape[0] > 0)


def test_rows_that_no_copy_makes_fetchable_are_refused(monkeypatch):
    """Tokens of 2^22 elements or more, whichever way they are laid out: refused, not copied over and over."""
    import types
    import transformer as M
    from s2g import causal
    from s2g.lib import S2GError
    monkeypatch.setattr(causal, "_check", lambda *args, **tensors: None)
    tiles = torch.zeros(1, 8, dtype=torch.int32)
    pack = object.__new__(M.PackedSequences)
    for name, value in dict(device=torch.device("cpu"), rows=1, key_rows=1, _plans={}, _work=types.SimpleNamespace(query_tiles=lambda *a: tiles)).items():
        setattr(pack, name, value)
    q, k = torch.zeros(1, 32768, 128, dtype=torch.float16), torch.zeros(1, 256, 128, dtype=torch.float16)
    wide = torch.zeros(1, 32768, 128, dtype=torch.float16)
    for args in ((q, k, k), (q.transpose(1, 2).contiguous().transpose(1, 2), k, k), (wide, wide, wide)):
        with pytest.raises(S2GError, match="2\\^22"):
            M.packed_attention(*args, pack)
    batch = object.__new__(M.PagedBatch)
    for name, value in dict(device=torch.device("cpu"), table=torch.zeros(1, 1, dtype=torch.int32), rows=1, max_length=1, max_new=1, sequences=1,
                            _length=torch.ones(1).numpy(), _new=torch.ones(1).numpy(), _plans={}, _cuts={}).items():
        setattr(batch, name, value)
    pool = torch.zeros(1, 16, 256, 128, dtype=torch.float16)
    with pytest.raises(S2GError, match="2\\^22"):
        M.paged_attention(q, pool, pool, batch)


def test_module_runs_on_its_inputs_device(monkeypatch):
    """The projections' kernels go to the current device's stream: the module makes that its input's while it runs."""
    import contextlib
    import types
    import transformer as M
    from s2g import causal
    current, seen = [0], []

    @contextlib.contextmanager
    def device(to):
        before, current[0] = current[0], to
        try:
            yield
        finally:
            current[0] = before
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)

    class Stop(Exception):
        pass

    def project(self, x):
        seen.append(current[0])
        raise Stop
    monkeypatch.setattr(M.GroupedQueryAttention, "_project", project)
    net = M.GroupedQueryAttention(64, 4, 2)
    for index in (1, 0):
        x = types.SimpleNamespace(is_cuda=True, get_device=lambda: index, device=torch.device("cuda", index))
        for call in (lambda: net(x, None), lambda: net.step(x, None, None)):
            with pytest.raises(Stop):
                call()
    assert seen == [1, 1, 0, 0] and current == [0]
    assert type(causal.current_device(torch.zeros(1))) is contextlib.nullcontext


def test_module_loaded_onto_another_device_makes_its_frequencies_anew(monkeypatch):
    """A module saved whole and loaded with map_location has its copies of the frequencies moved with the rest."""
    import io
    import transformer as M
    from s2g import causal
    monkeypatch.setattr(causal, "_no_capture", lambda *args: None)
    net = M.GroupedQueryAttention(64, 4, 2)
    there = torch.device("meta")
    net._frequencies[there] = net._frequencies[torch.device("cpu")].clone()          # what map_location="cpu" makes of a device's copy
    assert net._turns(there).device == there
    file = io.BytesIO()
    torch.save(net, file)
    file.seek(0)
    again = torch.load(file, weights_only=False)
    assert torch.equal(again._turns(torch.device("cpu")), net._turns(torch.device("cpu")))
