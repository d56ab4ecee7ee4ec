"""CPU-only checks of the paged and windowed entry points: what the C ABI and the binding refuse before anything is
launched, and the 64-bit statement of the plan itself."""
import pytest
import torch

import paged_reference as R
from shareprefill_b200 import native

PTR = 1 << 20      # never dereferenced: every call below is refused first


def _attention(**kw):
    a = dict(q=PTR, qn=1024, qh=128, rows=4, heads=8, k=PTR, kp=4096, kt=256, kh=128, v=PTR, vp=4096, vt=256, vh=128, pages=9,
             page=16, kv=2, dim=128, dtype=0, table=PTR, ts=4, tw=4, cu=PTR, seq=PTR, req=2, most=1, scale=0.1, window=0, sinks=0,
             out=PTR, scratch=PTR, bytes=1, stream=None)
    assert set(kw) <= set(a)
    return native.load().spf_paged_attention(*{**a, **kw}.values())


def test_paged_attention_refusals():
    assert _attention(rows=0) == 0
    for name in ("q", "k", "v", "table", "cu", "seq", "out", "scratch"):
        assert _attention(**{name: None}) == -1, name
    for bad in (dict(dim=96), dict(heads=7), dict(kv=0), dict(page=24), dict(page=8), dict(page=512), dict(page=0)):
        assert _attention(**bad) == -2, bad
    for bad in (dict(q=PTR + 8), dict(k=PTR + 2), dict(out=PTR + 4), dict(scratch=PTR + 1), dict(qn=1020), dict(kt=252),
                dict(vh=4), dict(vp=4097)):
        assert _attention(**bad) == -3, bad
    for bad in (dict(dtype=2), dict(dtype=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=0.0), dict(scale=1e-60), dict(scale=1e39),
                dict(window=-1), dict(sinks=-1), dict(rows=-1), dict(pages=0), dict(req=0), dict(most=0), dict(tw=0), dict(ts=3),
                dict(bytes=1)):
        assert _attention(**bad) == -4, bad
    for bad in (dict(heads=512, kv=2), dict(req=4097), dict(tw=1 << 27, ts=1 << 27), dict(rows=(1 << 30) + 1)):
        assert _attention(**bad) == -6, bad


def test_window_plan_and_write_refusals():
    lib = native.load()

    def window(new=4, keys=9, dim=128, n=1024, scale=0.1, bytes_=1):
        return lib.spf_window_attention(PTR, n, 128, PTR, 256, 128, PTR, 256, 128, new, keys, 8, 2, dim, 0, scale, 4, 0, PTR, PTR,
                                        bytes_, None)
    assert window(new=0) == 0 and window(new=-1) == -4 and window(new=10) == -4 and window(dim=32) == -2
    assert window(n=1023) == -3 and window(scale=-1.0) == -4 and window(keys=(1 << 30) + 1) == -6
    assert window(bytes_=1) == -4       # scratch too small

    def plan(req=2, page=16, ts=4, tw=4, cap=8, rows=4, cached=PTR):
        return lib.spf_paged_plan(cached, PTR, req, page, PTR, ts, tw, PTR, cap, PTR, PTR, PTR, PTR, PTR, PTR, PTR, rows, None)
    assert plan(cached=None) == -1 and plan(page=48) == -2 and plan(req=0) == -4 and plan(req=4097) == -6
    assert plan(ts=3) == -4 and plan(tw=0) == -4 and plan(cap=0) == -4 and plan(rows=-1) == -4

    def write(rows=4, dim=128, page=16, pages=3, slot=PTR, kc=PTR):
        return lib.spf_paged_write(PTR, 256, 128, PTR, 256, 128, slot, rows, 2, dim, kc, 4096, 256, 128, PTR, 4096, 256, 128,
                                   pages, page, None)
    assert write(rows=0) == 0 and write(slot=None) == -1 and write(dim=72) == -2 and write(page=20) == -2
    assert write(pages=0) == -4 and write(rows=-1) == -4 and write(kc=PTR + 8) == -3


def test_packed_calls_are_the_calls():
    import ctypes
    import struct
    lib = native.load()
    kinds = {ctypes.c_void_p: "q", ctypes.c_int: "q", ctypes.c_int64: "q", ctypes.c_double: "d"}
    for number, name in enumerate(("spf_paged_plan", "spf_paged_write", "spf_paged_attention", "spf_window_attention")):
        types = native.SIGNATURES[name][1]
        pack = struct.Struct("".join(kinds[t] for t in types)).pack
        good = [PTR if t is ctypes.c_void_p else 0.1 if t is ctypes.c_double else 128 for t in types]
        ints = [i for i, t in enumerate(types) if t is ctypes.c_int]
        seen = set()
        for change in [()] + [(i, v) for i in range(len(types)) for v in (-1, 0, 3, 1 << 40)]:
            args = list(good)
            if change:
                if change[0] in ints and change[1] == 1 << 40:
                    args[change[0]] = change[1]
                    assert lib.spf_packed_call(number, pack(*args)) == -4
                    continue
                args[change[0]] = change[1] if types[change[0]] is not ctypes.c_double else float(change[1])
            args[ints[-1]] = -1                       # whatever else it is, nothing is launched
            if name in ("spf_paged_attention", "spf_window_attention"):
                args[-2] = 0                          # scratch of no bytes
            flat = getattr(lib, name)(*args)
            assert lib.spf_packed_call(number, pack(*args)) == flat <= 0, (name, change)      # no rows: nothing to do
            seen.add(flat)
        assert len(seen) >= 2, name
    assert lib.spf_packed_call(0, None) == -1 and lib.spf_packed_call(4, b"") == -4 and lib.spf_packed_call(-1, b"") == -4


def test_scratch_grows_with_the_tile_not_with_the_lengths():
    lib = native.load()
    one, many = lib.spf_paged_scratch_bytes(1, 32, 8, 128), lib.spf_paged_scratch_bytes(1 << 20, 32, 8, 128)
    assert 0 < one <= 32 << 20 and 0 < many <= 64 << 20
    assert lib.spf_paged_scratch_bytes(0, 32, 8, 128) == 0 and lib.spf_paged_scratch_bytes(1, 32, 5, 128) == 0


def test_binding_refuses_cpu_tensors():
    q, c, i = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: native.paged_attention(q, c, c, i[:, None], i, i, 1, 0.1), lambda: native.window_attention(q, q, q, 0.1, 4),
                 lambda: native.paged_write(q, q, i.long(), c, c), lambda: native.paged_plan(i, i, i[:, None], i, i, 4, 16)):
        with pytest.raises(native.SpfError, match="CUDA"):
            call()


def test_statement_of_the_plan():
    p = R.plan([15, 0, 16], [2, 40, 0], [[4, -1, -1], [-1] * 3, [6, -1, -1]], 3, [9, 8, 7, 5], 3, 3, 44, 16)
    assert p["table"] == [[4, 5, -1], [-1, -1, -1], [6, -1, -1]]        # the second lacks three pages, two are left
    assert p["refused"] == [0, 1, 0] and p["seq_len"] == [17, 0, 16] and p["cu_new"] == [0, 2, 42, 42]
    assert p["slot_map"] == [4 * 16 + 15, 5 * 16] + [-1] * 42 and p["ring_state"] == [0, 2]


def test_statement_of_the_attention():
    q, k = torch.randn(3, 2, 8), torch.randn(5, 1, 8)
    v = torch.randn(5, 1, 8)
    out, _ = R.attention(q, k, v, 2, 0.3, window=1)
    assert torch.allclose(out, v[2:].double().expand(-1, 2, -1))       # a window of one: the token's own value
    out, _ = R.attention(q, k, v, 2, 0.3, present=torch.zeros(5, dtype=torch.bool))
    assert bool((out == 0).all())


def test_sliding_window_layers_refuse_what_they_cannot_do():
    from types import SimpleNamespace

    from shareprefill_b200.attention import shareprefill_attention_forward as forward
    module = SimpleNamespace(training=False, attention_dropout=0.1, scaling=0.1)
    x = torch.zeros(1, 4, 9, 64, dtype=torch.bfloat16)
    with pytest.raises(native.SpfError, match="CUDA"):
        forward(module, x, x[:, :2], x[:, :2], None, sliding_window=4)
    for kw, q in ((dict(s_aux=torch.zeros(4)), x), (dict(softcap=30.0), x), (dict(gqa_interleave=True), x), ({}, x.expand(2, -1, -1, -1))):
        with pytest.raises(NotImplementedError):
            forward(module, q, x[:, :2], x[:, :2], None, sliding_window=4, **kw)
    with pytest.raises(native.SpfError, match="neither"):
        forward(module, x[:, :, :5], x[:, :2], x[:, :2], None, sliding_window=4)
    with pytest.raises(native.SpfError, match="at least 1"):
        forward(module, x, x[:, :2], x[:, :2], None, sliding_window=0)
    module.training = True
    with pytest.raises(native.SpfError, match="dropout"):
        forward(module, x, x[:, :2], x[:, :2], None, sliding_window=4)


def test_plans_of_more_rows_than_a_batch_may_have_are_refused():
    # (the kernel's row counter would pass 32 bits just below 2^31 rows)
    for rows in ((1 << 28) + 1, (1 << 31) - 4097, (1 << 31) - 1):
        assert native.load().spf_paged_plan(PTR, PTR, 2, 16, PTR, 4, 4, PTR, 8, PTR, PTR, PTR, PTR, PTR, PTR, PTR, rows, None) == -6


def test_more_work_than_a_call_can_count_is_refused():
    # a causal prompt of 2^28 tokens is 2^40 units of keys, 2^33 a CTA; with a window it is a line that fits
    lib = native.load()
    for heads, n in ((64, 1 << 28), (8, 1 << 28), (64, 1 << 26)):
        assert lib.spf_window_attention(PTR, 1 << 14, 128, PTR, 1 << 14, 128, PTR, 1 << 14, 128, n, n, heads, 8, 128, 0, 0.1, 0, 0, PTR, PTR,
                                        1 << 40, None) == -6
    assert _attention(rows=1 << 24, req=4096, most=1 << 12, tw=1 << 24, ts=1 << 24, bytes=1 << 40) == -6


def test_gradients_are_refused_not_dropped():
    from types import SimpleNamespace

    from shareprefill_b200.attention import shareprefill_attention_forward as forward
    q, c, i = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    g, gc = q.clone().requires_grad_(), c.clone().requires_grad_()
    module = SimpleNamespace(training=True, attention_dropout=0.0, scaling=0.1)
    x = torch.zeros(1, 4, 9, 64, dtype=torch.bfloat16, requires_grad=True)
    calls = [lambda: native.paged_attention(g, c, c, i[:, None], i, i, 1, 0.1), lambda: native.paged_attention(q, gc, c, i[:, None], i, i, 1, 0.1),
             lambda: native.paged_attention(q, c, gc, i[:, None], i, i, 1, 0.1), lambda: native.window_attention(g, q, q, 0.1, 4),
             lambda: native.window_attention(q, g, q, 0.1, 4), lambda: native.window_attention(q, q, g, 0.1, 4),
             lambda: native.paged_write(g, q, i.long(), c, c), lambda: native.paged_write(q, q, i.long(), c, gc),
             lambda: forward(module, x, x[:, :2], x[:, :2], None, sliding_window=4)]
    for call in calls:
        with pytest.raises(native.SpfError, match="no backward"):
            call()
        with torch.no_grad(), pytest.raises(native.SpfError, match="CUDA"):
            call()


def test_sliding_window_layers_refuse_masks_other_orders_and_buffers_that_are_not_full():
    from types import SimpleNamespace

    from shareprefill_b200.attention import shareprefill_attention_forward as forward
    x = torch.zeros(1, 4, 9, 64, dtype=torch.bfloat16)
    module = SimpleNamespace(training=False, attention_dropout=0.0, scaling=0.1)
    with pytest.raises(NotImplementedError, match="mask"):
        forward(module, x, x[:, :2], x[:, :2], torch.zeros(1, 1, 9, 9), sliding_window=4)
    with pytest.raises(NotImplementedError, match="causal"):
        forward(module, x, x[:, :2], x[:, :2], None, sliding_window=4, is_causal=False)
    for causal in (True, None):
        with pytest.raises(native.SpfError, match="CUDA"):
            forward(module, x, x[:, :2], x[:, :2], None, sliding_window=4, is_causal=causal)
    with pytest.raises(NotImplementedError, match="causal"):
        forward(SimpleNamespace(**vars(module), is_causal=False), x, x[:, :2], x[:, :2], None, sliding_window=4)
    for tokens, error, words in ((5, NotImplementedError, "5 tokens"), (8, NotImplementedError, "8 tokens"), (9, native.SpfError, "CUDA"),
                                 (40, native.SpfError, "CUDA"), (None, native.SpfError, "CUDA")):
        module.attention_sharing = SimpleNamespace(tokens_so_far=tokens)
        with pytest.raises(error, match=words):
            forward(module, x[:, :, :1], x[:, :2], x[:, :2], None, sliding_window=8)


def test_writes_into_expanded_caches_are_refused():
    def write(kp=4096, kt=256, kh=128, vp=4096, vt=256, vh=128, heads=2, pages=0):
        return native.load().spf_paged_write(PTR, 256, 128, PTR, 256, 128, PTR, 4, heads, 128, PTR, kp, kt, kh, PTR, vp, vt, vh, pages or 3, 16, None)
    for name in ("kp", "kt", "kh", "vp", "vt", "vh"):
        assert write(**{name: 0}) == -4, name
