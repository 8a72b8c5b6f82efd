"""Refusals of the paged-cache and linear-attention entry points, before anything is launched."""
import ctypes

import pytest

import qwfn_kv as K

FAKE = 0x7F0000000000          # never dereferenced: validation fails first
GB = 1 << 30


def refused(rc, code, needle):
    assert rc == code, (rc, K.load().qwfn_last_error())
    assert needle in K.load().qwfn_last_error().decode(), K.load().qwfn_last_error()


def extend(**kw):
    a = dict(past=FAKE, new=FAKE + GB, n_seq=4, page=16, table=FAKE + 2 * GB, stride=8, cols=8, free=FAKE + 3 * GB, cap=10,
             n_free=FAKE + 4 * GB, n_free_out=FAKE + 5 * GB, n_kv=FAKE + 6 * GB, cu=FAKE + 7 * GB, slots=FAKE + 8 * GB,
             pos=None, seq=None, n_tok=9, pad=-1, ws=FAKE + 9 * GB, ws_bytes=1 << 20)
    a.update(kw)
    return K.load().qwfn_paged_extend(*a.values(), None)


def trim(**kw):
    a = dict(keep=FAKE, n_kv=FAKE + GB, n_seq=4, page=16, table=FAKE + 2 * GB, stride=8, cols=8, free=FAKE + 3 * GB, cap=10,
             n_free=FAKE + 4 * GB, n_free_out=FAKE + 5 * GB, n_kv_out=FAKE + 6 * GB, ws=FAKE + 9 * GB, ws_bytes=1 << 20)
    a.update(kw)
    return K.load().qwfn_paged_trim(*a.values(), None)


@pytest.mark.parametrize("call", [extend, trim])
def test_tables_refusals(call):
    refused(call(n_free=None), K.EINVAL, "NULL")
    refused(call(table=None), K.EINVAL, "NULL")
    refused(call(n_seq=0), K.EINVAL, "n_seq")
    refused(call(n_seq=65537), K.EINVAL, "n_seq")
    refused(call(page=0), K.EINVAL, "page_size")
    refused(call(cols=0), K.EINVAL, "max_pages")
    refused(call(page=1 << 20, cols=1 << 11, stride=1 << 11), K.EINVAL, "2^31")
    refused(call(stride=7), K.EINVAL, "overlap")
    refused(call(cap=-1), K.EINVAL, "free_cap")
    refused(call(ws=None), K.ENOMEM, "ws")
    refused(call(ws_bytes=16), K.ENOMEM, "ws")
    refused(call(ws=FAKE + 9 * GB + 4), K.EALIGN, "16-byte")
    refused(call(table=FAKE + 2 * GB + 2), K.EALIGN, "table")
    refused(call(free=FAKE + 2 * GB + 4), K.EINVAL, "overlaps")
    refused(call(n_free=FAKE + 5 * GB + 4, n_free_out=FAKE + 5 * GB + 2), K.EALIGN, "n_free_out")
    assert K.paged_workspace_size(0) == 0 and K.paged_workspace_size(65537) == 0 and K.paged_workspace_size(5) > 0


def test_extend_refusals():
    refused(extend(n_tok=-1), K.EINVAL, "n_tok")
    refused(extend(n_tok=1 << 31), K.EINVAL, "n_tok")
    refused(extend(slots=None), K.EINVAL, "NULL")
    refused(extend(n_kv=FAKE + 4), K.EINVAL, "n_kv overlaps n_past")
    refused(extend(n_kv=FAKE + GB), K.EINVAL, "n_kv overlaps n_new")
    refused(extend(pos=FAKE + 8 * GB + 32), K.EINVAL, "pos overlaps slots")
    refused(extend(cu=FAKE + 9 * GB + 64), K.EINVAL, "ws overlaps cu_new")
    refused(trim(n_kv_out=FAKE + GB + 8), K.EINVAL, "n_kv_out overlaps n_kv")


def paged_views(D=256, T=1, nh=16, B=4, kvh=2, rows=640, qtype=K.TYPE_F32, nb1=None, nb2=None):
    es = 4 if qtype == K.TYPE_F32 else 2
    seg = D // 32 * 34
    q = K.tensor(FAKE, qtype, (D, T, nh, B), (es, nh * D * es, D * es, T * nh * D * es))
    k = K.tensor(FAKE + GB, K.TYPE_Q8_0, (D, rows, kvh, 1), (34, nb1 or kvh * seg, nb2 or seg, rows * kvh * seg))
    o = K.tensor(FAKE + 2 * GB, qtype, (D, nh, T, B), (es, D * es, nh * D * es, T * nh * D * es))
    return q, k, o


def paged(q, k, o, v=None, table=FAKE, stride=40, cols=40, page=16, n_kv=FAKE, scale=0.0625, gate=None, variant=1,
          ws=FAKE + 3 * GB, ws_bytes=1 << 30):
    r = ctypes.byref
    return K.load().qwfn_flash_attn_ext_q8_0_paged(r(q), r(k), r(v or k), table, stride, cols, page, n_kv, scale,
                                                   r(gate) if gate else None, r(o), variant, ws, ws_bytes, None)


def test_paged_attention_refusals():
    q, k, o = paged_views()
    assert K.load().qwfn_fattn_workspace_size_paged(ctypes.byref(q), ctypes.byref(k), ctypes.byref(k), 40, 16) > 0
    for D in (32, 96, 512):
        refused(paged(*paged_views(D=D)), K.ENOTSUP, "head size")
    refused(paged(*paged_views(qtype=K.TYPE_I32)), K.EINVAL, "f32, f16 or bf16")
    refused(paged(*paged_views(nh=15)), K.EINVAL, "multiple of n_head_kv")
    refused(paged(*paged_views(T=9)), K.ENOTSUP, "64 query rows")
    refused(paged(*paged_views(rows=15)), K.EINVAL, "no whole page")
    refused(paged(*paged_views(nb1=544 + 8)), K.EALIGN, "aligned")
    refused(paged(*paged_views(nb1=528)), K.EINVAL, "overlap")
    refused(paged(*paged_views(nb2=256)), K.EINVAL, "overlap")
    refused(paged(q, k, o, table=None), K.EINVAL, "NULL")
    refused(paged(q, k, o, n_kv=None), K.EINVAL, "NULL")
    refused(paged(q, k, o, page=0), K.EINVAL, "page_size")
    refused(paged(q, k, o, cols=1 << 27, stride=1 << 27), K.EINVAL, "2^31")
    refused(paged(q, k, o, stride=39), K.EINVAL, "overlap")
    refused(paged(q, k, o, scale=float("inf")), K.EINVAL, "finite")
    refused(paged(q, k, o, variant=3), K.EINVAL, "variant")
    refused(paged(q, k, o, ws_bytes=64), K.ENOMEM, "ws")
    refused(paged(q, k, o, ws=FAKE + 8), K.EALIGN, "ws")
    refused(paged(q, k, o, n_kv=FAKE + 2), K.EALIGN, "n_kv")
    refused(paged(q, k, o, v=paged_views(rows=641)[1]), K.EINVAL, "same shape")
    half = paged_views(qtype=K.TYPE_BF16)[2]
    refused(paged(q, k, half), K.EINVAL, "dst must have q's type")
    refused(paged(q, k, o, gate=half), K.EINVAL, "gate must have q's type")
    wrong = paged_views(B=3)[2]
    refused(paged(q, k, wrong), K.EINVAL, "dst must be contiguous")
    refused(paged(q, k, o, gate=wrong), K.EINVAL, "gate must be contiguous")
    q.data = FAKE + 4
    refused(paged(q, k, o), K.EALIGN, "q must be")
    q.data = None
    refused(paged(q, k, o), K.EINVAL, "NULL")


def heads(d, h, n, typ=K.TYPE_BF16, at=FAKE, stride=None):
    es = 4 if typ == K.TYPE_F32 else 2
    return K.tensor(at, typ, (d, h, n, 1), (es, d * es, stride or d * h * es, (n or 1) * d * h * es))


def linear(q=None, k=None, v=None, g=FAKE, g_ts=6, cu=FAKE, n_seq=3, max_len=50, slots=None, n_slots=4, s_in=FAKE,
           s_out=FAKE + GB, scale=1.0, dst=None, ws=FAKE, ws_bytes=1 << 30):
    r = ctypes.byref
    q, k = q or heads(128, 2, 100), k or heads(128, 2, 100)
    v, dst = v or heads(128, 6, 100), dst or heads(128, 6, 100)
    return K.load().qwfn_linear_attn(r(q), r(k), r(v), g, g_ts, cu, n_seq, max_len, slots, n_slots, s_in, s_out, scale, r(dst),
                                     ws, ws_bytes, None)


def test_results_over_inputs_and_wide_strides_refused():
    """Results that would be written over what other workgroups still read, and strides that pass the address space."""
    for call in (extend, trim):
        refused(call(stride=1 << 31), K.EINVAL, "table_stride")
    q, k, o = paged_views()
    refused(paged(q, k, o, stride=1 << 31), K.EINVAL, "table_stride")
    q.data = o.data
    refused(paged(q, k, o), K.EINVAL, "dst overlaps q")
    q.data = o.data + 4 * 16 * 256 * 4 - 16                # the last 16 bytes of dst
    refused(paged(q, k, o), K.EINVAL, "dst overlaps q")
    q, k, o = paged_views()
    gate = paged_views()[2]
    gate.data = o.data + 16
    refused(paged(q, k, o, gate=gate), K.EINVAL, "dst overlaps gate")
    at = FAKE + 3 * GB
    for name, d, n in (("q", 128, 2), ("k", 128, 2), ("v", 128, 6)):
        refused(linear(**{name: heads(d, n, 100, at=at + 100 * 6 * 128 * 2 - 16)}, dst=heads(128, 6, 100, at=at)), K.EINVAL,
                "dst overlaps")


def test_more_work_than_a_launch_has_threads():
    refused(paged(*paged_views(D=64, nh=2048, kvh=32, B=65536), cols=1, stride=1), K.ENOTSUP, "too many query rows")
    far = dict(q=heads(16, 1, 100), k=heads(16, 1, 100), v=heads(16, 1024, 100, at=FAKE + GB), g_ts=1024, n_seq=65535,
               n_slots=65535, s_in=None, s_out=FAKE + 8 * GB, dst=heads(16, 1024, 100, at=FAKE + 2 * GB))
    for max_len in (1, 50):
        refused(linear(max_len=max_len, ws_bytes=1 << 60, **far), K.ENOTSUP, "too many sequences")


def test_linear_attention_refusals():
    refused(linear(g=None), K.EINVAL, "NULL")
    refused(linear(cu=None), K.EINVAL, "NULL")
    refused(linear(s_out=None), K.EINVAL, "NULL")
    refused(linear(q=heads(128, 2, 100, K.TYPE_I32)), K.EINVAL, "f32, f16 or bf16")
    refused(linear(k=heads(128, 2, 100, K.TYPE_F16)), K.EINVAL, "one type")
    refused(linear(dst=heads(128, 6, 100, K.TYPE_F32)), K.EINVAL, "one type")
    refused(linear(q=heads(120, 2, 100), k=heads(120, 2, 100)), K.ENOTSUP, "multiples of 16")
    refused(linear(q=heads(272, 2, 100), k=heads(272, 2, 100)), K.ENOTSUP, "at most 256")
    refused(linear(v=heads(528, 6, 100), dst=heads(528, 6, 100)), K.ENOTSUP, "dv at most 512")
    refused(linear(v=heads(128, 5, 100), dst=heads(128, 5, 100)), K.EINVAL, "multiple of n_k_heads")
    refused(linear(v=heads(128, 6, 99)), K.EINVAL, "same tokens")
    refused(linear(k=heads(128, 2, 99)), K.EINVAL, "same shape")
    refused(linear(dst=heads(128, 6, 99)), K.EINVAL, "v's shape")
    refused(linear(dst=heads(128, 6, 100, stride=128 * 6 * 2 + 16)), K.EINVAL, "contiguous")
    refused(linear(q=heads(128, 2, 100, at=FAKE + 8)), K.EALIGN, "16-byte")
    refused(linear(q=heads(128, 2, 100, stride=520)), K.EALIGN, "16-byte")
    refused(linear(k=heads(128, 2, 100, stride=1 << 24)), K.ENOTSUP, "token strides")
    refused(linear(n_seq=0), K.EINVAL, "n_seq")
    refused(linear(max_len=0), K.EINVAL, "max_len")
    refused(linear(g_ts=5), K.EINVAL, "g_token_stride")
    refused(linear(n_slots=2), K.EINVAL, "slots")
    refused(linear(scale=float("nan")), K.EINVAL, "scale")
    refused(linear(s_in=FAKE + 4), K.EALIGN, "16-byte")
    refused(linear(s_in=FAKE + GB + 4096), K.EINVAL, "overlap")
    assert linear(q=heads(128, 2, 0), k=heads(128, 2, 0), v=heads(128, 6, 0), dst=heads(128, 6, 0)) == K.OK   # no tokens


class Elsewhere:
    """A [4, 1, 16, 256] float32 tensor of another device, as far as the wrappers look."""
    shape = (4, 1, 16, 256)

    def __init__(self, device=3):
        import torch
        self.dtype, self.device = torch.float32, device

    def dim(self):
        return 4

    def is_contiguous(self):
        return True

    def element_size(self):
        return 4

    def data_ptr(self):
        return FAKE + 5 * GB

    def get_device(self):
        return self.device


def test_a_gate_on_another_device_is_refused(monkeypatch):
    """Host tensors stand in for those of the current device; dst is NULL, so that the library refuses the call that passes."""
    import torch
    monkeypatch.setattr(K._Torch(), "device", staticmethod(lambda: -1))
    q, k, o = paged_views()
    o.data = None
    table, n_kv = torch.zeros((4, 40), dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    call = lambda gate: K.flash_attn_ext_paged(q, k, k, table, 16, n_kv, 0.0625, o, gate=gate, stream=0)  # noqa: E731
    for gate in (None, Elsewhere(device=-1)):
        with pytest.raises(K.QwfnError, match="dst is NULL"):
            call(gate)
    with pytest.raises(ValueError, match="gate must be on the current device"):
        call(Elsewhere())


@pytest.mark.parametrize("at", range(9))
def test_first_use_from_two_threads(monkeypatch, at):
    """A second thread that comes at the first's `at`-th question to torch, while it still fills what the wrappers keep of
    the answers, finds all of them, or fills them itself."""
    import sys
    import threading

    import torch
    names, found, asked = ("int32", "float32", "types", "device", "stream"), [], []
    K._Torch()
    for name in names:
        monkeypatch.delattr(K._Torch, name)
    monkeypatch.setattr(K._Torch, "mod", None)

    def second():
        t = K._Torch()
        found.append([n for n in names if not hasattr(t, n)])

    class Slow:
        def __getattr__(self, name):
            asked.append(name)
            if len(asked) == at + 1:
                th = threading.Thread(target=second)
                th.start()
                th.join()
            return getattr(torch, name)

    monkeypatch.setitem(sys.modules, "torch", Slow())
    K._Torch()
    assert found in ([[]], []) and (found or len(asked) <= at), (found, asked)


def spans_linear():
    """A call of linear_attn in parts, each tensor at a place of its own: the arguments, and each one's place and bytes."""
    n, n_slots = 5000, 4
    at = {name: FAKE + i * GB for i, name in enumerate(("q", "k", "v", "dst", "g", "cu", "slots", "s_in", "s_out", "ws"))}
    size = dict(q=n * 256 * 2, k=n * 256 * 2, v=n * 768 * 2, dst=n * 768 * 2, g=n * 6 * 4, cu=16, slots=12,
                s_in=n_slots * 6 * 128 * 128 * 4, s_out=n_slots * 6 * 128 * 128 * 4)
    a = dict(q=heads(128, 2, n, at=at["q"]), k=heads(128, 2, n, at=at["k"]), v=heads(128, 6, n, at=at["v"]),
             dst=heads(128, 6, n, at=at["dst"]), g=at["g"], cu=at["cu"], slots=at["slots"], s_in=at["s_in"], s_out=at["s_out"],
             ws=at["ws"], max_len=n, n_slots=n_slots)
    size["ws"] = K.load().qwfn_linear_attn_workspace_size(ctypes.byref(a["q"]), ctypes.byref(a["v"]), 3, n)
    assert size["ws"] > 0
    return a, at, size


@pytest.mark.parametrize("out", ["dst", "s_out", "ws"])
def test_linear_attention_outputs_over_other_tensors_refused(out):
    """dst, the states and the workspace over the last bytes of every other tensor."""
    label = dict(s_in="state_in", s_out="state_out")
    _, at, size = spans_linear()
    for name in at:
        if name == out:
            continue
        a, at, size = spans_linear()
        place = at[name] + (size[name] + 15) // 16 * 16 - 16
        if out == "dst":
            a["dst"].data = place
        else:
            a[out] = place
        refused(linear(**a), K.EINVAL, "overlap")
        msg = K.load().qwfn_last_error().decode()
        assert label.get(out, out) in msg and label.get(name, name) in msg, msg


@pytest.mark.parametrize("out", ["dst", "ws"])
def test_paged_attention_outputs_over_other_tensors_refused(out):
    def spans():
        q, k, o = paged_views()
        v = paged_views()[1]
        gate = paged_views()[2]
        at = {name: FAKE + i * GB for i, name in enumerate(("q", "k", "v", "dst", "gate", "table", "n_kv", "ws"))}
        for t, name in ((q, "q"), (k, "k"), (v, "v"), (o, "dst"), (gate, "gate")):
            t.data = at[name]
        row = 4 * 16 * 256 * 4
        size = dict(q=row, k=640 * 544, v=640 * 544, dst=row, gate=row, table=(3 * 43 + 40) * 4, n_kv=16,
                    ws=K.load().qwfn_fattn_workspace_size_paged(ctypes.byref(q), ctypes.byref(k), ctypes.byref(v), 40, 16))
        return dict(q=q, k=k, v=v, o=o, gate=gate, table=at["table"], stride=43, n_kv=at["n_kv"], ws=at["ws"]), at, size

    for name in ("q", "k", "v", "dst", "gate", "table", "n_kv", "ws"):
        if name == out:
            continue
        a, at, size = spans()
        place = at[name] + (size[name] + 15) // 16 * 16 - 16
        if out == "dst":
            a["o"].data = place
        else:
            a["ws"] = place
        refused(paged(**a), K.EINVAL, "overlap")
        msg = K.load().qwfn_last_error().decode()
        assert out in msg and name in msg, msg


def test_linear_attention_without_tokens_has_no_addresses():
    """An empty tensor of torch's has the address 0: a call of no tokens with it is one like another."""
    import torch
    assert torch.empty((0, 2, 64)).data_ptr() == 0
    none = lambda h: heads(128, h, 0, at=None)  # noqa: E731
    a = dict(q=none(2), k=none(2), v=none(6), dst=none(6))
    assert linear(**a) == K.OK
    assert linear(ws=None, ws_bytes=0, **a) == K.OK
    assert linear(g=None, **a) == K.OK
    assert K.load().qwfn_linear_attn_workspace_size(ctypes.byref(a["q"]), ctypes.byref(a["v"]), 3, 50) == 0
    refused(linear(**{**a, "max_len": 0}), K.EINVAL, "max_len")
    refused(linear(q=heads(128, 2, 100, at=None)), K.EINVAL, "q is NULL")


def test_linear_attention_takes_empty_tensors_of_any_strides(monkeypatch):
    """An empty tensor out of numpy has strides of 0: they say nothing, as there is nothing to step over."""
    import numpy as np
    import torch
    empty = lambda *s: torch.from_numpy(np.zeros(s, np.float32))  # noqa: E731
    assert empty(0, 4).stride() == (0, 0)
    monkeypatch.setattr(K._Torch(), "device", staticmethod(lambda: -1))         # host tensors stand in; nothing is launched
    q, v, g, state = empty(0, 2, 64), empty(0, 4, 64), empty(0, 4), torch.zeros((3, 4, 64, 64))
    assert K.linear_attn_workspace_size(q, v, 3, 50) == 0
    K.linear_attn(q, q, v, g, torch.zeros(4, dtype=torch.int32), 50, state, state, empty(0, 4, 64), stream=0)


def test_extend_states_refusals():
    def call(states=FAKE + 10 * GB, state_slots=FAKE + 11 * GB, **kw):
        a = dict(past=FAKE, new=FAKE + GB, n_seq=4, page=16, table=FAKE + 2 * GB, stride=8, cols=8, free=FAKE + 3 * GB, cap=10,
                 n_free=FAKE + 4 * GB, n_free_out=FAKE + 5 * GB, n_kv=FAKE + 6 * GB, cu=FAKE + 7 * GB, slots=FAKE + 8 * GB,
                 pos=None, seq=None, n_tok=9, pad=-1)
        a.update(kw)
        return K.load().qwfn_paged_extend_states(*a.values(), states, state_slots, FAKE + 9 * GB, 1 << 20, None)
    refused(call(state_slots=None), K.EINVAL, "NULL")
    refused(call(n_seq=0), K.EINVAL, "n_seq")
    refused(call(state_slots=FAKE + 11 * GB + 2), K.EALIGN, "state_slots")
    refused(call(states=FAKE + 10 * GB + 1), K.EALIGN, "states")
    refused(call(states=FAKE + 11 * GB + 12), K.EINVAL, "state_slots overlaps states")
    refused(call(state_slots=FAKE + 4), K.EINVAL, "state_slots overlaps n_past")
    refused(call(state_slots=FAKE + 8 * GB + 32), K.EINVAL, "state_slots overlaps slots")
