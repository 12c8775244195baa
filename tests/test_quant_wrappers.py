"""What the Python calls of the quantised operators refuse before anything is launched, and whose memory they use."""
import contextlib
import types

import pytest
import torch


def test_rows_that_overlap_have_no_stride(gsv):
    from gsv_b200 import quant

    assert quant._row_stride(torch.zeros(1, 8).expand(1, 8), 1, 8, "x") == 8
    assert quant._row_stride(torch.zeros(4, 12)[:, :8], 4, 8, "x") == 12
    for t in (torch.zeros(8).expand(4, 8), torch.zeros(40).as_strided((4, 8), (7, 1))):
        with pytest.raises(ValueError, match="overlap"):
            quant._row_stride(t, 4, 8, "x")


@pytest.mark.gpu
def test_expanded_tensors_are_refused(dev):
    """A broadcast row, weight or residual: its stride of 0 must not reach the C ABI."""
    x = torch.zeros(64, device="cuda")
    a = torch.zeros(4, 64, dtype=torch.int8, device="cuda")
    s = torch.ones(64, device="cuda")
    wide, wide8 = x.expand(4, 64), a[0].expand(4, 64)
    for call in (lambda: dev.quantize_rows_i8(wide), lambda: dev.quantize_rows_i8(wide.half()[:1].expand(4, 64)),
                 lambda: dev.quantize_rows_i8(x.repeat(4, 1), q=wide8), lambda: dev.gemm_i8(wide8, s, a, s),
                 lambda: dev.gemm_i8(a, s, wide8, s), lambda: dev.gemm_i8(a, s, a, s, residual=x[:4].expand(4, 4)),
                 lambda: dev.gemm_i8(a, s, a, s, residual=x[:1].expand(4, 4)),
                 lambda: dev.gemm_i8(a, s, a, s, c=x[:4].expand(4, 4)),
                 lambda: dev.gemm_i8(a, s, a, s, c_f16=x[:4].half().expand(4, 4))):
        with pytest.raises(ValueError):
            call()
    # one row has no stride
    assert dev.gemm_i8(a[:1].expand(1, 64), s, a, s, residual=x[:4].expand(1, 4)).shape == (1, 4)


def test_outputs_on_another_stream_are_its_memory(gsv, monkeypatch):
    """The allocator is asked from within the call's stream, and told of the one that reads the result."""
    from gsv_b200 import quant

    asked, told, inside = [], [], []

    @contextlib.contextmanager
    def use(stream):
        inside.append(stream)
        yield
        inside.pop()

    def empty(shape, **kw):
        asked.append(inside[-1] if inside else "current")
        return types.SimpleNamespace(record_stream=told.append)

    monkeypatch.setattr(torch.cuda, "stream", use)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: inside[-1] if inside else "current")
    monkeypatch.setattr(torch, "empty", empty)
    for stream in (None, "other"):
        quant._allocator(stream)((2, 3), dtype=torch.float16, device="cuda:0")
    assert asked == ["current", "other"] and told == ["current"]


@pytest.mark.gpu
def test_outputs_on_another_stream_are_not_the_current_ones_memory(dev):
    """Blocks that the current stream has given back may still be written by its queued work: a call on another stream gets
    none of them."""
    other = torch.cuda.Stream()
    x = torch.randn(2048, 1024, device="cuda").half()
    w, ws = dev.quantize_rows_i8(x)
    c = dev.KV4Cache.empty(8, 64, 4, 128)
    slots = torch.arange(512, device="cuda")
    c.append(x.view(-1, 4, 128)[:512], x.view(-1, 4, 128)[:512], slots)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table, space = torch.arange(8, dtype=torch.int32, device="cuda")[None], dev.KV4Workspace(1, 512, 4, 4, 128)
    rows, q_start, kv_len = x.view(-1, 4, 128)[:512], i32(0, 512), i32(512)
    calls = (lambda s: dev.quantize_rows_i8(x, stream=s), lambda s: [dev.gemm_i8(w, ws, w, ws, stream=s)],
             lambda s: c.read(slots, stream=s),
             lambda s: [c.attention(rows, q_start, kv_len, table, 0.1, 512, space, stream=s)])
    torch.cuda.synchronize()
    for call in calls:
        given_back = {t.data_ptr() for t in call(None)}
        torch.cuda.synchronize()
        out = call(other)
        other.synchronize()
        assert not given_back & {t.data_ptr() for t in out}


def _foreign(index):
    """What the checks ask of a contiguous fp32 tensor [4, 8] on a device."""
    return types.SimpleNamespace(dtype=torch.float32, is_cuda=True, shape=(4, 8), dim=lambda: 2, stride=lambda i: (8, 1)[i],
                                 is_contiguous=lambda: True, numel=lambda: 32, data_ptr=lambda: 256, get_device=lambda: index)


def test_tensors_streams_and_buffers_of_another_device_are_refused(gsv, monkeypatch):
    from gsv_b200 import quant

    for f in (lambda t: quant._tensor(t, torch.float32, 2, "x", 0), lambda t: quant._vector(t, torch.float32, 32, "x", 0)):
        assert f(_foreign(0)) == 256
        with pytest.raises(ValueError, match="cuda:1"):
            f(_foreign(1))
    stream = types.SimpleNamespace(cuda_stream=77, device_index=1)
    assert quant._stream_for(stream, 1) == 77
    with pytest.raises(ValueError, match="cuda:1"):
        quant._stream_for(stream, 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    for make in (lambda d: gsv.KVPlan(2, 4, 16, 8, 8, device=d), lambda d: gsv.KV4Workspace(2, 2, 2, 2, 32, device=d),
                 lambda d: gsv.KV4Cache.empty(2, 16, 2, 32, device=d)):
        for device in ("cuda:1", torch.device("cuda", 1), "cpu"):
            with pytest.raises(ValueError, match="current device"):
                make(device)


@pytest.mark.gpu
def test_calls_run_where_the_current_device_is(dev, monkeypatch):
    """With another device current, every call refuses this one's tensors; given as the current one, a device is taken."""
    from gsv_b200 import quant

    x = torch.randn(4, 64, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q, s = dev.quantize_rows_i8(x)
    for device in (None, "cuda", "cuda:0", torch.device("cuda", 0)):
        c, ws = dev.KV4Cache.empty(4, 16, 2, 32, device=device), dev.KV4Workspace(1, 4, 2, 2, 32, device=device)
        p = dev.KVPlan(1, 4, 16, 4, 4, device=device)
    rows, slots, table = x.view(4, 2, 32).half(), torch.arange(4, device="cuda"), i32(0, 1, 2, 3)[None]
    plan = (i32(0), i32(4), table, i32(0, 1, 2, 3), i32(4))
    calls = (lambda: dev.quantize_rows_i8(x), lambda: dev.gemm_i8(q, s, q, s), lambda: c.append(rows, rows, slots),
             lambda: c.read(slots), lambda: c.attention(rows, i32(0, 4), i32(4), table, 0.1, 4, ws), lambda: p.run(*plan),
             lambda: p.release(i32(1), *plan[0:1], *plan[2:]))
    for call in calls:
        call()
    monkeypatch.setattr(quant, "_device", lambda: 1)
    for call in calls:
        with pytest.raises(ValueError, match="cuda:0"):
            call()
    monkeypatch.undo()
    ws.index = 1
    with pytest.raises(ValueError, match="workspace"):
        calls[4]()
    for held, at in ((c, (2, 3, 4)), (p, (5, 6))):  # memory of another device behind arguments of this one
        held._index = 1
        for i in at:
            with pytest.raises(ValueError, match="cuda:1"):
                calls[i]()


def test_buffers_are_filled_before_a_constructor_returns(gsv, monkeypatch):
    from gsv_b200 import quant

    waited = []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: types.SimpleNamespace(synchronize=lambda: waited.append(1)))
    monkeypatch.setattr(quant, "_device_for", lambda device: torch.device("cpu"))
    gsv.KVPlan(2, 4, 16, 8, 8)
    gsv.KV4Workspace(2, 2, 2, 2, 32)
    assert len(waited) == 2


@pytest.mark.gpu
def test_new_buffers_serve_another_stream(dev):
    """Made behind queued work of the current stream, used at once on another one."""
    other = torch.cuda.Stream()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    rows = torch.randn(512, 4, 64, device="cuda").half()
    cache, slots = dev.KV4Cache.empty(64, 16, 4, 64), torch.arange(512, device="cuda")
    cache.append(rows, rows, slots)
    table, q_start, kv_len = torch.arange(32, dtype=torch.int32, device="cuda")[None], i32(0, 512), i32(512)
    state = (i32(0), i32(512), i32(*range(32))[None], i32(*range(64)), i32(64))
    out = [torch.empty_like(rows) for _ in range(2)]
    torch.cuda.synchronize()
    cache.attention(rows, q_start, kv_len, table, 0.1, 512, dev.KV4Workspace(1, 512, 4, 4, 64), out=out[0])
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)  # some 50 ms
    ws, plan = dev.KV4Workspace(1, 512, 4, 4, 64), dev.KVPlan(1, 32, 16, 64, 512)
    cache.attention(rows, q_start, kv_len, table, 0.1, 512, ws, out=out[1], stream=other)
    plan.run(*state, stream=other)
    other.synchronize()
    assert torch.equal(out[0], out[1])
    assert plan.q_start.tolist() == [0, 512] and plan.slots.tolist() == [(63 - i // 16) * 16 + i % 16 for i in range(512)]


@pytest.mark.gpu
def test_memory_of_a_call_on_another_stream_is_kept_until_it_has_run(dev):
    """Inputs that are given up while the call is still queued: their memory goes to nobody before it has run."""
    other = torch.cuda.Stream()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    n = 1024
    table, q_start, kv_len = torch.arange(64, dtype=torch.int32, device="cuda")[None], i32(0, n), i32(n)
    slots = torch.arange(n, device="cuda")
    rows = lambda: torch.ones(n, 4, 128, dtype=torch.float16, device="cuda")  # noqa: E731
    codes = lambda: torch.ones(n, 1024, dtype=torch.int8, device="cuda")  # noqa: E731
    cache = dev.KV4Cache.empty(64, 16, 4, 128)
    space = dev.KV4Workspace(1, n, 4, 4, 128)
    one, out, i8 = torch.ones(n, device="cuda"), rows(), codes()

    def quantise(x):
        dev.quantize_rows_i8(x, stream=other)

    def attention(q):
        cache.attention(q, q_start, kv_len, table, 0.1, n, space, out=out, stream=other)

    makes = ((lambda: torch.ones(n, 1024, device="cuda"), quantise), (rows, attention),
             (codes, lambda a: dev.gemm_i8(a, one, i8, one, stream=other)),
             (codes, lambda b: dev.gemm_i8(i8, one, b, one, stream=other)),
             (rows, lambda k: cache.append(k, out, slots, stream=other)),
             (lambda: torch.empty(1 << 20, dtype=torch.int64, device="cuda").fill_(-1), lambda s: cache.read(s, k=out_wide, stream=other)),
             (lambda: dev.KV4Cache.empty(256, 16, 4, 128), lambda c: c.append(out, out, slots, stream=other)),
             (lambda: dev.KV4Workspace(1, n, 4, 4, 128), lambda ws: cache.attention(out, q_start, kv_len, table, 0.1, n, ws, out=out,
                                                                                  stream=other)))
    out_wide = torch.empty(1 << 20, 4, 128, dtype=torch.float16, device="cuda")
    cache.append(out, out, slots)
    for make, call in makes:
        given = make()
        t = given.pages if isinstance(given, dev.KV4Cache) else given.buffer if isinstance(given, dev.KV4Workspace) else given
        shape, dtype, at = t.shape, t.dtype, t.data_ptr()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            torch.cuda._sleep(20_000_000)  # some 10 ms
        call(given)
        del given, t
        again = torch.empty(shape, dtype=dtype, device="cuda")
        assert again.data_ptr() != at
        other.synchronize()
