"""The bounded-cache operators' refusals and host bookkeeping (no GPU needed)."""

import contextlib
import ctypes
import random
import re
import threading
import time

import pytest
import torch

from nano_vllm_b200 import DevicePageTable, TinyKvPagedCache, TinyKvPagedPool, evict_tokens, flash_attention, paged_attention
from nano_vllm_b200 import _native as nv


def test_window_arguments_are_checked_first():
    q, k = torch.zeros(1, 4, 1, 64), torch.zeros(1, 2, 8, 64)
    pages, bt, cl = torch.zeros(2, 2, 16, 64), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for w in (0, -1):
        with pytest.raises(RuntimeError, match="flash_attention: window must be at least 1"):
            flash_attention(q, k, k, window=w)
        with pytest.raises(RuntimeError, match="paged_attention: window must be at least 1"):
            paged_attention(q, pages, pages, bt, cl, 16, window=w)
    with pytest.raises(RuntimeError, match="sinks must not be negative"):
        flash_attention(q, k, k, window=4, sinks=-1)
    with pytest.raises(RuntimeError, match="sinks must not be negative"):
        paged_attention(q, pages, pages, bt, cl, 16, window=4, sinks=-2)


def test_operators_have_no_cpu_path():
    q, k = torch.zeros(1, 4, 1, 64), torch.zeros(1, 2, 8, 64)
    pages, bt, cl = torch.zeros(2, 2, 16, 64), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA device"):
        flash_attention(q, k, k, window=4)
    with pytest.raises(RuntimeError, match="CUDA device"):
        paged_attention(q, pages, pages, bt, cl, 16, window=4)
    with pytest.raises(RuntimeError, match="CUDA device"):
        evict_tokens(pages, pages, bt, cl, torch.zeros(1, 2, 32), 4)


def _window_call(**kw):
    a = dict(B=1, Hq=4, Hkv=2, L=1, D=128, P=4, ps=16, mp=4, window=8, sinks=0, mass=None, sb=0, sh=0, ml=0, kv=2)
    a.update(kw)
    return nv.lib().nvm_paged_attention_window(None, 2, None, None, a["kv"], None, None, 1, None, None, None, 0, a["B"],
                                               a["Hq"], a["Hkv"], a["L"], a["D"], a["P"], a["ps"], a["mp"], 0.1, 1,
                                               a["window"], a["sinks"], a["mass"], a["sb"], a["sh"], a["ml"], None, 0, None)


def test_c_entry_refusals():
    L = nv.lib()
    assert _window_call() == -1  # null tensors
    assert _window_call(B=0) == 0
    assert _window_call(B=0, window=-1) == -1
    assert L.nvm_last_error().decode() == "paged_attention: window must be positive, or 0 for none"
    assert _window_call(B=0, sinks=-1) == -1
    assert _window_call(B=0, window=1 << 40) == -2
    assert _window_call(Hq=3) == -1
    assert _window_call(D=512) == -2
    args = [None, None, None, 2, None, 0, 1, 4, 2, 8, 8, 64, 0.1, 1]
    assert L.nvm_flash_attention_window(*args, 4, 0, None) == -1
    assert L.nvm_flash_attention_window(*args, -4, 0, None) == -1


def test_workspace_sizes():
    size = nv.lib().nvm_paged_attention_window_workspace_size
    assert size(1, 3, 2, 1, 128, 16, 8, 2, 64, 0, 0) == 0  # refused sizes need none
    with_mass = size(2, 32, 8, 1, 128, 16, 8, 2, 0, 0, 1)
    assert with_mass >= (1 << 20) + 2 * 32 * 4  # the first MiB holds tickets that stay zero
    assert with_mass > size(2, 32, 8, 1, 128, 16, 8, 2, 0, 0, 0)


def _window_workspace_required(causal, B, Hq, Hkv, L, D, ps, mp, kv, window, sinks, mass):
    """What the entry says it needs.  It refuses a missing workspace before any launch; with ``mass`` it always
    needs one, so the addresses below (any that are aligned) are never used."""
    L_ = nv.lib()
    at, q_dtype, scale_dtype = 1 << 20, 1 if kv == 3 else kv, 1
    st = L_.nvm_paged_attention_window(at, q_dtype, at, at, kv, at, at, scale_dtype, at, at, at, 0, B, Hq, Hkv, L, D, 64, ps, mp,
                                       0.1, causal, window, sinks, at if mass else None, Hkv * mp * ps, mp * ps, mp * ps, None, 0,
                                       None)
    if st != -3:
        assert not mass
        return 0
    return int(re.search(r"workspace of (\d+) bytes", L_.nvm_last_error().decode()).group(1))


def test_workspace_size_covers_what_the_call_needs():
    rng = random.Random(4)
    shapes = [(1, 8, 8, 512, 64, 16, 64, 2, 64, 0), (2, 8, 8, 1024, 128, 16, 128, 3, 256, 4), (1, 2, 1, 1024, 128, 16, 64, 2, 64, 0)]
    for _ in range(1500):
        Hkv = rng.choice([1, 2, 8])
        shapes.append((rng.randint(1, 40), Hkv * rng.choice([1, 4, 7, 8]), Hkv, int(2 ** rng.uniform(0, 11)), rng.choice([64, 128]),
                       rng.choice([16, 128]), rng.randint(1, 300), rng.choice([1, 2, 3]),
                       rng.choice([0, int(2 ** rng.uniform(0, 12))]), rng.choice([0, 4, 100])))
    size = nv.lib().nvm_paged_attention_window_workspace_size
    for shape in shapes:
        # without a workspace to miss, a call of those addresses would reach the GPU, so only where there is none
        for mass in (0, 1) if not torch.cuda.is_available() else (1,):
            for causal in (0, 1):
                need = _window_workspace_required(causal, *shape, mass)
                assert size(*shape, mass) >= need, (shape, causal, mass, need)


def test_more_units_than_merge_tickets_go_in_parts():
    """257 prompts of 1024 row blocks are 263168 units, the first MiB of the workspace holds 262144 tickets:
    two launches of at most 129 prompts, in the workspace of one of them."""
    L_ = nv.lib()
    base = lambda B: L_.nvm_paged_attention_workspace_size(B, 8, 1, 8192, 64, 16, 545, 2)  # noqa: E731
    window = lambda B, w=5000: L_.nvm_paged_attention_window_workspace_size(B, 8, 1, 8192, 64, 16, 545, 2, w, 4, 0)  # noqa: E731
    assert base(257) == base(129) > base(128) > 1 << 20
    assert window(257) == window(129) > window(128) > 1 << 20
    assert L_.nvm_paged_attention_workspace_size(2, 8, 1, 262144 * 9, 64, 16, 545, 2) == 0  # too many in one prompt


@pytest.mark.parametrize("L,Hq", [(1, 64), (1, 32), (2, 32), (1, 8)])
def test_kept_scores_do_not_grow_with_the_batch(L, Hq):
    """4 bytes a query row (their number made even) and key of the table: kept for 2.25 GiB's worth of requests at a
    time."""
    size = lambda B, width: nv.lib().nvm_paged_attention_window_workspace_size(B, Hq, 8, L, 128, 16, width // 16, 2, 0, 0, 1)  # noqa: E731
    bare = lambda B, width: nv.lib().nvm_paged_attention_workspace_size(B, Hq, 8, L, 128, 16, width // 16, 2)  # noqa: E731
    for B, width in ((64, 131072), (256, 131072), (300, 70000), (1024, 40000), (77, 1 << 20)):
        assert size(B, width) <= (9 << 28) + bare(B, width) + (1 << 22), (B, width, size(B, width), bare(B, width))
    one = 8 * ((L * Hq // 8 + 1) // 2 * 2) * 4 << 23  # one request is never split
    assert one <= size(1, 1 << 23) <= 1.02 * one + bare(1, 1 << 23) + (1 << 22)


def test_evict_c_entry_refusals():
    def call(B=1, D=128, budget=4, sinks=0, recent=0, kv=2, sb=8):
        return nv.lib().nvm_paged_evict(None, None, kv, None, None, 1, None, None, None, None, sb, 8, 8, None, 8, 8, B, 2, D,
                                        4, 16, 4, budget, sinks, recent, None, None, None, None, None, None)
    assert call() == -1
    assert call(B=0) == 0
    for bad in (dict(budget=0), dict(sinks=-1), dict(recent=-1), dict(sinks=3, recent=2), dict(kv=4), dict(sb=-1)):
        assert call(B=0, **bad) == -1, bad
    assert call(B=0, D=300) == -2


@pytest.mark.parametrize("ps,pages", [(16, 1 << 27), (1 << 20, 2048), (7, (1 << 31) // 7)])
def test_evict_refuses_rows_past_its_32_bit_positions(ps, pages):
    """A sweep looks up to 32 * 1024 positions past a row's end."""
    def call(S, mp):
        return nv.lib().nvm_paged_evict(None, None, 2, None, None, 1, None, None, None, None, S, S, S, None, S, S, 0, 2, 128, 4, ps,
                                        mp, 4, 0, 0, None, None, None, None, None, None)
    assert call(2 ** 31 - 1, pages) == -2 and call(2 ** 31 - 65536, pages) == -2 and call(1 << 40, pages) == -2
    assert call(2 ** 31 - 65537, pages) == 0 and call(1 << 40, pages // 2) == 0


def test_request_cache_evict_checks_on_the_host():
    pool = TinyKvPagedPool(page_size=4)
    cache = TinyKvPagedCache(pool)
    cache.plan_append(10)
    mass = torch.zeros(1, 2, 16)
    assert cache.evict(mass, 10) is None and cache.evict(mass, 32, sinks=4) is None
    for bad in (dict(budget=0), dict(budget=4, sinks=3, recent=2), dict(budget=4, sinks=-1)):
        with pytest.raises(RuntimeError, match="budget"):
            cache.evict(mass, **bad)
    with pytest.raises(RuntimeError, match="key_mass"):
        cache.evict(torch.zeros(1, 2, 9), 8)
    pool.incref(cache.page_ids[1])
    with pytest.raises(ValueError, match="shared"):
        cache.evict(mass, 8)
    assert cache.offset == 10 and cache.num_pages == 3


def test_evict_refuses_a_mass_out_that_overlaps(monkeypatch):
    """Rows would be written where other requests' weights have yet to be read."""
    calls = []

    class Lib:
        def nvm_paged_evict(self, *args):
            calls.append(args)
            return 0

    monkeypatch.setattr(nv, "lib", Lib)
    monkeypatch.setattr(nv, "require_cuda", lambda op, *t: torch.device("cpu"))
    monkeypatch.setattr(nv, "stream_ptr", lambda dev: 0)
    k, v = (torch.zeros(8, 2, 16, 64) for _ in range(2))
    bt, cl, store = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(1000)
    mass = store[100:484].view(3, 2, 64)
    for at in (99, 101, 100 - 383, 483):
        with pytest.raises(RuntimeError, match="mass_out"):
            evict_tokens(k, v, bt, cl, mass, 8, mass_out=store[max(at, 0):max(at, 0) + 384].view(3, 2, 64))
    assert calls == []
    evict_tokens(k, v, bt, cl, mass, 8, mass_out=mass)
    evict_tokens(k, v, bt, cl, mass, 8, mass_out=store[484:868].view(3, 2, 64))
    both = torch.zeros(3, 2, 2, 64)  # side by side, row after row
    evict_tokens(k, v, bt, cl, both[:, 0], 8, mass_out=both[:, 1])
    assert len(calls) == 3


def _layer(int8=False, P=8, D=64):
    dt = torch.int8 if int8 else torch.bfloat16
    k, v = (torch.zeros(P, 2, 16, D, dtype=dt) for _ in range(2))
    scales = [torch.zeros(P, 2, 16, 1, dtype=torch.float16) for _ in range(2)] if int8 else []
    return (k, v, *scales, torch.zeros(1, 2, 64))


def _changed(layer, **at):
    layer = list(layer)
    for i, x in at.items():
        layer[int(i[1:])] = x
    return tuple(layer)


def test_table_evict_checks_every_layer_before_it_launches_any(monkeypatch):
    calls = []

    class Lib:
        def nvm_paged_evict(self, *args):
            calls.append(args)
            return 0

    monkeypatch.setattr(nv, "lib", Lib)
    monkeypatch.setattr(nv, "require_cuda", lambda op, *t: torch.device("cpu"))
    monkeypatch.setattr(nv, "stream_ptr", lambda dev: 0)
    table = DevicePageTable(1, 4, 16, 8, device="cpu")
    monkeypatch.setattr(table, "rewind", lambda n: calls.append("rewind"))
    good, other, wide = _layer(), _layer(int8=True), _layer(D=32)
    assert len(table.evict([good, other, wide], 20)) == 3 and len(calls) == 4 and calls[-1] == "rewind"
    calls.clear()
    shared = _layer()
    for bad in (_changed(_layer(), i2=torch.zeros(1, 2, 64, dtype=torch.float64)),  # weights of another type,
                _changed(_layer(), i2=torch.zeros(1, 3, 64)),                       # of other heads,
                _changed(_layer(), i2=torch.zeros(2, 2, 64)),                       # another batch,
                _changed(_layer(), i2=torch.zeros(1, 2, 128)[:, :, ::2]),           # with gaps between them
                _layer(int8=True)[:2] + _layer()[2:],                               # 8-bit pages without scales
                _changed(_layer(int8=True), i2=torch.zeros(8, 2, 16, dtype=torch.float16)),
                _changed(_layer(), i1=torch.zeros(8, 2, 16, 64, dtype=torch.float16)),  # K and V of two types
                _changed(_layer(), i0=torch.zeros(8, 2, 64, 16).bfloat16().transpose(2, 3)),
                _layer(D=300),
                _changed(_changed(_layer(), i0=torch.zeros(8, 2, 16, 64, dtype=torch.int32)),
                         i1=torch.zeros(8, 2, 16, 64, dtype=torch.int32)),
                _changed(_changed(_layer(int8=True), i2=torch.zeros(8, 2, 16, 1, dtype=torch.int32)),
                         i3=torch.zeros(8, 2, 16, 1, dtype=torch.int32)),
                _changed(shared, i1=shared[0]),                                     # K is V
                _changed(_layer(), i0=good[0]),                                     # pages of the other layer
                _changed(_layer(), i1=good[1]),
                _changed(_layer(), i2=good[2])):                                    # weights of the other layer
        with pytest.raises((RuntimeError, ValueError), match="evict"):
            table.evict([good, bad], 20)
        assert calls == []


class _Turns:
    """Counts how many threads are inside at once."""

    def __init__(self, inside=lambda: time.sleep(0.02)):
        self.now = self.most = 0
        self.inside, self.lock = inside, threading.Lock()

    def __call__(self, *args):
        with self.lock:
            self.now += 1
            self.most = max(self.most, self.now)
        self.inside()
        with self.lock:
            self.now -= 1
        return 0


def _in_threads(n, f):
    failed = []

    def run(i):
        try:
            f(i)
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_threads_on_one_stream_take_turns(monkeypatch):
    """The kernels of a call find what its first one left in the stream's workspace."""
    dev = torch.device("cuda", 0)
    streams = {}
    monkeypatch.setattr(nv, "stream_ptr", lambda d: streams.get(threading.get_ident(), 7))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    call = _Turns()
    _in_threads(4, lambda i: [nv.call_with_workspace(dev, lambda: 0, call) for _ in range(3)])
    assert call.most == 1
    both = _Turns(threading.Barrier(2, timeout=20).wait)  # streams of their own: side by side

    def other_stream(i):
        streams[threading.get_ident()] = 100 + i
        nv.call_with_workspace(dev, lambda: 0, both)

    _in_threads(2, other_stream)
    assert both.most == 2


def test_a_call_inside_a_call_of_the_same_thread(monkeypatch):
    """As a signal handler makes it, between a refused workspace and the larger one."""
    dev, calls = torch.device("cuda", 0), []
    monkeypatch.setattr(nv, "stream_ptr", lambda d: 8)
    monkeypatch.setattr(nv, "workspace", lambda d, n: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)

    def inner(*args):
        calls.append("inner")
        return 0

    def outer(*args):
        calls.append("outer")
        return nv.NVM_ERR_WORKSPACE if calls == ["outer"] else 0

    def size():
        nv.call_with_workspace(dev, lambda: 0, inner)
        return 0

    t = threading.Thread(target=nv.call_with_workspace, args=(dev, size, outer), daemon=True)
    t.start()
    t.join(20)
    assert not t.is_alive() and calls == ["outer", "inner", "outer"]


def test_threads_on_one_stream_take_turns_without_a_window(monkeypatch):
    call = _Turns()

    class Lib:
        nvm_paged_attention = call
        nvm_paged_attention_workspace_size = staticmethod(lambda *args: 0)

    monkeypatch.setattr(nv, "lib", lambda: Lib)
    monkeypatch.setattr(nv, "require_cuda", lambda op, *t: torch.device("cuda", 0))
    monkeypatch.setattr(nv, "stream_ptr", lambda d: 7)
    monkeypatch.setattr(nv, "on_device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    pages, q = torch.zeros(2, 2, 16, 64), torch.zeros(1, 4, 1, 64)
    bt, cl = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    _in_threads(4, lambda i: [paged_attention(q, pages, pages, bt, cl, 16, out=torch.zeros_like(q)) for _ in range(3)])
    assert call.most == 1


@pytest.mark.parametrize("window", [None, 8])
def test_a_capture_has_a_workspace_of_its_own(monkeypatch, window):
    """A graph replays with the addresses it captured, beside other graphs and whatever eager calls need: its calls
    share a buffer whose tickets it zeroes itself, and the stream's buffer stays out of it."""
    seen, capture, need = [], [5], [2 << 20]

    def attend(*args):
        ws, nbytes = args[-3], args[-2]
        if nbytes < need[0]:
            return nv.NVM_ERR_WORKSPACE
        seen.append((ws, ctypes.string_at(ws, 1 << 20) == bytes(1 << 20)))
        ctypes.memset(ws + (1 << 20), 7, nbytes - (1 << 20))  # the tickets are zero again
        return 0

    class Lib:
        nvm_paged_attention = nvm_paged_attention_window = staticmethod(attend)
        nvm_paged_attention_workspace_size = nvm_paged_attention_window_workspace_size = staticmethod(lambda *args: need[0])

    monkeypatch.setattr(nv, "lib", lambda: Lib)
    monkeypatch.setattr(nv, "require_cuda", lambda op, *t: torch.device("cpu"))
    monkeypatch.setattr(nv, "stream_ptr", lambda d: 9)
    monkeypatch.setattr(nv, "capture_id", lambda s: capture[0], raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capture[0] != 0)
    monkeypatch.setattr(nv, "_workspaces", {})
    monkeypatch.setattr(nv, "_captured", {}, raising=False)
    pages, q = torch.zeros(2, 2, 16, 64), torch.zeros(1, 4, 1, 64)
    bt, cl = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)

    def run():
        paged_attention(q, pages, pages, bt, cl, 16, window=window, out=torch.zeros_like(q))
        at, zero = seen[-1]
        assert zero
        return at

    first = run()
    assert run() == first and nv._workspaces == {}
    held = nv._captured[(0, 9)][1]  # as the graph's pool would
    capture[0] = 0
    eager = run()
    assert eager != first and [ws.data_ptr() for ws in nv._workspaces.values()] == [eager]
    capture[0] = 6  # another graph on the same stream
    other = run()
    assert other not in (first, eager) and run() == other
    need[0] = 4 << 20
    larger = run()
    assert larger != other and run() == larger
    capture[0] = 0
    run()
    assert held.data_ptr() == first
