"""The workspaces that the paged operators keep: one per context and stream, so
that threads which share a stream, with a context each, do not meet in one."""
import contextlib
import threading
import types

import pytest
import torch

from _paged import Pool, attend, tolerance


class _Ctx:
    def __init__(self):
        self.workspaces = {}


@pytest.fixture
def paged(monkeypatch):
    """The module with torch's CUDA calls replaced by ones that work on the CPU; ``state`` sets stream and capture."""
    from streaming_attention_b200 import paged
    state = types.SimpleNamespace(stream=7, capturing=False, device=0, other_capturing=False)

    @contextlib.contextmanager
    def device(dev):
        before, state.device = state.device, dev
        yield
        state.device = before

    fake = types.SimpleNamespace(
        uint8=torch.uint8,
        zeros=lambda n, dtype, device: torch.zeros(n, dtype=dtype),
        empty=lambda n, dtype, device: torch.full((n,), 9, dtype=dtype),
        cuda=types.SimpleNamespace(device=device),
        _C=types.SimpleNamespace(_cuda_isCurrentStreamCapturing=lambda: state.capturing if state.device == 0
                                 else state.other_capturing,
                                 _cuda_getCurrentRawStream=lambda dev: state.stream,
                                 _cuda_getDevice=lambda: state.device))
    monkeypatch.setattr(paged, "_torch", fake)
    paged.state = state
    return paged


def test_one_per_context_and_stream(paged):
    a, b = _Ctx(), _Ctx()
    first = paged._workspace(a, 0, 9000)
    assert paged._workspace(a, 0, 5000) is first                # kept, and grown only
    assert paged._workspace(b, 0, 5000).data_ptr() != first.data_ptr()      # another thread's on the same stream
    paged.state.stream = 8
    assert paged._workspace(a, 0, 9000).data_ptr() != first.data_ptr()
    paged.state.stream = 7
    assert paged._workspace(a, 0, 9000) is first
    grown = paged._workspace(a, 0, 20000)
    assert grown.numel() == 20000 and not grown.any() and paged._workspace(a, 0, 9000) is grown


def test_a_captured_call_has_its_own_with_a_zero_head(paged):
    a = _Ctx()
    kept = paged._workspace(a, 0, 9000)
    paged.state.capturing = True
    one, two = paged._workspace(a, 0, 9000), paged._workspace(a, 0, 9000)
    assert len({kept.data_ptr(), one.data_ptr(), two.data_ptr()}) == 3
    assert not one[:4096].any() and not two[:4096].any()
    paged.state.capturing = False
    assert paged._workspace(a, 0, 9000) is kept


def test_the_capture_is_looked_for_on_the_pages_gpu(paged):
    """Pages on GPU 0 while GPU 1 is the current one: whose stream is captured decides."""
    a = _Ctx()
    kept = paged._workspace(a, 0, 9000)
    paged.state.device, paged.state.other_capturing = 1, True
    assert paged._workspace(a, 0, 9000) is kept                 # GPU 1's capture is not this call's
    paged.state.other_capturing, paged.state.capturing = False, True
    own = paged._workspace(a, 0, 9000)
    assert own.data_ptr() != kept.data_ptr() and not own[:4096].any()
    assert paged.state.device == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_threads_on_one_stream(dtype):
    """Threads on torch's default stream, a context each: decodes of one launch and prefix calls of two and three,
    enqueued at once, give what they give one after the other."""
    import streaming_attention_b200 as sa
    jobs = []
    for i, (lens, prefix, hq, hkv) in enumerate([([300, 5, 0, 64], 1000, 8, 2),            # joined in the decode
                                                 ([i % 90 for i in range(40)], 3000, 8, 2),    # joined by a kernel
                                                 ([2000, 17, 900], 200, 4, 1),
                                                 ([50] * 20, 5000, 16, 4)]):
        pool = Pool([prefix] + lens, hkv, 128, 16, dtype, seed=40 + i)
        q = pool.q(len(lens), hq)
        jobs.append((pool, prefix, q.cuda(), q))

    def calls(job, ctx):
        pool, prefix, q, _ = job
        args = (pool.kp, pool.vp)
        return (sa.attn_paged_decode_prefix(q, *args, pool.table[0], prefix, pool.table[1:], pool.kv_lens[1:], 0.1, ctx=ctx),
                sa.attn_paged_decode(q, *args, pool.table[1:], pool.kv_lens[1:], 0.1, ctx=ctx))

    ctxs = [sa.Context(0) for _ in jobs]
    want = [calls(j, c) for j, c in zip(jobs, ctxs)]
    torch.cuda.synchronize()
    pool, prefix, _, q = jobs[0]
    ref = attend(q[:1], torch.cat([pool.k[0], pool.k[1]], 1), torch.cat([pool.v[0], pool.v[1]], 1), [prefix + 299], 0.1)
    v_max = max(pool.v[0].abs().max().item(), pool.v[1].abs().max().item())
    assert ((want[0][0][:1].double().cpu() - ref).abs() <= tolerance(dtype, ref, v_max)).all()
    got, errors = [[] for _ in jobs], []
    gate = threading.Barrier(len(jobs))

    def work(i):
        try:
            gate.wait()
            for _ in range(150):
                got[i].append(calls(jobs[i], ctxs[i]))
        except Exception as e:                          # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for i, job in enumerate(want):
        for pair in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(pair, job)), i
    for c in ctxs:
        c.synchronize()
        c.close()
