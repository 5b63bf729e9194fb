"""Host side of the serving operators on the CPU: a stand-in for the library
that records its calls, and stand-ins for tensors on a GPU."""
import threading
import time

import pytest
import torch

BF16, I32 = torch.bfloat16, torch.int32


class OnGpu:
    """What the checks look at of a contiguous tensor on device 0."""

    def __init__(self, *shape, dtype=BF16, address=1 << 20):
        self.shape, self.dtype, self.address, self.requires_grad, self.device = shape, dtype, address, False, None

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self.address

    def numel(self):
        n = 1
        for s in self.shape:
            n *= s
        return n

    def dim(self):
        return len(self.shape)


class Library:
    """Counts the calls, and those of one workspace that were in it together."""

    def __init__(self, wait=0.0):
        self.wait, self.calls, self.together, self.inside, self.lock = wait, 0, 0, [], threading.Lock()

    def qb_op_scratch_bytes(self):
        return 64

    def qb_paged_zero_bytes(self):
        return 8192

    def qb_paged_workspace_bytes(self, max_queries, hq, hkv, prefix_tokens, out):
        out._obj.value = 8192 + 256 * max_queries
        return 0

    def _call(self, workspace):
        with self.lock:
            self.calls += 1
            self.together += workspace in self.inside
            self.inside.append(workspace)
        time.sleep(self.wait)  # as a call's launches, without the interpreter's lock
        with self.lock:
            self.inside.remove(workspace)
        return 0

    def qb_paged_attention(self, *a):
        return self._call(a[17])

    def qb_shared_prefix_attention(self, *a):
        return self._call(a[18])

    def qb_rope_paged_append(self, *a):
        return self._call(None)

    def qb_sample_token(self, *a):
        return self._call(None)


@pytest.fixture
def lib(monkeypatch):
    from hackthenorth_b200 import _lib, ops

    lib = Library()
    empty = torch.empty
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(ops, "_workspaces", {})
    monkeypatch.setattr(ops, "_workspace_bytes", {})
    monkeypatch.setattr(ops, "_capturing", lambda: False)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 7)
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    monkeypatch.setattr(ops, "_status", lambda index: 1 << 20)
    monkeypatch.setattr(ops.torch, "empty", lambda *s, dtype=None, device=None: empty(*s, dtype=dtype))
    return lib


def _batch(seqs=2, tokens=40, width=4, pages=9, page=16, hkv=2):
    pool = OnGpu(pages, hkv, page, 128)
    return dict(k_pages=pool, v_pages=pool, page_table=OnGpu(seqs, width, dtype=I32), q_start=OnGpu(seqs + 1, dtype=I32),
                kv_lens=OnGpu(seqs, dtype=I32)), OnGpu(tokens, 4, 128)


def _attend(tokens=40, max_queries=None, **kw):
    from hackthenorth_b200 import ops

    batch, q = _batch(tokens=tokens, **kw)
    return ops.paged_attention(q, **batch, max_queries=max_queries, out=q)


def _attend_prefix(tokens=40, table=5, length=70, **kw):
    from hackthenorth_b200 import ops

    batch, q = _batch(tokens=tokens, **kw)
    return ops.shared_prefix_attention(q, prefix_table=OnGpu(table, dtype=I32), prefix_len=length, **batch, out=q)


def test_threads_on_one_stream_take_turns(lib):
    """A call is several launches with its pieces in the workspace between them:
    another thread's call may not come in between, whichever kernel it takes."""
    lib.wait = 0.002
    calls = [lambda: _attend(40), lambda: _attend(500), lambda: _attend(2, max_queries=1), lambda: _attend_prefix(3),
             lambda: _attend_prefix(300)]
    threads = [threading.Thread(target=lambda c=c: [c() for _ in range(10)]) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert lib.calls == 50 and lib.together == 0


def _calls(make, plain):
    """Every operator with one differentiable argument after the other from ``make``, the others plain."""
    from hackthenorth_b200 import ops

    append = ["qkv", "q_norm", "k_norm", "cos", "sin", "k_pages", "v_pages", "out"]
    attend = ["q", "k_pages", "v_pages", "out"]
    tables = dict(page_table=plain, q_start=plain, kv_lens=plain)
    for op, names, rest in ((ops.rope_paged_append, append, tables), (ops.paged_attention, attend, tables),
                            (ops.shared_prefix_attention, attend, dict(tables, prefix_table=plain, prefix_len=0)),
                            (ops.sample_token, ["logits"], dict(uniforms=plain))):
        for name in names:
            yield op, {**{n: plain for n in names}, **rest, name: make}


def test_arguments_that_require_a_gradient_are_refused():
    plain = torch.zeros(2, 3)
    for op, kw in _calls(torch.zeros(2, 3, requires_grad=True), plain):
        with pytest.raises(ValueError, match="backward"):
            op(**kw)
        with torch.no_grad(), pytest.raises(ValueError, match="expected"):  # on to the next check
            op(**kw)


def test_dual_tensors_are_refused():
    import torch.autograd.forward_ad as fwd

    plain = torch.zeros(2, 3)
    with fwd.dual_level():
        for op, kw in _calls(fwd.make_dual(torch.zeros(2, 3), torch.ones(2, 3)), plain):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="forward-mode"):
                    op(**kw)
        with pytest.raises(ValueError, match="expected"):
            next(_calls(plain, plain))[0](**next(_calls(plain, plain))[1])


@pytest.mark.parametrize("kw", [dict(seqs=(1 << 32) + 2), dict(width=(1 << 32) + 4), dict(seqs=1 << 31)])
def test_batches_beyond_32_bits_are_refused(lib, kw):
    """Numbers whose low 32 bits would be a call of another size."""
    with pytest.raises(ValueError):
        _attend(**kw)
    with pytest.raises(ValueError):
        _attend_prefix(**kw)
    assert lib.calls == 0


@pytest.mark.parametrize("kw", [dict(table=1 << 29, length=(1 << 32) + 5), dict(table=1 << 29, length=1 << 32),
                                dict(table=(1 << 32) + 5), dict(length=81), dict(length=-1)])
def test_prefixes_beyond_their_table_or_32_bits_are_refused(lib, kw):
    with pytest.raises(ValueError):
        _attend_prefix(**kw)
    assert lib.calls == 0
    _attend_prefix(length=80)
    assert lib.calls == 1


@pytest.mark.parametrize("shape", [(1, (1 << 32) + 5), ((1 << 32) + 5,), ((1 << 32) + 1, 1), ((1 << 24) + 1, 8), (2, 262145)])
def test_logits_beyond_the_limits_are_refused(lib, shape):
    from hackthenorth_b200 import ops

    rows = shape[0] if len(shape) == 2 else 1
    with pytest.raises(ValueError):
        ops.sample_token(OnGpu(*shape), OnGpu(rows, dtype=torch.float32), out=OnGpu(rows, dtype=torch.int64))
    assert lib.calls == 0
    ops.sample_token(OnGpu(2, 262144), OnGpu(2, dtype=torch.float32), out=OnGpu(2, dtype=torch.int64))
    assert lib.calls == 1


def test_a_batch_of_no_sequences_leaves_every_row(lib):
    from hackthenorth_b200 import ops

    for tokens in (0, 3):
        batch, q = _batch(seqs=0, tokens=tokens)
        assert ops.paged_attention(q, **batch, out=q) is q
        assert ops.shared_prefix_attention(q, prefix_table=OnGpu(5, dtype=I32), prefix_len=70, **batch, out=q) is q
        cos = OnGpu(64, 128)
        assert ops.rope_paged_append(OnGpu(tokens, 8 * 128), None, None, cos, cos, **batch, out=q) is q
    assert lib.calls == 0
