"""The wrapper around the q4_0 cache's calls without a GPU: where workspaces come from, which tensors are refused."""
import contextlib
from types import SimpleNamespace

import pytest

import tsrc


class _FakeTorch:
    """As much of torch as a workspace takes, noting the stream that is current at an allocation."""
    uint8 = "uint8"

    def __init__(self):
        self.now, self.made = "current", []
        self.cuda = SimpleNamespace(stream=self._stream, ExternalStream=lambda handle, device=None: ("external", handle, device))

    @contextlib.contextmanager
    def _stream(self, s):
        was, self.now = self.now, s
        yield
        self.now = was

    def empty(self, n, dtype, device):
        self.made.append((n, device, self.now))
        return SimpleNamespace(data_ptr=lambda: 4096, numel=lambda: n, element_size=lambda: 1, record_stream=lambda s: None)


@pytest.mark.parametrize("stream,want", [(None, "current"), ("side", "side"), (77, ("external", 77, "cuda:0")), (0, ("external", 0, "cuda:0"))])
def test_workspace_comes_from_the_calls_own_stream(monkeypatch, stream, want):
    """A block that the current stream still works on may be handed out again to that stream alone."""
    fake = _FakeTorch()
    monkeypatch.setattr(tsrc, "_torch", fake)
    tsrc._workspace(SimpleNamespace(device="cuda:0"), 512, None, stream)
    assert fake.made == [(512, "cuda:0", want)] and fake.now == "current"


class _OnDevice:
    """A CPU tensor that says it lies on a GPU; no call with one gets past the checks and the library's own refusal."""

    def __init__(self, t, index=0):
        self._t, self.is_cuda, self.device = t, True, SimpleNamespace(index=index)
        self.get_device = lambda: index

    def __getattr__(self, name):
        return getattr(self._t, name)


def _on(t, index=0):
    return _OnDevice(t, index)


@pytest.fixture
def stub(monkeypatch):
    """A device handle without a device: a call that passes the wrapper's checks is refused by the library as NULL."""
    pytest.importorskip("torch")
    dev = tsrc.Device.__new__(tsrc.Device)
    dev.handle, dev.index = None, 0
    monkeypatch.setattr(tsrc, "_stream_on", lambda index, stream: None)
    yield dev, tsrc.Kv4Cache(dev, None, 2, 64, 100)
    dev.handle = None


def _refused(call, what):
    with pytest.raises(tsrc.TsrcError) as e:
        call()
    assert e.value.code == tsrc.E_ARG and what in str(e.value), str(e.value)


def test_attention_refuses_tensors_that_do_not_hold_the_call(stub):
    import torch
    dev, kv = stub
    q, out = torch.zeros(6, 4, 64), torch.zeros(6, 4, 64)

    def call(**kw):
        a = dict(q=_on(q), out=_on(out), T=6, n_head=4, n_kv=100, scale=0.1, ranges=None, mask=None) | kw
        dev.flash_attn_q4(kv, a.pop("q"), a.pop("out"), **a)

    wide = torch.zeros(6, 3, 4, 64)
    i32, f16 = torch.int32, torch.float16
    passes = [dict(), dict(q=_on(wide[:, 1])), dict(q=_on(wide.view(6, -1)[:, 256:512])), dict(q=_on(wide.flatten()[7:]), q_stride=768),
              dict(out=_on(wide[:, 2]), out_stride=768), dict(ranges=_on(torch.zeros(6, 2, dtype=i32))), dict(T=0),
              dict(mask=_on(torch.zeros(6, 100, dtype=f16))), dict(mask=_on(torch.zeros(5 * 104 + 100, dtype=f16)), mask_stride=104),
              dict(workspace=_on(torch.zeros(64, dtype=torch.uint8)))]
    for kw in passes:
        _refused(lambda: call(**kw), "NULL")
    bad = [(dict(q=q), "q "), (dict(out=out), "out "), (dict(q=_on(q, 1)), "q "), (dict(out=_on(out, 1)), "out "),
           (dict(q=_on(q[:5])), "q "), (dict(out=_on(out[:5])), "out "), (dict(q=_on(q.transpose(0, 1))), "q "),
           (dict(q=_on(torch.zeros(6, 64, 4).transpose(1, 2))), "q "), (dict(q=_on(wide[:, 1]), q_stride=256), "q "),
           (dict(out=_on(out[:1].expand(6, 4, 64))), "out "), (dict(q=_on(wide[:, :2])), "q "), (dict(q=_on(q), q_stride=300), "q "),
           (dict(ranges=_on(torch.zeros(5, 2, dtype=i32))), "ranges"), (dict(ranges=torch.zeros(6, 2, dtype=i32)), "ranges"),
           (dict(mask=_on(torch.zeros(5, 100, dtype=f16))), "mask"), (dict(mask=_on(torch.zeros(6, 200, dtype=f16)[:, :100])), "mask"),
           (dict(mask=_on(torch.zeros(6, 100, dtype=f16), 1)), "mask"), (dict(workspace=torch.zeros(64, dtype=torch.uint8)), "workspace"),
           (dict(q=4096), "type"), (dict(q_stride=-256), "q"), (dict(out_stride=-1), "out"), (dict(T=-1), "q"),
           (dict(mask=_on(torch.zeros(6, 100, dtype=f16)), mask_stride=-100), "mask_stride")]
    for kw, what in bad:
        _refused(lambda: call(**kw), what)


def test_beam_select_refuses_tensors_that_do_not_hold_the_call(stub):
    import torch
    dev, _ = stub
    x, s = torch.zeros(2, 4, 100), torch.zeros(2, 6)
    i = torch.zeros(2, 6, dtype=torch.int32)

    def call(**kw):
        a = dict(x=_on(x), scores=_on(torch.zeros(2, 4)), s=_on(s), b=_on(i), t=_on(i), n_group=2, n_beam=4, n_vocab=100, n_out=6,
                 workspace=_on(torch.zeros(1 << 16, dtype=torch.uint8))) | kw
        dev.beam_select(a.pop("x"), a.pop("scores"), a.pop("s"), a.pop("b"), a.pop("t"), **a)

    padded = torch.zeros(2, 4, 128)
    for kw in (dict(), dict(scores=None), dict(x=_on(padded[..., :100])), dict(x=_on(padded), stride=128), dict(n_group=0)):
        _refused(lambda: call(**kw), "NULL")
    for kw, what in ((dict(x=x), "logits"), (dict(x=_on(x, 1)), "logits"), (dict(x=_on(x[:, :3])), "logits"), (dict(x=_on(x[:1])), "logits"),
                     (dict(x=_on(torch.zeros(2, 100, 4).transpose(1, 2))), "logits"), (dict(x=_on(padded[..., :100]), stride=100), "logits"),
                     (dict(scores=_on(torch.zeros(2, 3))), "scores"), (dict(s=_on(s[:1])), "out_scores"), (dict(b=_on(i[:, :5])), "out_beam"),
                     (dict(t=_on(i[:1])), "out_token"), (dict(t=_on(i, 1)), "out_token"), (dict(b=i), "out_beam")):
        _refused(lambda: call(**kw), what)


@pytest.mark.parametrize("name", ["set_rows", "get_rows"])
def test_rows_refuse_tensors_that_do_not_hold_the_call(stub, name):
    import torch
    _, kv = stub
    move = getattr(kv, name)
    x = torch.zeros(5, 128)
    fused = torch.zeros(5, 3, 128)
    cells = torch.zeros(5, dtype=torch.int64)
    for k, v, kw in ((_on(x), _on(x), {}), (_on(fused[:, 1]), _on(fused[:, 2]), {}), (None, _on(fused[:, 2]), {}), (_on(x), None, dict(cells=_on(cells))),
                     (_on(fused.flatten()[128:]), _on(fused[:, 2]), dict(n=5, row_stride=384)), (_on(x), None, dict(n=0))):
        _refused(lambda: move(k, v, **kw), "NULL")
    for k, v, kw, what in ((x, None, {}, "k "), (None, x, {}, "v "), (_on(x, 1), None, {}, "k "), (_on(x), _on(x[:4]), {}, "v "),
                           (_on(x), None, dict(n=6), "k "), (_on(torch.zeros(128, 5).t()), None, {}, "k "), (_on(x), _on(fused[:, 1]), {}, "apart"),
                           (_on(fused[:, 1]), None, dict(row_stride=128), "k "), (_on(x), None, dict(cells=_on(cells[:4])), "cells"),
                           (_on(x), None, dict(cells=cells), "cells"), (_on(x[:1].expand(5, 128)), None, {}, "k "), (None, None, {}, "neither"),
                           (_on(x), None, dict(row_stride=-128), "k"), (None, _on(x), dict(n=-1, cells=_on(cells)), "-1 rows")):
        _refused(lambda: move(k, v, **kw), what)


def test_reorder_refuses_a_selection_that_was_not_gathered(stub):
    """out_beam of n_out = 2 n_beam: rows twice as long as the parents', whose entries would be read as other groups'."""
    import torch
    _, kv = stub
    wide = torch.zeros(3, 8, dtype=torch.int32)
    _refused(lambda: kv.reorder(_on(wide[:, :4].contiguous()), 3, 4, 8, 8), "NULL")
    for parent in (wide, wide.flatten(), wide[:, :4], wide[:2, :4].contiguous()):
        _refused(lambda: kv.reorder(_on(parent), 3, 4, 8, 8), "parent")
    _refused(lambda: kv.reorder(wide[:, :4].contiguous(), 3, 4, 8, 8), "parent")
