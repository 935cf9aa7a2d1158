"""The Python layer of the microscaled operators, with the library's calls replaced: what lives while a kernel may
read it.  Runs without a GPU."""
import ctypes as C

import pytest
import torch
from torch.multiprocessing.reductions import StorageWeakRef
from torch.utils.checkpoint import checkpoint

from turboloader_b200 import mx


class _Library:
    """Takes the entry points' calls; ``on_grad(a, b, grad_a, grad_b)`` sees the operands of a gradient."""

    def __init__(self):
        self.on_grad = self.on_write = lambda *a: None

    def tlb_mx_write(self, cache, *a):
        self.on_write(cache)
        return 0

    def tlb_mx_quantize(self, *a):
        return 0

    def tlb_mx_read_codes(self, *a):
        return 0

    def tlb_mx_read(self, *a):
        return 0

    def tlb_mx_matmul(self, *a):
        return 0

    def tlb_mx_linear(self, *a):
        return 0

    def tlb_mx_matmul_workspace(self, *a):
        return 0

    def tlb_mx_grad_workspace(self, *a):
        return 1 << 16

    def tlb_mx_grad(self, g, g_dtype, m, n, a, b, grad_a, a_dtype, grad_b, b_dtype, *rest):
        self.on_grad(a, b, grad_a, grad_b)
        return 0


@pytest.fixture
def library(monkeypatch):
    lib = _Library()
    monkeypatch.setattr(mx._capi, "load", lambda: lib)
    monkeypatch.setattr(mx, "_cuda", lambda t, what: t)
    monkeypatch.setattr(mx, "_away", lambda device, stream: False)
    monkeypatch.setattr(mx, "_raw_stream", lambda index: None)
    return lib


class _Watched:
    """A context whose saved tensors are watched, not kept."""

    def __init__(self, ctx, watched):
        self._ctx, self._watched = ctx, watched

    def __getattr__(self, name):
        return getattr(self._ctx, name)

    @property
    def saved_tensors(self):
        saved = self._ctx.saved_tensors
        self._watched += [(StorageWeakRef(t.untyped_storage()), t.data_ptr(), t.data_ptr() + t.nbytes) for t in saved]
        return saved


@pytest.mark.parametrize("how", ["plain", "hooks", "checkpoint"])
@pytest.mark.parametrize("held", [False, True])
def test_saved_rows_live_until_the_gradients_are_launched(library, monkeypatch, how, held):
    """Under hooks and checkpoints the node does not own what it unpacks: only the backward pass keeps it alive."""
    x = torch.randn(6, 64, requires_grad=True)
    w = torch.randn(5, 64, requires_grad=True)
    q = mx.MxTensor(torch.zeros(6, 64, dtype=torch.uint8), torch.zeros(6, 8, dtype=torch.uint8), (6, 64), "nvfp4") if held else x
    watched, launched = [], []
    backward = mx._MxLinear.backward
    monkeypatch.setattr(mx._MxLinear, "backward", staticmethod(lambda ctx, g: backward(_Watched(ctx, watched), g)))

    def on_grad(a, b, grad_a, grad_b):
        assert watched and not any(storage.expired() for storage, _, _ in watched)
        for rows in (a, b):
            if rows is not None:
                assert all(any(low <= at < high for _, low, high in watched) for at in (rows.codes, rows.scales))
        launched.append((a is not None, b is not None, bool(grad_a), bool(grad_b)))

    library.on_grad = on_grad
    if how == "checkpoint":
        y = checkpoint(lambda w: mx.mx_linear(q, w, "nvfp4"), w, use_reentrant=False)
    elif how == "hooks":
        with torch.autograd.graph.saved_tensors_hooks(torch.clone, torch.clone):
            y = mx.mx_linear(q, w, "nvfp4")
    else:
        y = mx.mx_linear(q, w, "nvfp4")
    y.sum().backward()
    assert launched == [(True, not held, not held, True)]


@pytest.mark.parametrize("lead", [(), (3,), (2, 3), (0,), (2, 0), (2, 1, 3)])
@pytest.mark.parametrize("n", [0, 5])
def test_gradients_of_any_leading_dimensions_and_of_no_rows(library, lead, n):
    x = torch.randn(*lead, 40, requires_grad=True)
    w = torch.randn(n, 40, requires_grad=True)
    y = mx.mx_linear(x, w, "mxfp8")
    assert y.shape == (*lead, n)
    gx, gw = torch.autograd.grad(y, [x, w], torch.ones(*lead, n))
    assert gx.shape == x.shape and gw.shape == w.shape


def test_the_claims_of_a_write_belong_to_its_stream(library, monkeypatch):
    """No write sees words that one on another stream may be claiming or has yet to fill, and a captured one fills its own."""
    cache = mx.MxCache(torch.zeros(700, 1, 64, dtype=torch.uint8), torch.zeros(700, 1, 8, dtype=torch.uint8), 40, "nvfp4")
    stream, capturing, seen = [0], [False], []
    monkeypatch.setattr(mx, "_raw_stream", lambda index: stream[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])

    def write(n, on, captured=False):
        stream[0], capturing[0] = on, captured
        cache.write(torch.arange(n), torch.zeros(n, 1, 40))
        return seen[-1]

    def on_write(c):
        words = (C.c_int32 * 700).from_address(c.owner) if c.owner else None
        seen.append((c.owner, words and list(words)))
        if words:
            words[:] = [stream[0]] * 700

    library.on_write = on_write
    unused = [-1] * 700
    assert write(256, 1) == (None, None)
    at, words = write(257, 1)
    assert words == unused
    assert write(600, 2, captured=True)[1] == unused      # before the stream's first eager one
    other, words = write(600, 2)
    assert words == unused and other != at
    assert write(300, 1) == (at, [1] * 700)               # the stream's own, in its order
    captured, words = write(300, 1, captured=True)
    assert words == unused and captured not in (at, other)


def _value(address):
    return C.c_float.from_address(address).value


def test_scales_on_the_device_are_those_of_the_forward_pass(library):
    """A caller may change its tensor before the gradients: the rows were made with the old value."""
    x, w = torch.randn(6, 64, requires_grad=True), torch.randn(5, 64, requires_grad=True)
    sx, sw = torch.tensor([0.5]), torch.tensor(0.25)
    y = mx.mx_linear(x, w, "nvfp4", scale=sx, weight_scale=sw)
    sx.fill_(7), sw.fill_(9)
    seen = []
    library.on_grad = lambda a, b, *rest: seen.append((_value(a.scale_dev), _value(b.scale_dev)))
    y.sum().backward()
    assert seen == [(0.5, 0.25)]


def test_a_held_scale_that_changed_before_the_gradients_is_refused(library):
    scale = torch.tensor([0.5])
    held = mx.MxTensor(torch.zeros(6, 64, dtype=torch.uint8), torch.zeros(6, 8, dtype=torch.uint8), (6, 64), "nvfp4", scale=scale)
    w = torch.randn(5, 64, requires_grad=True)
    seen = []
    library.on_grad = lambda a, *rest: seen.append(_value(a.scale_dev))
    mx.mx_linear(held, w, "nvfp4").sum().backward()
    assert seen == [0.5]
    y = mx.mx_linear(held, w, "nvfp4")
    scale.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    assert seen == [0.5]


def test_rows_made_with_a_scale_on_the_device_keep_its_value(library):
    scale = torch.tensor([0.5])
    q = mx.mx_quantize(torch.randn(6, 64), scale=scale)
    cache = mx.MxCache(torch.zeros(3, 1, 64, dtype=torch.uint8), torch.zeros(3, 1, 8, dtype=torch.uint8), 64, "nvfp4", scale=scale)
    batch = cache.read_mx(torch.arange(2))
    scale.fill_(3)
    assert float(q.scale) == float(batch.scale) == 0.5 and float(cache.scale) == 3


def test_forward_mode_is_refused_not_dropped(library):
    x, w = torch.randn(6, 64), torch.randn(5, 64)
    with torch.autograd.forward_ad.dual_level():
        assert mx.mx_linear(x, w).shape == (6, 5)      # no tangent: an ordinary call
        for a, b in ((torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), w), (x, torch.autograd.forward_ad.make_dual(w, torch.ones_like(w)))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    mx.mx_linear(a, b)


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_tracing_is_refused():
    def call(x):
        mx._away(torch.device("cuda", 0), None)        # what every entry point asks before it allocates
        return x

    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, torch.ones(1))


@pytest.mark.parametrize("x_held,w_held,x_grad,w_grad", [(False, False, True, True), (False, False, True, False), (False, False, False, True),
                                                         (True, False, False, True), (False, True, True, False)])
def test_only_rows_that_the_gradients_read_are_saved(library, x_held, w_held, x_grad, w_grad):
    """The input's gradient reads the weight's rows and the weight's gradient the input's."""
    def operand(rows, held, grad):
        if held:
            return mx.MxTensor(torch.zeros(rows, 512, dtype=torch.uint8), torch.zeros(rows, 64, dtype=torch.uint8), (rows, 1024), "nvfp4")
        return torch.randn(rows, 1024, requires_grad=grad)

    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t.nbytes) or t, lambda t: t):
        mx.mx_linear(operand(2, x_held, x_grad), operand(3, w_held, w_grad), "nvfp4")
    size = {2: 1024 + 256, 3: 1536 + 256} if not (x_held or w_held) else {2: 2 * 576, 3: 3 * 576}  # parts of a buffer start at multiples of 256
    assert sum(saved) == (size[2] if w_grad else 0) + (size[3] if x_grad else 0)


def _rows(*lead, cols=64):
    return mx.MxTensor(torch.zeros(*lead, 64, dtype=torch.uint8), torch.zeros(*lead, 8, dtype=torch.uint8), (*lead, cols), "nvfp4")


@pytest.mark.parametrize("call", [lambda out: mx.mx_dequantize(_rows(4), out=out), lambda out: mx.mx_matmul(_rows(4), _rows(64), torch.float32, out=out),
                                  lambda out: mx.MxCache(_rows(4, 1).codes, _rows(4, 1).scales, 64, "nvfp4").read(None, torch.float32, out=out.view(4, 1, 64))])
def test_writes_into_a_tensor_that_a_graph_saved_are_seen(library, call):
    out = torch.zeros(4, 64)
    w = torch.ones(64, requires_grad=True)
    call(out)
    (out * w).sum().backward()
    y = (out * w).sum()
    call(out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    out.requires_grad_(True)
    with pytest.raises(ValueError, match="gradients"):
        call(out)
    with torch.no_grad():
        call(out)


def test_a_cache_written_before_the_gradients_of_its_rows_is_seen(library):
    codes, scales = torch.zeros(4, 1, 64, dtype=torch.uint8), torch.zeros(4, 1, 8, dtype=torch.uint8)
    cache = mx.MxCache(codes, scales, 64, "nvfp4")
    w = torch.randn(5, 64, requires_grad=True)
    y = mx.mx_linear(mx.MxTensor(codes, scales, (4, 1, 64), "nvfp4"), w, "nvfp4")
    cache.write(torch.arange(2), torch.zeros(2, 1, 64))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---- the loader --------------------------------------------------------------------------------------------------

class _Images:
    """What a feature loader sees of an image loader."""

    def __init__(self, n, batch_size, items, **kw):
        self._n, self.batch_size, self._items = n, batch_size, items
        self.__dict__.update(kw)

    def __iter__(self):
        return iter(self._items)


def _feature_loader(monkeypatch):
    from turboloader_b200 import CudaFeatureLoader

    loader = CudaFeatureLoader.__new__(CudaFeatureLoader)
    loader._torch, loader._device, loader._n = torch, torch.device("cpu"), 100
    written = []
    monkeypatch.setattr(loader, "write", lambda indices, features, lengths=None: written.append((list(indices), features, lengths)), raising=False)
    return loader, written


def test_fill_refuses_loaders_that_leave_samples_out(monkeypatch):
    loader, written = _feature_loader(monkeypatch)
    batch = (torch.zeros(4, 3), [0, 1, 2, 3])
    with pytest.raises(ValueError, match="last 2 of its 10"):
        loader.fill(_Images(10, 4, [batch, batch], drop_last=True, return_indices=True), lambda x: x)
    with pytest.raises(ValueError, match="return_indices"):   # images and labels
        loader.fill(_Images(8, 4, [batch, batch], drop_last=True, return_indices=False), lambda x: x)
    assert not written
    for images in (_Images(10, 4, [batch, batch], drop_last=False, return_indices=True), _Images(8, 4, [batch, batch], drop_last=True, return_indices=True),
                   [batch, batch]):
        assert loader.fill(images, lambda x: x) == 8
    assert len(written) == 6


@pytest.mark.parametrize("a,b", [(1e30, 1e30), (1e-30, 1e-30), (2.0 ** -100, 2.0 ** -27), (2.0 ** 127, 2.0)])
def test_tensor_scales_whose_product_leaves_the_range_are_refused(a, b):
    """They would turn sums of zero into NaN, or everything into zero."""
    from turboloader_b200 import _capi

    lib = _capi.load()
    rows = [_capi.MxRows(0x1000, 0x2000, 8, 64, 0, s, None) for s in (a, b)]
    ready = (0x9000, 1 << 20, None)
    assert lib.tlb_mx_matmul(*rows, 0x8000, 0, *ready) == 1 and b"scales" in lib.tlb_last_error()
    assert lib.tlb_mx_linear(rows[0], 0x5000, 0, 64, rows[1], 0x6000, 0, 64, 0x8000, 0, *ready) == 1
    assert lib.tlb_mx_matmul_workspace(*rows, 0) == -1
    rows[1].scale = 1.0
    assert lib.tlb_mx_matmul_workspace(*rows, 0) > 0
