"""Arguments of plan_rotation, and the C entry points' refusals, without a GPU."""

import ctypes

import numpy as np
import pytest
import torch

from nexusquant_amd import _lib, rotary


def test_frequencies_belong_to_their_axes():
    f = rotary.frequency_axes
    assert f(64, None, False).tolist() == [0] * 32
    assert f(64, [8, 12, 12], False).tolist() == [0] * 8 + [1] * 12 + [2] * 12
    got = f(128, [24, 20, 20], True)
    assert got[:60].tolist() == [0, 1, 2] * 20 and got[60:].tolist() == [0] * 4
    assert f(64, [16, 16], True).tolist() == [0, 1] * 16
    assert f(64, [32, 0], True).tolist() == [0] * 32
    for sections, interleaved in (([8, 8], False), ([40, -8], False), ([], False), ([8, 24], True), ([8, 12, 12], True)):
        with pytest.raises(ValueError):
            f(64, sections, interleaved)


def test_arguments_are_checked_before_any_device():
    with pytest.raises(ValueError, match="head_dim"):
        rotary.plan_rotation([1, 2], 96)
    with pytest.raises(TypeError):
        rotary.plan_rotation([1.5], 64)
    with pytest.raises(TypeError):
        rotary.plan_rotation([True], 64)
    with pytest.raises(_lib.NexusQuantError):
        rotary.plan_rotation([1], 64, device="cpu")


def test_which_outputs_are_apart():
    x = torch.empty(6, 8, 16)
    apart = rotary.same_or_apart
    assert apart(x, x) and apart(x[:, :4], x[:, 4:]) and apart(x[:3], x[3:])
    assert not apart(x[:, :4], x[:, 3:]) and not apart(x[:, :5], x[:, 2:3]) and not apart(x, x[1:])
    assert apart(x, torch.empty(6, 8, 16)) and apart(x[:0], x)
    assert not apart(x, x.transpose(0, 1))
    own = rotary.vectors_apart
    assert own(x) and own(x.transpose(0, 1)) and own(x[:, ::2]) and own(x[:1].expand(1, 8, 16))
    assert not own(x[:, :1].expand(6, 8, 16)) and not own(x[:1].expand(6, 8, 16))
    assert not own(torch.empty(6 * 8 * 16).as_strided((6, 8, 16), (16, 16, 1)))


def test_entry_points_refuse_bad_arguments():
    lib = _lib.load()
    freq, axis = np.ones(64, np.float32), np.zeros(64, np.uint8)
    dummy = ctypes.c_void_p(4096)

    def rotation(axes=1, rows=4, half=64, positions=dummy, out=dummy, axis=axis):
        return lib.nq_rotation(positions, 0, axes, rows, rows, half, freq.ctypes.data, axis.ctypes.data, out, None)

    assert rotation(axes=0) == rotation(axes=256) == rotation(rows=-1) == rotation(half=0) == rotation(half=129) == -1
    assert rotation(rows=1 << 27) == rotation(positions=None) == rotation(out=None) == rotation(axis=axis + 1) == -1
    assert rotation(rows=0) == 0

    def desc(rows=4, hq=2, hk=1, d=64, dtype=0, q=4096, k=4096, qo=8192, ko=8192, angles=4096, strides=(128, 64) * 4):
        return rotary._PACK.pack(rows, hq, hk, d, dtype, 0, q, k, qo, ko, angles, *strides)

    assert lib.nq_rotate(None, None) == -1
    for kw in (dict(rows=-1), dict(hq=-1), dict(hk=-2), dict(d=96), dict(dtype=3), dict(q=0), dict(ko=0), dict(angles=0),
               dict(q=4098), dict(angles=4100), dict(strides=(128, 60) + (128, 64) * 3), dict(strides=(128, 64) * 3 + (1, 64)),
               dict(rows=(1 << 31) - 1, hq=1 << 20)):
        assert lib.nq_rotate(desc(**kw), None) == -1, kw
    assert lib.nq_rotate(desc(rows=0), None) == lib.nq_rotate(desc(hq=0, hk=0), None) == 0


def test_frequencies_live_until_the_call_has_read_them(monkeypatch):
    """Another thread may empty the tables while a call is on its way to the device."""
    import contextlib
    import gc
    import weakref

    class OnDevice(torch.Tensor):  # a tensor of the host that says it is on a device
        is_cuda = True

    held, read = [], []
    table = rotary._table

    def watched(*args):
        got = table(*args)
        held.extend(weakref.ref(a) for a in got[1:3])
        return got

    class Lib:
        @staticmethod
        def nq_rotation(positions, wide, axes, stride, rows, half, freq, axis_of, out, stream):
            rotary._tables.clear()
            gc.collect()
            assert all(a() is not None for a in held)
            read.append(np.ctypeslib.as_array(ctypes.cast(freq, ctypes.POINTER(ctypes.c_float)), (half,)).copy())
            read.append(np.ctypeslib.as_array(ctypes.cast(axis_of, ctypes.POINTER(ctypes.c_uint8)), (half,)).copy())
            return 0

    monkeypatch.setattr(rotary, "_table", watched)
    monkeypatch.setattr(rotary._lib, "load", Lib)
    monkeypatch.setattr(rotary._lib, "current_stream_handle", lambda dev: None)
    monkeypatch.setattr(rotary, "on_device", lambda dev: contextlib.nullcontext())
    positions = torch.zeros(2, 3, dtype=torch.int64).as_subclass(OnDevice)
    rotary.plan_rotation(positions, 64, base=12345.0, sections=[20, 12])
    assert len(held) == 2
    assert np.array_equal(read[0], rotary.inv_freq(64, 12345.0).numpy())
    assert np.array_equal(read[1], rotary.frequency_axes(64, [20, 12], False))


def turned(x, angles, inverse):
    c, s = angles[:, None, 0], angles[:, None, 1] * (-1.0 if inverse else 1.0)
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def host_rotation(monkeypatch, rows=5, d=64):
    """A rotation of the host, and what is launched: pairs (query or not, key or not), computed in torch's operations."""
    launched = []

    def launch(query, key, angles, inverse, q_out, k_out):
        launched.append((query is not None, key is not None))
        for x, y in ((query, q_out), (key, k_out)):
            if x is not None:  # (by memory alone, as a kernel)
                y.detach().numpy()[:] = turned(torch.from_numpy(x.detach().numpy()), angles, inverse).numpy()

    monkeypatch.setattr(rotary, "_launch", launch)
    angle = torch.rand(rows, d // 2, generator=torch.Generator().manual_seed(1)) * 6
    return rotary.Rotation(angles=torch.stack([angle.cos(), angle.sin()], dim=1), rows=rows, head_dim=d), launched


def check_gradients_of_those_that_need_one(r, launched):
    """The query alone, the key alone: the other's output needs no gradient, and none is computed.  Both, of which one is used."""
    dev, (rows, d) = r.device, (r.rows, r.head_dim)
    g = torch.Generator().manual_seed(2)
    for of_query, of_key in ((True, False), (False, True)):
        q, k = (torch.randn(rows, h, d, generator=g).to(dev).requires_grad_(need) for h, need in ((4, of_query), (2, of_key)))
        w = [torch.randn(x.shape, generator=g).to(dev) for x in (q, k)]
        y = rotary.rotate(q, k, r)
        assert (y[0].requires_grad, y[1].requires_grad) == (of_query, of_key)
        before = len(launched)
        got, = torch.autograd.grad((y[0] * w[0]).sum() + (y[1] * w[1]).sum(), (q if of_query else k,))
        assert launched[before:] in ([(of_query, of_key)], [])  # (empty: the kernel itself ran)
        assert (got - turned(w[0 if of_query else 1], r.angles, True)).abs().max() <= 1e-5
    q, k = (torch.randn(rows, h, d, generator=g).to(dev).requires_grad_() for h in (4, 2))
    y = rotary.rotate(q, k, r)
    assert y[0].requires_grad and y[1].requires_grad
    w = torch.randn(k.shape, generator=g).to(dev)
    got = torch.autograd.grad((y[1] * w).sum(), (q, k), allow_unused=True)
    assert got[0] is None and (got[1] - turned(w, r.angles, True)).abs().max() <= 1e-5


def test_gradients_of_those_that_need_one(monkeypatch):
    check_gradients_of_those_that_need_one(*host_rotation(monkeypatch))


def check_forward_mode(r):
    """Tangents turn as their tensors do; with them gradients, tangents of gradients and gradients of tangents."""
    from torch.autograd import forward_ad
    dev, (rows, d) = r.device, (r.rows, r.head_dim)
    g = torch.Generator().manual_seed(3)
    q, k, tq, tk, w = (torch.randn(rows, h, d, generator=g).to(dev) for h in (4, 2, 4, 2, 4))

    def close(x, want):
        assert (x - want).abs().max() <= 1e-5

    for inverse in (False, True):
        for grads in (False, True):
            with torch.set_grad_enabled(grads), forward_ad.dual_level():
                y = rotary.rotate(forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk), r, inverse=inverse)
                for out, x, t in ((y[0], q, tq), (y[1], k, tk)):
                    got = forward_ad.unpack_dual(out)
                    close(got.primal, turned(x, r.angles, inverse))
                    close(got.tangent, turned(t, r.angles, inverse))
                # of one of the two, and of a query alone
                y = rotary.rotate(q, forward_ad.make_dual(k, tk), r, inverse=inverse)
                assert forward_ad.unpack_dual(y[0]).tangent is None
                close(forward_ad.unpack_dual(y[1]).tangent, turned(tk, r.angles, inverse))
                y = rotary.rotate(forward_ad.make_dual(q, tq), None, r, inverse=inverse)
                assert y[1] is None
                close(forward_ad.unpack_dual(y[0]).tangent, turned(tq, r.angles, inverse))
    with forward_ad.dual_level():
        # a gradient with respect to the query beside a tangent of the key
        leaf = q.clone().requires_grad_()
        y = rotary.rotate(leaf, forward_ad.make_dual(k, tk), r)
        t = forward_ad.unpack_dual(y[0]).tangent
        assert t is None or not t.any()
        close(forward_ad.unpack_dual(y[1]).tangent, turned(tk, r.angles, False))
        got, = torch.autograd.grad(y[0], leaf, forward_ad.make_dual(w, tq))  # a gradient's tangent
        close(got, turned(w, r.angles, True))
        close(forward_ad.unpack_dual(got).tangent, turned(tq, r.angles, True))
        leaf = tq.clone().requires_grad_()  # a tangent's gradient
        y = rotary.rotate(forward_ad.make_dual(q, leaf), None, r)[0]
        got, = torch.autograd.grad(forward_ad.unpack_dual(y).tangent, leaf, w)
        close(got, turned(w, r.angles, True))
        for args in ((forward_ad.make_dual(q, tq), None), (q, forward_ad.make_dual(k, tk))):
            with torch.no_grad(), pytest.raises(NotImplementedError):
                rotary.rotate(*args, r, out=(torch.empty_like(q), None if args[1] is None else torch.empty_like(k)))


def test_forward_mode(monkeypatch):
    check_forward_mode(host_rotation(monkeypatch)[0])


def saved_by_a_graph(x):
    """The output of a graph that has saved x."""
    return (torch.ones_like(x, requires_grad=True) * x).sum()


def check_written_tensors_are_seen(write, *outs):
    """A graph that has saved what `write` writes into raises in its backward pass."""
    graphs, before = [saved_by_a_graph(x) for x in outs], [x._version for x in outs]
    write()
    for y, x, version in zip(graphs, outs, before):
        assert x._version > version
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_writes_in_place_are_seen_by_autograd(monkeypatch):
    r, _ = host_rotation(monkeypatch)
    qkv = torch.randn(5, 8, 64)
    q, k = qkv[:, :4], qkv[:, 4:6]
    into = torch.empty(5, 4, 64), torch.empty(5, 2, 64)
    check_written_tensors_are_seen(lambda: rotary.rotate(q, k, r, out=(q, k)), q, k, qkv)
    check_written_tensors_are_seen(lambda: rotary.rotate(q, k, r, out=into), *into)
    check_written_tensors_are_seen(lambda: rotary.rotate(q, None, r, out=(q, None)), q)
    version = qkv._version
    rotary.rotate(q, k, r)
    assert qkv._version == version
    with torch.inference_mode():  # such tensors have no versions
        q, k = torch.randn(5, 4, 64), torch.randn(5, 2, 64)
        rotary.rotate(q, k, r, out=(q, k))
    rotary.rotate(q, k, r, out=(q, k))


def test_a_capture_is_looked_for_on_the_rotation_s_device(monkeypatch):
    """Which need not be the current one."""
    import contextlib
    current = [torch.device("cuda", 0)]

    @contextlib.contextmanager
    def on_device(dev):
        current.append(dev)
        yield
        current.pop()

    monkeypatch.setattr(rotary, "on_device", on_device)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[-1].index == 1)
    with pytest.raises(RuntimeError, match="before capturing"):
        rotary.plan_rotation([1, 2], 64, device="cuda:1")


def test_function_transforms_are_refused(monkeypatch):
    """Not passed by: their tensors have no memory that a kernel could read."""
    r, _ = host_rotation(monkeypatch)
    q = torch.randn(5, 4, 64)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: rotary.rotate(x, None, r)[0], (q,), (q,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: rotary.rotate(x, None, r)[0].sum())(q)
    with pytest.raises((RuntimeError, ValueError)):
        torch.func.vmap(lambda x: rotary.rotate(x, None, r)[0])(q[None])
