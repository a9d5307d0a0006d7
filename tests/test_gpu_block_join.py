"""The join of a block to the residual stream on the GPU, against the float64 restatement.

Tolerances: a bf16 result is its exact value rounded once (half a unit in the last place; a whole one, 2^-8, is granted)
plus f32 arithmetic on terms whose absolute sum is A: 2^-20 A (a norm's sum of cols squares is relative, its
rounding a few 2^-24).  Sums over rows: 2^-20 of the sum of absolute terms (at most 2^9 rows a line, summed in f32
in a fixed order).  f32 results: 2^-20 A."""
import numpy as np
import pytest

from jaxpp_amd import runtime as rt
from oracle import student as O
from oracle.layers import bf16_round

pytestmark = pytest.mark.gpu

SHARE, ULP = 2.0 ** -20, 2.0 ** -8
EPS = 1e-5


def _close(got, want, scale, f32, what):
    assert np.isfinite(got).all(), f"{what}: not finite"
    bound = SHARE * scale + (0 if f32 else ULP) * np.abs(want) + 1e-30
    worst = np.max(np.abs(got.astype(np.float64) - want) / bound)
    assert worst <= 1, f"{what}: {worst:.3g} x the bound"


def _up(a, f32):
    if a is None:
        return None
    return rt.DeviceBuffer.from_numpy(np.asarray(a, np.float32)) if f32 else rt.DeviceBuffer.from_f32_as_bf16(a)


def _ptr(b):
    return None if b is None else b.ptr


def _down(b, shape, f32):
    return b.download(np.float32, shape) if f32 else b.download_bf16(shape)


class Problem:
    def __init__(self, rows, cols, f32=False, post=True, gate_rows=0, pre=True, alpha=0.9, seed=0):
        rng = np.random.default_rng(seed + rows * 10000 + cols)
        rnd = (lambda a: np.asarray(a, np.float32)) if f32 else (lambda a: bf16_round(np.asarray(a, np.float32)))
        r = lambda *s, scale=1.0: rnd(scale * rng.standard_normal(s))
        self.rows, self.cols, self.f32, self.gate_rows, self.alpha = rows, cols, f32, gate_rows, alpha
        self.x, self.b = r(rows, cols), r(rows, cols, scale=2.0)
        self.gamma_post = rnd(1 + 0.2 * rng.standard_normal(cols)) if post else None
        self.gate = r(rows // gate_rows, cols) if gate_rows else None
        self.gamma_pre = rnd(1 + 0.2 * rng.standard_normal(cols)) if pre else None
        self.h, self.dh, self.dy = r(rows, cols), r(rows, cols), r(rows, cols)
        # sums that are there before, as large as a row's contribution
        self.before = {n: rng.standard_normal(cols if n != "dgate" else (rows // gate_rows, cols)).astype(np.float32)
                       for n in ("dgamma_post", "dgate", "dgamma_pre")
                       if (n != "dgate" or gate_rows) and (n != "dgamma_post" or post) and (n != "dgamma_pre" or pre)}

    def _weights(self):
        return {n: _up(getattr(self, n), self.f32) for n in ("gamma_post", "gate", "gamma_pre")}

    def check_forward(self, over=None):
        """`over`: the operand whose place the new residual stream takes."""
        w, shape = self._weights(), (self.rows, self.cols)
        dev = {"x": _up(self.x, self.f32), "b": _up(self.b, self.f32)}
        es = 4 if self.f32 else 2
        h = dev[over] if over else rt.DeviceBuffer(es * self.rows * self.cols)
        y = rt.DeviceBuffer(es * self.rows * self.cols)
        r_post, r_pre = rt.DeviceBuffer(4 * self.rows), rt.DeviceBuffer(4 * self.rows)
        rt.block_join_fwd(dev["x"].ptr, dev["b"].ptr, h.ptr, *shape, y=y.ptr if w["gamma_pre"] else None,
                          gate_rows=self.gate_rows, rstd_post=r_post.ptr, rstd_pre=r_pre.ptr, alpha=self.alpha, eps=EPS,
                          f32=self.f32, **{n: _ptr(v) for n, v in w.items()})
        rt.sync()
        want = O.block_join(self.x, self.b, self.gamma_post, self.gate, self.gate_rows, self.gamma_pre, self.alpha, EPS)
        gate = 1.0 if self.gate is None else np.repeat(np.abs(self.gate), self.gate_rows, 0)
        n = np.abs(self.b.astype(np.float64))
        if self.gamma_post is not None:
            n = n * want["rstd_post"][:, None] * np.abs(self.gamma_post)
            _close(r_post.download(np.float32, (self.rows,)), want["rstd_post"], want["rstd_post"], True, "rstd_post")
        size = self.alpha * np.abs(self.x) + gate * n
        _close(_down(h, shape, self.f32), want["h"], size, self.f32, "h")
        if self.gamma_pre is not None:
            # what the terms of h lose enters the mean of their squares too
            grow = np.sqrt(np.mean(size ** 2, 1) / (np.mean(want["h"] ** 2, 1) + EPS))
            _close(r_pre.download(np.float32, (self.rows,)), want["rstd_pre"], want["rstd_pre"] * (1 + grow), True, "rstd_pre")
            _close(_down(y, shape, self.f32), want["y"],
                   (size + np.abs(want["h"]) * grow[:, None]) * want["rstd_pre"][:, None] * np.abs(self.gamma_pre), self.f32, "y")

    def check_backward(self, accumulate=True, with_dh=True, over=None, wanted=("dgamma_post", "dgate", "dgamma_pre")):
        w, shape, f32 = self._weights(), (self.rows, self.cols), self.f32
        r_post = (1 / np.sqrt(np.mean(self.b.astype(np.float64) ** 2, 1) + EPS)).astype(np.float32)
        r_pre = (1 / np.sqrt(np.mean(self.h.astype(np.float64) ** 2, 1) + EPS)).astype(np.float32)
        pre, post = self.gamma_pre is not None, self.gamma_post is not None
        dev = {"b": _up(self.b, f32), "dh": _up(self.dh, f32) if with_dh else None,
               "h": _up(self.h, f32) if pre else None, "dy": _up(self.dy, f32) if pre else None}
        es = 4 if f32 else 2
        dx = dev[over[0]] if over else rt.DeviceBuffer(es * self.rows * self.cols)
        db = dev[over[1]] if over else rt.DeviceBuffer(es * self.rows * self.cols)
        sums = {n: rt.DeviceBuffer.from_numpy(a) for n, a in self.before.items() if n in wanted}
        groups = 1 if self.gate is None else self.gate.shape[0]
        need = rt.load().jpp_workspace_bytes(7, self.cols, groups, 0)
        ws = rt.DeviceBuffer.from_numpy(np.full(need // 4 + 16, np.nan, np.float32))
        post_dev, pre_dev = rt.DeviceBuffer.from_numpy(r_post), rt.DeviceBuffer.from_numpy(r_pre)
        rt.block_join_bwd(_ptr(dev["h"]), dev["b"].ptr, _ptr(dev["dh"]), _ptr(dev["dy"]), dx.ptr, db.ptr, *shape,
                          gate_rows=self.gate_rows, rstd_post=post_dev.ptr, rstd_pre=pre_dev.ptr, workspace=ws.ptr,
                          alpha=self.alpha, accumulate=accumulate, f32=f32, **{n: _ptr(v) for n, v in w.items()},
                          **{n: b.ptr for n, b in sums.items()})
        rt.sync()
        assert np.isnan(ws.download(np.float32, (16,), need)).all(), "wrote behind the workspace"
        want = O.block_join_bwd(self.h, self.b, self.dh if with_dh else None, self.dy, self.gamma_post, self.gate,
                                self.gate_rows, self.gamma_pre, r_post, r_pre, self.alpha)
        # absolute sizes of the terms
        gate = 1.0 if self.gate is None else np.repeat(np.abs(self.gate), self.gate_rows, 0)
        total = np.abs(self.dh).astype(np.float64) if with_dh else np.zeros(shape)
        size = {}
        if pre:
            hat = np.abs(self.h * r_pre[:, None].astype(np.float64))
            t = np.abs(self.dy * self.gamma_pre)
            total = total + r_pre[:, None] * (t + hat * np.mean(t * hat, 1, keepdims=True))
            size["dgamma_pre"] = (np.abs(self.dy) * hat).sum(0)
        n = np.abs(self.b).astype(np.float64)
        if post:
            n = n * r_post[:, None]
            u = total * gate * np.abs(self.gamma_post)
            size["db"] = r_post[:, None] * (u + n * np.mean(u * n, 1, keepdims=True))
            size["dgamma_post"] = (total * gate * n).sum(0)
            n = n * np.abs(self.gamma_post)
        else:
            size["db"] = total * gate
        if self.gate is not None:
            size["dgate"] = (total * n).reshape(-1, self.gate_rows, self.cols).sum(1)
        _close(_down(dx, shape, f32), want["dx"], self.alpha * total, f32, "dx")
        _close(_down(db, shape, f32), want["db"], size["db"], f32, "db")
        for name, buf in sums.items():
            got = buf.download(np.float32, self.before[name].shape)
            old = self.before[name] if accumulate else 0.0
            _close(got, want[name] + old, size[name] + np.abs(old), True, name)


# rows of one wave (up to 1024 bf16, 512 f32) and of a workgroup, whole and partly filled units
COLS = [8, 64, 520, 1000, 1024, 1032, 2048, 2056, 4096, 5000, 8184, 8192]


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("cols", COLS)
def test_widths(cols, f32):
    for rows in (1, 5, 131):
        p = Problem(rows, cols, f32, gate_rows=rows)
        p.check_forward()
        p.check_backward()


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("post,gate_rows,pre", [(True, 0, True), (False, 0, True), (False, 6, True), (True, 6, False), (False, 12, False),
                                                (True, 3, True), (True, 1, True)])
@pytest.mark.parametrize("cols", [264, 2064])
def test_parts_that_are_left_out(post, gate_rows, pre, cols, f32):
    p = Problem(12, cols, f32, post, gate_rows, pre, seed=1)
    p.check_forward()
    p.check_backward(accumulate=False)
    if pre:
        p.check_backward(with_dh=False)
    p.check_backward(wanted=("dgate",))
    p.check_backward(wanted=())


@pytest.mark.parametrize("gate_rows,rows", [(1, 1030), (2, 1030), (7, 1400), (515, 1030), (1030, 1030)])
def test_gates_of_many_rows_and_of_one(gate_rows, rows):
    """From a gate for every row to one for all: more gate rows than workgroups, and fewer."""
    Problem(rows, 136, False, gate_rows=gate_rows, seed=2).check_backward()
    Problem(rows, 1160, True, gate_rows=gate_rows, seed=2).check_backward(accumulate=False)


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("cols", [512, 4096])
def test_results_over_operands(cols, f32):
    for over in ("x", "b"):
        Problem(37, cols, f32, gate_rows=37).check_forward(over)
    for over in (("dh", "b"), ("dy", "b")):
        Problem(37, cols, f32, gate_rows=37).check_backward(over=over)


def test_rows_of_zeros_and_alpha_of_zero():
    p = Problem(9, 256, True, gate_rows=9, alpha=0.0)
    p.b[4] = 0
    p.h[4] = 0
    p.check_forward()
    p.check_backward()


def test_repeats_are_bit_identical_on_another_stream_and_in_a_graph():
    rows, cols = 700, 1536
    p = Problem(rows, cols, False, gate_rows=350, seed=5)
    keep = p._weights()
    w = {n: v.ptr for n, v in keep.items()}
    x, b, dh, dy = (_up(a, False) for a in (p.x, p.b, p.dh, p.dy))
    bufs = {n: rt.DeviceBuffer(2 * rows * cols) for n in ("h", "y", "dx", "db")}
    bufs.update({n: rt.DeviceBuffer(4 * rows) for n in ("rstd_post", "rstd_pre")})
    bufs.update(dgamma_post=rt.DeviceBuffer(4 * cols), dgamma_pre=rt.DeviceBuffer(4 * cols), dgate=rt.DeviceBuffer(8 * cols))
    ws = rt.DeviceBuffer(rt.load().jpp_workspace_bytes(7, cols, 2, 0))
    st = rt.Stream()

    def calls(stream):
        rt.block_join_fwd(x.ptr, b.ptr, bufs["h"].ptr, rows, cols, y=bufs["y"].ptr, gate_rows=350, alpha=0.9,
                          rstd_post=bufs["rstd_post"].ptr, rstd_pre=bufs["rstd_pre"].ptr, stream=stream, **w)
        rt.block_join_bwd(bufs["h"].ptr, b.ptr, dh.ptr, dy.ptr, bufs["dx"].ptr, bufs["db"].ptr, rows, cols, gate_rows=350,
                          alpha=0.9, workspace=ws.ptr, accumulate=False, stream=stream,
                          **{n: bufs[n].ptr for n in ("rstd_post", "rstd_pre", "dgamma_post", "dgamma_pre", "dgate")}, **w)

    def read():
        rt.sync()
        out = {n: v.download(np.uint32, (v.nbytes // 4,)) for n, v in bufs.items()}
        for v in (*bufs.values(), ws):
            v.zero()
        rt.sync()
        return out

    calls(None)
    want = read()
    calls(st.ptr)
    runs = [read()]
    graph = rt.Graph(st)
    with graph:
        calls(st.ptr)
    for _ in range(3):
        graph.launch()
        runs.append(read())
    for got in runs:
        for n in want:
            np.testing.assert_array_equal(got[n], want[n], err_msg=n)


@pytest.mark.parametrize("rows,cols,f32", [(2056, 8192, False), (16392, 1024, False), (4112, 4096, True)])
def test_gradients_of_more_than_the_caches(rows, cols, f32):
    """Gradients of 16 M elements and more are stored past the caches; a workgroup has several rows."""
    Problem(rows, cols, f32, gate_rows=rows // 2, seed=6).check_backward()


def test_more_elements_than_31_bits_count():
    """A few rows of tensors of 4 GiB and more are given and looked at."""
    rows, cols = (1 << 18) + 8, 8192
    pick = [0, 77, (1 << 18) - 1, (1 << 18) + 3, rows - 1]
    p = Problem(len(pick), cols, seed=10)
    dev = p._weights()
    w = {n: _ptr(v) for n, v in dev.items()}
    big = {n: rt.DeviceBuffer(2 * rows * cols) for n in ("x", "b", "h", "y", "dx", "db")}
    stat = {n: rt.DeviceBuffer(4 * rows) for n in ("rstd_post", "rstd_pre")}

    def put(buf, a):
        for i, r in enumerate(pick):
            buf.upload(rt.to_bf16_bits(a[i]), 2 * r * cols)

    def get(buf):
        return np.stack([rt.from_bf16_bits(buf.download(np.uint16, (cols,), 2 * r * cols)) for r in pick])

    put(big["x"], p.x)
    put(big["b"], p.b)
    rt.block_join_fwd(big["x"].ptr, big["b"].ptr, big["h"].ptr, rows, cols, y=big["y"].ptr, rstd_post=stat["rstd_post"].ptr,
                      rstd_pre=stat["rstd_pre"].ptr, alpha=p.alpha, eps=EPS, **w)
    rt.sync()
    want = O.block_join(p.x, p.b, p.gamma_post, None, 0, p.gamma_pre, p.alpha, EPS)
    size = p.alpha * np.abs(p.x) + np.abs(p.b) * want["rstd_post"][:, None] * np.abs(p.gamma_post)
    grow = np.sqrt(np.mean(size ** 2, 1) / (np.mean(want["h"] ** 2, 1) + EPS))[:, None]
    _close(get(big["h"]), want["h"], size, False, "h")
    _close(get(big["y"]), want["y"], (size + np.abs(want["h"]) * grow) * want["rstd_pre"][:, None] * np.abs(p.gamma_pre), False, "y")

    put(big["h"], p.h)
    put(big["x"], p.dh)
    put(big["y"], p.dy)
    r_post, r_pre = ((1 / np.sqrt(np.mean(a.astype(np.float64) ** 2, 1) + EPS)).astype(np.float32) for a in (p.b, p.h))
    for i, r in enumerate(pick):
        stat["rstd_post"].upload(r_post[i:i + 1], 4 * r)
        stat["rstd_pre"].upload(r_pre[i:i + 1], 4 * r)
    rt.block_join_bwd(big["h"].ptr, big["b"].ptr, big["x"].ptr, big["y"].ptr, big["dx"].ptr, big["db"].ptr, rows, cols,
                      rstd_post=stat["rstd_post"].ptr, rstd_pre=stat["rstd_pre"].ptr, alpha=p.alpha, **w)
    rt.sync()
    want = O.block_join_bwd(p.h, p.b, p.dh, p.dy, p.gamma_post, None, 0, p.gamma_pre, r_post, r_pre, p.alpha)
    hat, t = np.abs(p.h * r_pre[:, None].astype(np.float64)), np.abs(p.dy * p.gamma_pre)
    total = np.abs(p.dh) + r_pre[:, None] * (t + hat * np.mean(t * hat, 1, keepdims=True))
    n, u = np.abs(p.b) * r_post[:, None], total * np.abs(p.gamma_post)
    _close(get(big["dx"]), want["dx"], p.alpha * total, False, "dx")
    _close(get(big["db"]), want["db"], r_post[:, None] * (u + n * np.mean(u * n, 1, keepdims=True)), False, "db")
