"""Norms around a block with its gate and residual scale, and their gradients, against the formulas in float64 on the CPU.

Tolerances: an output is rounded once, half a step of its type (`eps / 2` relative). Before that each element is a product or sum of at most a dozen
float32 values, each off by at most 2^-24 relative (sigmoid: 4), and row statistics are sums of D terms of one sign added in chains of 8 and a
tree of at most 16 levels: 24 roundings. So C = 48 roundings of the largest magnitude that enters: of the sum for residual', of
(|residual'| / sigma) * |weight| for normed, of r * (|d| + |unit| * mean |d unit|) for a gradient. Sums over rows add `rows` such terms."""
import gc
import subprocess
import sys

import pytest
import torch

from conftest import ROOT
from helpers import DEV, gen

U = 2.0 ** -24
C = 48.0
EPS = 1e-6
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def run(*args, **kwargs):
    from triton_snn_fusion_amd.runtime.hip_block_norm_backend import run_hip_block_norm
    return run_hip_block_norm(*args, **kwargs)


def norm64(x, kind, eps=EPS):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)


def reference(v, kind, gate_form, factor):
    """float64 tensors with gradients on: residual', normed."""
    residual = v["residual"]
    if v.get("branch") is not None:
        y = norm64(v["branch"], kind)
        if v.get("branch_weight") is not None:
            y = y * v["branch_weight"]
        if v.get("gate") is not None:
            y = y * (v["gate"] * torch.sigmoid(v["gate"]) if gate_form == "silu" else torch.sigmoid(v["gate"]))
        if v.get("scale") is not None:
            y = y * v["scale"]
        residual = residual + factor * y
    normed = norm64(residual, kind)
    if v.get("next_weight") is not None:
        normed = normed * v["next_weight"]
    return residual, normed


NAMES = ("residual", "branch", "gate", "branch_weight", "next_weight", "scale")


def operands(lead, D, dtype, residual_dtype, vector_dtype, gate, scale, seed, weights=True):
    g = gen(seed)
    t = {"residual": (torch.randn(*lead, D, generator=g) * 2).to(residual_dtype), "branch": (torch.randn(*lead, D, generator=g) * 0.7 + 0.2).to(dtype)}
    t["gate"] = torch.randn(*lead, D, generator=g).to(dtype) if gate else None
    t["branch_weight"] = (torch.randn(D, generator=g) * 0.1 + 1).to(vector_dtype) if weights else None
    t["next_weight"] = (torch.randn(D, generator=g) * 0.1 + 1).to(vector_dtype) if weights else None
    t["scale"] = (torch.randn(D, generator=g) * 0.3 + 0.5).to(vector_dtype) if scale is True else scale
    grads = torch.randn(*lead, D, generator=g).to(residual_dtype), torch.randn(*lead, D, generator=g).to(dtype)
    return t, grads


def near(got, want, room, what):
    got, want = got.detach().double().cpu(), want.double()
    room = room + (torch.finfo(got_dtype[0]).eps / 2 * want.abs() if got_dtype[0] != torch.float32 else 0.0)
    if got_dtype[0] == torch.float16:
        room = room + 2.0 ** -25
    off = (got - want).abs()
    assert bool((off <= room).all()), f"{what}: off by at most {float(off.max()):.3g}, over the tolerance by {float((off - room).max()):.3g}"


got_dtype = [torch.float32]


def check(lead, D, dtype, kind="rms", gate="silu", scale=True, residual_dtype=None, vector_dtype=None, seed=1, weights=True):
    residual_dtype, vector_dtype = residual_dtype or dtype, vector_dtype or dtype
    t, (d_res, d_norm) = operands(lead, D, dtype, residual_dtype, vector_dtype, gate is not None, scale, seed, weights)
    dev = {n: (x.to(DEV).requires_grad_(True) if isinstance(x, torch.Tensor) else x) for n, x in t.items()}
    form = gate or "silu"
    out = run(dev["residual"], dev["branch"], gate=dev["gate"], branch_weight=dev["branch_weight"], next_weight=dev["next_weight"],
              scale=dev["scale"], kind=kind, gate_form=form, eps=EPS)
    leaves = [n for n in NAMES if isinstance(dev[n], torch.Tensor)]
    grads = torch.autograd.grad(out, [dev[n] for n in leaves], [d_res.to(DEV), d_norm.to(DEV)])
    torch.cuda.synchronize()
    with torch.no_grad():
        again = run(dev["residual"], dev["branch"], gate=dev["gate"], branch_weight=dev["branch_weight"], next_weight=dev["next_weight"],
                    scale=dev["scale"], kind=kind, gate_form=form, eps=EPS)
    assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])
    assert out[0].dtype == residual_dtype and out[1].dtype == dtype and out[0].shape == t["residual"].shape

    v = {n: t[n].double().requires_grad_(True) for n in leaves}
    factor = scale if isinstance(scale, float) else 1.0
    want = reference(v, kind, form, factor)
    want_grads = torch.autograd.grad(want, [v[n] for n in leaves], [d_res.double(), d_norm.double()], retain_graph=True)
    with torch.no_grad():
        # The sizes of the terms that enter, element by element, from the formulas
        def center(x):
            return x - x.mean(-1, keepdim=True) if kind == "layer" else x

        def sigma(x):
            return torch.sqrt((center(x) ** 2).mean(-1, keepdim=True) + EPS)

        act = 1.0 if v.get("gate") is None else (v["gate"].abs() + 1 if form == "silu" else torch.ones_like(v["gate"]))
        wb = v["branch_weight"].abs() if "branch_weight" in v else 1.0
        wn = v["next_weight"].abs() if "next_weight" in v else 1.0
        sc = (v["scale"].abs() if "scale" in v else 1.0) * abs(factor)
        unit = (v["branch"].abs() + v["branch"].abs().mean(-1, keepdim=True)) / sigma(v["branch"])
        size = v["residual"].abs() + unit * wb * act * sc
        unit2 = (size + size.mean(-1, keepdim=True)) / sigma(want[0])
        got_dtype[0] = residual_dtype
        near(out[0], want[0], C * U * size, "residual'")
        got_dtype[0] = dtype
        near(out[1], want[1], C * U * unit2 * wn, "normed")

        def through_norm(d, unit, x):
            return (d + unit * (d * unit).mean(-1, keepdim=True) + d.mean(-1, keepdim=True)) / sigma(x)
        d_size = d_res.double().abs() + through_norm(d_norm.double().abs() * wn, unit2, want[0])
        du = d_size * sc * act
        room = {"residual": C * U * d_size, "branch": C * U * through_norm(du * wb, unit, v["branch"]), "gate": C * U * d_size * sc * wb * unit * act}
        flat = lambda a: torch.broadcast_to(a, want[0].shape).reshape(-1, D).sum(0)  # noqa: E731
        room["branch_weight"] = C * U * flat(du * unit)
        room["next_weight"] = C * U * flat(d_norm.double().abs() * unit2)
        room["scale"] = C * U * flat(d_size * act * wb * unit) * abs(factor)
        for n, g, w in zip(leaves, grads, want_grads):
            assert g.dtype == t[n].dtype and g.shape == t[n].shape
            got_dtype[0] = t[n].dtype
            near(g, w, room[n], f"gradient of {n}")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", [(1, 1), (1, 1024), (3, 7), (5, 64), (9, 65), (6, 513), (130, 100), (2, 1025), (3, 2048), (2, 4096), (2, 5001), (1, 8192)])
def test_sizes(hip_ops, rows, D, dtype, kind):
    check((rows,), D, dtype, kind=kind, seed=rows + D)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [8200, 12288, 16384, 16383])
def test_widest_rows(hip_ops, D, dtype):
    check((3,), D, dtype, seed=D)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", ["silu", "sigmoid", None])
@pytest.mark.parametrize("scale", [True, None, 0.35])
def test_gates_and_scales(hip_ops, dtype, gate, scale):
    check((2, 11), 200, dtype, gate=gate, scale=scale, seed=3)
    check((7,), 77, dtype, kind="layer", gate=gate, scale=scale, weights=False, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [96, 1000, 777])
def test_float32_residual_and_vectors(hip_ops, dtype, D):
    check((17,), D, dtype, residual_dtype=torch.float32, seed=5)
    check((17,), D, dtype, vector_dtype=torch.float32, seed=6)
    check((17,), D, dtype, residual_dtype=torch.float32, vector_dtype=torch.float32, kind="layer", seed=7)


@pytest.mark.gpu
def test_many_rows(hip_ops):
    check((5000,), 72, torch.bfloat16, seed=8)
    check((4100,), 264, torch.float32, seed=9)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_without_a_branch(hip_ops, dtype):
    g = gen(10)
    x = torch.randn(4, 6, 333, generator=g).to(DEV, dtype).requires_grad_(True)
    w = (torch.randn(333, generator=g) * 0.1 + 1).to(DEV, dtype).requires_grad_(True)
    d = torch.randn(4, 6, 333, generator=g).to(DEV, dtype)
    residual, normed = run(x, next_weight=w)
    assert residual is x
    gx, gw = torch.autograd.grad(normed, [x, w], d)
    x64, w64 = x.detach().double().cpu().requires_grad_(True), w.detach().double().cpu().requires_grad_(True)
    want = norm64(x64, "rms") * w64
    wx, ww = torch.autograd.grad(want, [x64, w64], d.double().cpu())
    got_dtype[0] = dtype
    near(normed, want.detach(), C * U * 16.0, "normed")
    near(gx, wx, C * U * 64.0, "gradient of residual")
    near(gw, ww, C * U * 24 * 64.0, "gradient of next_weight")


@pytest.mark.gpu
def test_strided_rows_and_unused_outputs(hip_ops):
    g = gen(11)
    wide = torch.randn(3, 40, 3 * 130 + 1, generator=g).to(DEV, torch.bfloat16)
    parts = [wide[:, :, k * 130 + 1:(k + 1) * 130 + 1] for k in range(3)]
    a = run(parts[0], parts[1], gate=parts[2])
    b = run(*(p.contiguous() for p in parts[:2]), gate=parts[2].contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    turned = run(parts[0].transpose(0, 1), parts[1].transpose(0, 1), gate=parts[2].transpose(0, 1))
    assert torch.equal(turned[0], a[0].transpose(0, 1)) and torch.equal(turned[1], a[1].transpose(0, 1))
    # a gradient that reaches only one of the outputs, and an expanded one
    leaves = [p.contiguous().requires_grad_(True) for p in parts]
    for k in range(2):
        out = run(leaves[0], leaves[1], gate=leaves[2])
        lone = torch.autograd.grad(out[k].sum(), leaves)
        out = run(leaves[0], leaves[1], gate=leaves[2])
        zeros = [torch.zeros_like(o) for o in out]
        zeros[k] = torch.ones_like(out[k])
        both = torch.autograd.grad(out, leaves, zeros)
        assert all(torch.equal(x, y) for x, y in zip(lone, both))


@pytest.mark.gpu
def test_gates_at_the_ends_of_their_type(hip_ops):
    """A gate at its type's lowest value or minus infinity lets nothing through and has no slope; a sigmoid gate of infinity lets all through."""
    for dtype in DTYPES:
        g = gen(12)
        residual, branch = torch.randn(4, 64, generator=g).to(DEV, dtype), torch.randn(4, 64, generator=g).to(DEV, dtype)
        low = torch.finfo(dtype).min
        for form in ("silu", "sigmoid"):
            for value in (low, -float("inf")):
                gate = torch.full((4, 64), value, device=DEV, dtype=dtype).requires_grad_(True)
                out, _ = run(residual, branch, gate=gate, gate_form=form)
                assert torch.equal(out, residual)
                assert float(torch.autograd.grad(out.float().sum(), gate)[0].float().abs().max()) < 1e-30
        gate = torch.full((4, 64), float("inf"), device=DEV, dtype=dtype).requires_grad_(True)
        out, _ = run(residual, branch, gate=gate, gate_form="sigmoid")
        assert torch.equal(out, run(residual, branch)[0])
        assert float(torch.autograd.grad(out.float().sum(), gate)[0].float().abs().max()) == 0.0


@pytest.mark.gpu
def test_a_row_of_nan_stays_alone(hip_ops):
    g = gen(13)
    t = [torch.randn(6, 100, generator=g).to(DEV) for _ in range(3)]
    clean = run(t[0], t[1], gate=t[2])
    t[1][2, 5] = float("nan")
    dirty = run(t[0], t[1], gate=t[2])
    keep = [0, 1, 3, 4, 5]
    assert all(torch.equal(c[keep], d[keep]) and bool(d[2].isnan().any()) for c, d in zip(clean, dirty))


@pytest.mark.gpu
def test_gradient_against_differences(hip_ops):
    """Central differences of the operator itself, float32, step 2^-6: truncation and rounding stay below 1e-2 of the terms' sizes."""
    t, (d_res, d_norm) = operands((5,), 40, torch.float32, torch.float32, torch.float32, True, True, 14)
    dev = [t[n].to(DEV).requires_grad_(True) for n in NAMES]

    def call(x):
        return run(x[0], x[1], gate=x[2], branch_weight=x[3], next_weight=x[4], scale=x[5], kind="layer")
    grads = torch.autograd.grad(call(dev), dev, [d_res.to(DEV), d_norm.to(DEV)])
    step = 2.0 ** -6
    for k, n in enumerate(NAMES):
        way = torch.randn(t[n].shape, generator=gen(50 + k)).to(DEV)

        def loss(sign):
            out = call([x.detach() + (sign * step * way if i == k else 0) for i, x in enumerate(dev)])
            return (out[0].double() * d_res.to(DEV)).sum() + (out[1].double() * d_norm.to(DEV)).sum()
        slope = (loss(1) - loss(-1)) / (2 * step)
        assert abs(float(slope - (grads[k].double() * way).sum())) <= 1e-2 * float((grads[k].double() * way).abs().sum()), n


@pytest.mark.gpu
def test_graph_replays_and_other_streams(hip_ops):
    t, (d_res, d_norm) = operands((700,), 256, torch.bfloat16, torch.bfloat16, torch.bfloat16, True, True, 15)
    dev = [t[n].to(DEV).requires_grad_(True) for n in NAMES]
    d_res, d_norm = d_res.to(DEV), d_norm.to(DEV)

    def step():        # its autograd graph ends with it: none of the same leaves lives during a capture
        out = run(dev[0], dev[1], gate=dev[2], branch_weight=dev[3], next_weight=dev[4], scale=dev[5])
        return [*(t.detach() for t in out), *torch.autograd.grad(out, dev, [d_res, d_norm])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, step()))
    del on_side
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for k in range(4):
        with torch.no_grad():
            dev[1].copy_(torch.randn(700, 256, generator=gen(60 + k)).to(DEV, torch.bfloat16))
        want = [x.clone() for x in step()]
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_empty_and_refusals(hip_ops):
    x = torch.zeros(0, 8, device=DEV)
    assert run(x, x)[0].shape == (0, 8)
    x = torch.zeros(2, 8, device=DEV)
    for args, kwargs, words in (((x, x[:1]), {}, "unsupported_shape"), ((x, x.double()), {}, "unsupported_dtype"), ((x.half(), x), {}, "unsupported_dtype"),
                                ((x, x), {"gate": x.half()}, "unsupported_dtype"), ((x,), {"gate": x}, "without a branch"),
                                ((x, x), {"kind": "batch"}, "unsupported_kind"), ((x, x), {"gate_form": "tanh"}, "unsupported_gate"),
                                ((x, x), {"eps": -1.0}, "unsupported_eps"), ((x, x), {"scale": x[0, :4]}, "unsupported_shape"),
                                ((x.half(), x.half()), {"scale": x[0], "next_weight": x[0].half()}, "one dtype"),
                                ((x, x.cpu()), {}, "unsupported_device"), ((torch.zeros(1, 16385, device=DEV),), {}, "unsupported_shape")):
        with pytest.raises(RuntimeError, match=words):
            run(*args, **kwargs)


@pytest.mark.gpu
def test_python_implementation(hip_ops, monkeypatch):
    """What the dispatch module does not take runs in Python, on the same kernels: the same checks with the module out of the way, and equal bits."""
    from triton_snn_fusion_amd import _dispatch
    from triton_snn_fusion_amd.runtime import hip_block_norm_backend as backend
    t, grads = operands((33,), 130, torch.bfloat16, torch.float32, torch.float32, True, True, 21)
    dev = [t[n].to(DEV).requires_grad_(True) for n in NAMES]

    def step():
        out = run(dev[0], dev[1], gate=dev[2], branch_weight=dev[3], next_weight=dev[4], scale=dev[5])
        return [*out, *torch.autograd.grad(out, dev, [g.to(DEV) for g in grads])]
    assert _dispatch.module().block_norm(*dev, 1.0, 0, 2, EPS)[0].grad_fn is not None
    dispatched = step()
    monkeypatch.setattr(backend, "native", lambda t: None)
    assert all(torch.equal(a, b) for a, b in zip(step(), dispatched))
    for dtype in DTYPES:
        check((2, 5), 200, dtype, seed=22)
        check((9,), 77, dtype, kind="layer", gate=None, scale=0.5, seed=23)
    test_empty_and_refusals(hip_ops)


@pytest.mark.gpu
def test_differentiated_once(hip_ops):
    x = torch.randn(3, 16, device=DEV, requires_grad=True)
    out = run(x, x.detach() + 1)[1].sum()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(out, x, create_graph=True)[0].sum(), x)


def test_refusals_without_a_gpu():
    with pytest.raises(RuntimeError, match="unsupported_device"):
        run(torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="must be a tensor"):
        run(None)


def test_rows_too_wide_are_left_to_the_python_implementation(snnf_lib):
    """Widths that an int does not hold, 2^32 among them, which is 0 as an int: the dispatch module answers None before it divides by one."""
    code = ("import torch, triton_snn_fusion_amd\nfrom triton_snn_fusion_amd import _dispatch\nfrom torch._subclasses import FakeTensorMode\n"
            "module = _dispatch.module()\nwith FakeTensorMode():\n"
            "    for width in (16385, 1 << 32, (1 << 32) + 8):\n"
            "        x = torch.empty(2, width, dtype=torch.bfloat16, device='cuda')\n"
            "        assert module.block_norm(x, x, None, None, None, None, 1.0, 0, 2, 1e-6) is None\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, (done.returncode, done.stderr[-2000:])


@pytest.mark.gpu
def test_rows_too_wide_are_refused(hip_ops):
    for width in (16385, 1 << 32, (1 << 32) + 8):
        x = torch.empty(1, width, dtype=torch.bfloat16, device=DEV)
        with pytest.raises(RuntimeError, match="run_hip_block_norm: unsupported_shape: rows of 1 to 16384"):
            run(x, x)
        del x
    gc.collect()                        # the refusals' frames hold the tensors of 8 GB
    torch.cuda.empty_cache()


def test_entry_points_refuse_before_any_gpu_work(snnf_lib):
    def forward(rows=2, D=8, dtypes=(0, 0, 0), kind=0, gate_form=0, eps=1e-6, branch=16, gate=None, residual=16):
        return snnf_lib.snnf_block_norm(residual, 8, branch, 8, gate, 8, None, None, None, 1.0, rows, D, *dtypes, kind, gate_form, eps, 16, 16, None, None)
    assert forward(rows=-1) == -1 and forward(D=0) == -1 and forward(D=16385) == -2 and forward(dtypes=(0, 5, 0)) == -1
    assert forward(dtypes=(1, 0, 0)) == -2 and forward(dtypes=(0, 0, 1)) == -2 and forward(kind=2) == -1 and forward(gate_form=3) == -1
    assert forward(eps=-1.0) == -1 and forward(residual=None) == -1 and forward(gate_form=2) == -1 and forward(gate_form=2, branch=None, gate=16) == -1
    assert forward(rows=0, residual=None) == 0
    back = snnf_lib.snnf_block_norm_backward
    assert back(16, 8, 16, 8, None, 0, None, None, None, 1.0, None, 0, None, 0, 16, 2, 8, 0, 0, 0, 0, 0, 16, 16, None, None, None, None, None, 0, None) == -4
    assert back(16, 8, 16, 8, None, 0, None, None, None, 1.0, None, 0, None, 0, None, 2, 8, 0, 0, 0, 0, 0, 16, 16, None, None, None, None, 16, 1 << 20, None) == -1
    assert snnf_lib.snnf_block_norm_backward_workspace_bytes(0, 8) == 0 and snnf_lib.snnf_block_norm_backward_workspace_bytes(2, 16385) == 0
