"""Training-step calls as programs make them: tensors off their boundaries, tracing and mapping,
mixed devices, autocast, gradients that are kept.

Tolerances are those of test_training_gpu.py, derived there; comparisons of two calls that run the
same kernels on the same values are bitwise.
"""

import pytest
import torch

from test_training_gpu import (BF16_TOL, EPS, NORM_TYPES, TOL, check, conv_reference, gen,
                               norm_inputs, rel)

pytestmark = pytest.mark.gpu


def arm():
    import armhackathon_b200 as a
    return a


# ---------------------------------------------------------------------------
# causal conv1d + SiLU
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,dim,length", [(1, 3, 5000), (2, 2, 4097), (1, 1, 700)])
@pytest.mark.parametrize("kernel", [4, 8])
def test_conv_backward_of_tensors_that_lie_alike_off_a_boundary(batch, dim, length, kernel, dtype):
    # x, dout and dx start the same number of elements past a 16-byte boundary, and few rows are
    # split in time: the C entry sets no rule for where they start
    from armhackathon_b200 import _ffi
    g = gen(length)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w, bias = r(dim, kernel), r(dim)
    n, code = batch * dim * length, {torch.float32: 0, torch.bfloat16: 1}[dtype]
    for off in range(1, 4 if dtype == torch.float32 else 8):
        x, dout, dx = (r(n + 16).to(dtype) for _ in range(3))
        guard = dx.clone()
        cut = lambda t: t[off:off + n].view(batch, dim, length)  # noqa: E731
        dw, db = torch.empty_like(w), torch.empty_like(bias)
        nbytes = _ffi.conv_silu_backward_workspace_bytes(batch, dim, length, kernel)
        ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
        _ffi.conv_silu_backward_raw(batch, dim, length, kernel, code, cut(dout).data_ptr(),
                                    cut(x).data_ptr(), w.data_ptr(), bias.data_ptr(), ws.data_ptr(),
                                    nbytes, cut(dx).data_ptr(), dw.data_ptr(), db.data_ptr(),
                                    torch.cuda.current_stream().cuda_stream)
        want = conv_reference(cut(dout), cut(x), w, bias)
        # a channel's dbias may be a small rest of its terms, whose rounding is relative to them
        pre = torch.nn.functional.conv1d(torch.nn.functional.pad(cut(x).double(), (kernel - 1, 0)),
                                         w.double()[:, None], bias.double(), groups=dim)
        s = torch.sigmoid(pre)
        terms = (cut(dout).double() * s * (1 + pre * (1 - s))).norm() / want["db"].norm()
        assert rel(cut(dx), want["dx"]) <= (BF16_TOL if dtype == torch.bfloat16 else TOL), off
        assert rel(dw, want["dw"]) <= TOL, off
        assert rel(db, want["db"]) <= TOL * max(1.0, float(terms)), off
        assert torch.equal(dx[:off], guard[:off]) and torch.equal(dx[off + n:], guard[off + n:])


@pytest.mark.parametrize("length", [64, 77])
def test_conv_autograd_in_16_bits(length):
    g = gen(length)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, w, bias, dout = r(2, 30, length).to(torch.bfloat16), r(30, 4), r(30), r(2, 30, length)
    want = conv_reference(dout, x, w, bias)
    leaves = [t.clone().requires_grad_() for t in (x, w, bias)]
    out = arm().causal_conv1d_silu(*leaves)
    assert out.dtype == torch.float32
    (out * dout).sum().backward()
    got = [t.grad for t in leaves]
    assert got[0].dtype == torch.bfloat16
    check(dict(zip(("dx", "dw", "db"), got)), want, TOL)


def test_conv_differentiates_weights_of_another_device():
    g = gen(8)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, w, bias, dout = r(2, 12, 60), r(12, 1, 4), r(12), r(2, 12, 60)

    def grads(where):
        leaves = [t.clone().requires_grad_() for t in (x, w.to(where), bias.to(where))]
        (arm().causal_conv1d_silu(*leaves) * dout).sum().backward()
        return [t.grad for t in leaves]

    for got, want, where in zip(grads("cpu"), grads("cuda"), ("cuda", "cpu", "cpu")):
        assert got.device.type == where and torch.equal(got.cpu(), want.cpu())


# ---------------------------------------------------------------------------
# selective scan
def bf16_scan(seed, lead=()):
    """Arguments of a scan with bfloat16 activations; ``lead``: further leading axes of these."""
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    act = lambda *s: r(*lead, *s).to(torch.bfloat16)  # noqa: E731
    b, d, length, n = 2, 40, 50, 16
    inp = dict(u=act(b, d, length), delta=act(b, d, length),
               A=-torch.arange(1, n + 1, device="cuda").float().repeat(d, 1),
               B=act(b, 1, n, length), C=act(b, 1, n, length), D=r(d), z=act(b, d, length),
               delta_bias=r(d) - 3, initial_state=r(b, d, n))
    return inp, r(b, d, length), r(b, d, n)


def test_bf16_scan_differentiates_small_inputs_of_another_device():
    inp, dout, dlast = bf16_scan(1)

    def grads(where):
        leaves = {k: (t.to(where) if t.dtype == torch.float32 else t).clone().requires_grad_()
                  for k, t in inp.items()}
        out, last = arm().selective_scan(**leaves, delta_softplus=True, return_last_state=True)
        ((out * dout).sum() + (last * dlast).sum()).backward()
        return {k: t.grad for k, t in leaves.items()}

    want, got = grads("cuda"), grads("cpu")
    for k, t in got.items():
        assert t.dtype == inp[k].dtype
        assert t.device.type == ("cpu" if inp[k].dtype == torch.float32 else "cuda"), k
        assert torch.equal(t.cpu(), want[k].cpu()), k


def test_bf16_scan_traces_in_one_graph():
    inp, dout, dlast = bf16_scan(2)

    def call(inp):
        return arm().selective_scan(**inp, delta_softplus=True, return_last_state=True)

    def grads(f):
        leaves = {k: t.clone().requires_grad_() for k, t in inp.items()}
        out, last = f(leaves)
        ((out * dout).sum() + (last * dlast).sum()).backward()
        return [out, last, *[t.grad for t in leaves.values()]]

    torch._dynamo.reset()
    want = grads(call)
    got = grads(torch.compile(call, fullgraph=True, backend="aot_eager"))
    assert all(p.dtype == q.dtype and torch.equal(p, q) for p, q in zip(got, want))
    # one parameter of an evaluated model that requires grad is enough
    some = {**inp, "A": inp["A"].clone().requires_grad_()}
    out, _ = torch.compile(call, fullgraph=True, backend="aot_eager")(some)
    assert torch.equal(out, want[0])


def test_bf16_scan_maps_over_an_axis():
    inp, _, _ = bf16_scan(3, lead=(3,))
    inp["A"].requires_grad_()
    acts = [inp[k] for k in ("u", "delta", "B", "C", "z")]

    def call(u, delta, B, C, z):
        return arm().selective_scan(u, delta, inp["A"], B, C, D=inp["D"], z=z,
                                    delta_bias=inp["delta_bias"], delta_softplus=True)

    got = torch.func.vmap(call)(*acts)
    want = torch.stack([call(*[t[i] for t in acts]) for i in range(3)])
    assert torch.equal(got, want)


def test_bf16_scan_op_checks():
    inp, _, _ = bf16_scan(4)
    args = [inp[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial_state")]
    args = [t.clone().requires_grad_() for t in args]
    checks = ("test_schema", "test_autograd_registration", "test_faketensor",
              "test_aot_dispatch_dynamic")
    for flags in ((True, False), (True, True)):
        torch.library.opcheck(torch.ops.arm_scan.selective_scan_bf16, (*args, *flags),
                              test_utils=checks)


@pytest.mark.parametrize("inside", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("leaf", [None, "A", "u"])
def test_scan_of_tensors_without_memory(dtype, leaf, inside):
    # what a trace sees, within the mode that made them and outside it
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    mode = FakeTensorMode()
    inp = {k: mode.from_tensor(t.to(dtype) if t.dtype == torch.bfloat16 else t)
           for k, t in bf16_scan(5)[0].items()}
    if leaf:
        inp[leaf].requires_grad_()

    def run():
        out, last = arm().selective_scan(**inp, delta_softplus=True, return_last_state=True)
        if leaf:
            (out.sum() + last.sum()).backward()
        return out, last

    if inside:
        with mode:
            out, last = run()
    else:
        out, last = run()
    assert isinstance(out, FakeTensor) and out.dtype == last.dtype == torch.float32
    assert out.shape == inp["u"].shape and last.shape == inp["initial_state"].shape
    if leaf:
        g = inp[leaf].grad
        assert isinstance(g, FakeTensor) and g.shape == inp[leaf].shape
        assert g.dtype == inp[leaf].dtype


# ---------------------------------------------------------------------------
# the patch in 16 bits
def tiny_mamba(dtype=torch.float32):
    from transformers import MambaConfig, MambaForCausalLM
    cfg = MambaConfig(vocab_size=500, hidden_size=64, state_size=16, num_hidden_layers=2, expand=2,
                      conv_kernel=4, time_step_rank=8, use_cache=False)
    torch.manual_seed(0)
    return MambaForCausalLM(cfg).cuda().to(dtype)


@pytest.fixture
def seen(monkeypatch):
    """The conv's outputs and what the scan is given, call by call."""
    from armhackathon_b200 import hf_patch
    conv, scan, got = hf_patch.causal_conv1d_silu, hf_patch.selective_scan, []

    def conv1d(*a):
        got.append([conv(*a)])
        return got[-1][0]

    def selective_scan(u, *a, **kw):
        got[-1].append(u)
        return scan(u, *a, **kw)

    monkeypatch.setattr(hf_patch, "causal_conv1d_silu", conv1d)
    monkeypatch.setattr(hf_patch, "selective_scan", selective_scan)
    return got


def patched(call, training=False):
    assert arm().patch(training=training)
    try:
        return call()
    finally:
        assert arm().unpatch()


def test_patched_inference_under_autocast_scans_the_conv_in_32_bits(seen):
    model = tiny_mamba().eval()
    ids = torch.randint(0, 500, (2, 33), device="cuda")
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        logits = patched(lambda: model(ids).logits)
    assert len(seen) == 2 and torch.isfinite(logits).all()
    for conv, u in seen:
        assert u.dtype == torch.float32 and torch.equal(u, conv)


@pytest.mark.parametrize("own_x_proj", [False, True])
def test_patched_inference_of_a_bf16_model(seen, own_x_proj):
    # 16-bit weights throughout, or with an x_proj that is kept in fp32
    model = tiny_mamba(torch.bfloat16).eval()
    ids = torch.randint(0, 500, (2, 33), device="cuda")
    with torch.no_grad():
        if own_x_proj:
            from torch import nn

            class Wide(nn.Linear):
                def forward(self, x):
                    return super().forward(x).to(torch.bfloat16)

            for block in model.backbone.layers:
                p = block.mixer.x_proj
                wide = Wide(p.in_features, p.out_features, bias=False).cuda()
                wide.weight.copy_(p.weight.float())
                block.mixer.x_proj = wide
        got = patched(lambda: model(ids).logits)
        assert len(seen) == 2 and torch.isfinite(got).all()
        for conv, u in seen:
            assert u.dtype == (torch.float32 if own_x_proj else torch.bfloat16)
            assert torch.equal(u, conv.to(u.dtype))


@pytest.mark.parametrize("autocast", [False, True])
def test_patched_training_in_16_bits(seen, autocast):
    model = tiny_mamba(torch.float32 if autocast else torch.bfloat16).train()
    ids = torch.randint(0, 500, (2, 33), device="cuda")

    def step():
        model.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            loss = model(ids, labels=ids).loss
        loss.backward()
        return {n: p.grad for n, p in model.named_parameters()}

    grads = patched(step, training=True)
    assert len(seen) == 2 and all(u.dtype == torch.bfloat16 for _, u in seen)
    for n, p in model.named_parameters():
        assert grads[n].dtype == p.dtype and torch.isfinite(grads[n]).all(), n


# ---------------------------------------------------------------------------
# RMS norm
def test_norm_fp8_refuses_gradients():
    x = torch.randn(6, 64, device="cuda", generator=gen(5))
    res, w = torch.randn(6, 64, device="cuda", generator=gen(6)), torch.ones(64, device="cuda")
    want = arm().add_rms_norm_fp8(x, w, residual=res)
    for leaf in (x, w, res):
        leaf.requires_grad_()
        got = arm().add_rms_norm_fp8(x, w, residual=res)  # the call itself runs as ever
        for p, q in zip(got, want):
            assert p.dtype == q.dtype and torch.equal(p.detach().float(), q.float())
        for t in got:  # and no gradient is dropped on the way back
            with pytest.raises(RuntimeError, match="add_rms_norm_fp8"):
                t.float().sum().backward()
        with torch.no_grad():
            assert not any(t.requires_grad for t in arm().add_rms_norm_fp8(x, w, residual=res))
        leaf.requires_grad_(False)
    assert not any(t.requires_grad for t in want)


# ---------------------------------------------------------------------------
# clipping
def test_clip_is_noticed_by_autograd():
    p = torch.randn(50, device="cuda", generator=gen(7)).requires_grad_()
    g, = torch.autograd.grad((p ** 3).sum(), p, create_graph=True)
    penalty = (g * g).sum()  # keeps g for its own gradient
    before = g._version
    arm().grad_norm([g.detach()])
    assert g._version == before
    arm().clip_grads_([g.detach(), torch.ones(3, device="cuda")], 0.1)
    assert g._version > before
    with pytest.raises(RuntimeError, match="inplace operation"):
        penalty.backward()
    with torch.inference_mode():
        arm().clip_grads_([torch.ones(3, device="cuda")], 0.1)


# ---------------------------------------------------------------------------
# several turns of the persistent loops
@pytest.mark.parametrize("types", NORM_TYPES)
@pytest.mark.parametrize("rows,dim", [(4001, 40), (4001, 768), (4001, 33), (1501, 1030), (1501, 2560),
                                      (701, 5000), (701, 4099)])
def test_norm_backward_of_many_rows(rows, dim, types):
    # each warp or CTA takes several rows and the last turn is not full: rows loaded ahead, the
    # alternating buffer of the sums, dw in registers
    x, res, w = norm_inputs(rows, dim, types, seed=dim)
    dy, extra, _ = norm_inputs(rows, dim, types, seed=dim + 1)
    stored = (res.double().square().mean(-1) + EPS).rsqrt().float()
    for dres in (extra, None):
        rl, wl = res.double().requires_grad_(), w.double().requires_grad_()
        y = rl * (rl.square().mean(-1, keepdim=True) + EPS).rsqrt() * wl
        total = (y * dy.double()).sum() + (0 if dres is None else (rl * dres.double()).sum())
        wantr, wantw = torch.autograd.grad(total, [rl, wl])
        dx, dr, dw = arm().add_rms_norm_backward(dy, res, w, stored, dresidual_out=dres)
        # a difference: its rounding is relative to its parts
        parts = float((dy.double() * w.double() * stored.double()[:, None]).norm() / wantr.norm())
        check({"dx": dx, "dr": dr, "dw": dw}, {"dx": wantr, "dr": wantr, "dw": wantw},
              TOL * max(1.0, parts))
        # and row by row, so that one stale row shows
        off = (dr.double() - wantr).norm(dim=-1) / wantr.norm(dim=-1)
        assert float(off.max()) <= (BF16_TOL if dr.dtype == torch.bfloat16 else 4 * TOL)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clip_of_more_chunks_than_ctas(dtype):
    sizes = [9_000_001, 5, 7_654_321, 16384 * 200 + 3]
    flat = torch.randn(sum(sizes) + 1, device="cuda", generator=gen(9)).to(dtype)
    grads = list(torch.split(flat[1:], sizes))
    first, before = flat[0].clone(), flat[1:].double()
    norm = arm().clip_grads_(grads, 2.0)
    want = before.norm()
    assert rel(norm, want) <= TOL
    # one factor (3 roundings) and a product, each value on its own
    lim = (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -22) * before.abs() * float(2 / want)
    lim = lim + (1e-38 if dtype == torch.bfloat16 else 1e-44)
    assert ((flat[1:].double() - before * float(2 / (want + 1e-6))).abs() <= lim).all()
    assert torch.equal(flat[0], first)


@pytest.mark.parametrize("tensors", [3, 700])
def test_clip_captured_in_a_graph(tensors):
    a = arm()
    values = [torch.randn(40 + i, device="cuda", generator=gen(i)) for i in range(tensors)]
    grads = [torch.empty_like(v) for v in values]

    def fill(scale):
        for p, v in zip(grads, values):
            p.copy_(v * scale)

    fill(1.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a.clip_grads_(grads, 0.5)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = a.clip_grads_(grads, 0.5)
    for scale in (1.0, 3.0, 1e-5):
        fill(scale)
        want_norm = a.clip_grads_(grads, 0.5)
        want = [p.clone() for p in grads]
        fill(scale)
        graph.replay()
        assert torch.equal(norm, want_norm)
        assert all(torch.equal(p, q) for p, q in zip(grads, want))
