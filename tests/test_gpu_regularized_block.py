"""The drop-in halves with their regularised ends (post-norm, layer scale,
residual scale, dropout, hidden dropout, the norm handed from the attention half
to the MLP half), run together as a block trains, against a 64-bit composition
of the oracle's pieces with the same seeds.

Tolerances (2-norm of the difference over that of the reference).  fp32: an fp32
sum of at most 4C = 512 terms is off by about sqrt(512) eps = 2.7e-6 of its
scale; a forward chains seven of them, a gradient about twice as many and the
normalisations' amplification of a few: 2e-5 and 1e-4.  Autocast: each of about
ten roundings to bf16 in a half's forward adds 2^-8 / sqrt(3) of its value's
norm, 1e-2 in all; twice that for y's branch term and four times for gradients.
A mask, a gate or a term left out is off by over a tenth.
"""
import pytest
import torch
import torch.nn.functional as F

from oracle import regularize as rg
from oracle import swin_oracle as so
from terra_amd import kernels
from terra_amd.mlp import SequentialMlp
from terra_amd.transformer import SequentialSwinTransformer

pytestmark = pytest.mark.gpu

OPTIONS = dict(post_norm=True, layer_scale=0.3, residual_scale=0.9, dropout=0.15)
SEEDS = (0x1122334455667788, 0x0F0E0D0C0B0A0908)


def _blocks(C, heads, ws, H, W, layer=1, mlp=True, **kw):
    torch.manual_seed(3)
    opts = {**OPTIONS, **kw}
    hidden = opts.pop("hidden_dropout", 0.2)
    attn = SequentialSwinTransformer(layer, H, W, C, window_size=ws, num_heads=heads, init_seed_base=5, **opts)
    blocks = [attn, SequentialMlp(C, 4 * C, init_seed_base=6, hidden_dropout=hidden, **opts)]
    g = torch.Generator().manual_seed(7)
    with torch.no_grad():
        for b in blocks:
            for n, p in b.named_parameters():
                if "scale" in n or "norm" in n:
                    p.add_(0.1 * torch.randn(p.shape, generator=g))
                elif p.dim() == 2 and "table" not in n:
                    p.copy_(torch.randn(p.shape, generator=g) / p.shape[1] ** 0.5)
                else:
                    p.copy_(0.3 * torch.randn(p.shape, generator=g))
    return blocks


def _seeds(monkeypatch, dev):
    """Fixed seeds, in the order of the halves' draws."""
    given = iter(SEEDS * 4)
    monkeypatch.setattr(kernels, "dropout_seed", lambda *a, **k: torch.tensor([next(given)], device=dev))


def _oracle(blocks, x, train, hand_over):
    """(y, gradients by name) of the two halves in float64."""
    attn, mlp = blocks
    ps = {}
    for prefix, b in zip(("a.", "m."), blocks):
        ps.update({prefix + n: p.detach().double().cpu().requires_grad_() for n, p in b.named_parameters()})
    x = x.double().cpu().requires_grad_()
    B, L, C = x.shape
    geom, H, W = attn.geometry(B), *attn.input_resolution
    ws, s = attn.window_size, attn.shift_size

    def norm(prefix, module):
        return None if module is None else (ps[prefix + ".weight"], ps[prefix + ".bias"], module.eps, False)

    p = attn.dropout if train else 0.0
    n1 = F.layer_norm(x, (C,), ps["a.norm1.weight"], ps["a.norm1.bias"], attn.norm1.eps)
    win = so.partition_frame(n1.view(B, H, W, C), ws, s, s, geom.pad, geom.win_row_begin, geom.win_rows, geom.valid)
    lin = lambda t, n: F.linear(t, ps[n + ".weight"], ps[n + ".bias"])  # noqa: E731
    mask = so.shift_mask(geom.frame_h, geom.frame_w, ws, s) if s else None
    if mask is not None and geom.win_rows is not None:
        per = geom.cols
        mask = mask[geom.win_row_begin * per:(geom.win_row_begin + geom.rows) * per]
    o = so.window_attention_core(*(lin(win, f"a.attn.{n}_linear") for n in "qkv"), attn.attn.num_heads, attn.attn.scale,
                                 ps["a.attn.relative_position_bias_table"], (ws, ws), mask, compute_dtype=torch.float64)
    h = lin(o, "a.attn.proj")
    nxt = norm("m.norm2", mlp.norm2)
    y, z = rg.residual_norm(h, x.view(B, H, W, C), norm("a.post_norm1", attn.post_norm1), ps.get("a.layer_scale1"), nxt, geom,
                            attn.residual_scale, p, SEEDS[0], 0)
    y, z = y.view(B, L, C), z.view(B, L, C)
    seed = SEEDS[1] if p > 0 else SEEDS[0]
    hp, p = (mlp.hidden_dropout, mlp.dropout) if train else (0.0, 0.0)
    a = rg.dropout(rg.gelu(lin(z, "m.fc1")), hp, seed, 1)
    y, _ = rg.residual_norm(lin(a, "m.fc2"), y, norm("m.post_norm2", mlp.post_norm2), ps.get("m.layer_scale2"), None, None,
                            mlp.residual_scale, p, seed, 0)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(9), dtype=torch.float64)
    g = torch.autograd.grad(y, [x, *ps.values()], dy, allow_unused=True)
    return y.detach(), dict(zip(["x", *ps], g)), dy


def _run(blocks, x, dy, dev, hand_over):
    attn, mlp = blocks
    x = x.to(dev).requires_grad_()
    if hand_over:
        y, z = attn(x, next_norm=mlp.norm2)
        y = mlp(y, normed=z)
    else:
        y = mlp(attn(x))
    names = ["x"] + [p + n for p, b in zip(("a.", "m."), blocks) for n, _ in b.named_parameters()]
    ps = [x] + [p for b in blocks for p in b.parameters()]
    return y.detach(), dict(zip(names, torch.autograd.grad(y, ps, dy.to(dev, y.dtype))))


def _rel(got, ref, scale=None):
    got, ref = got.detach().double().cpu(), ref.double()
    return ((got - ref).norm() / (ref if scale is None else scale).norm()).item()


def _check_gradients(g, ref, tol):
    """The key bias moves all scores of a query alike, which a softmax does not
    see: its gradient is 0 exactly, a sum of terms that cancel.  Their scale is
    that of the query bias's gradient, a sum over the same rows of the same
    products with k in place of q."""
    for n in ref:
        scale = ref["a.attn.q_linear.bias"] if n == "a.attn.k_linear.bias" else None
        assert _rel(g[n], ref[n], scale) <= tol, n


@pytest.mark.parametrize("hand_over", [False, True])
@pytest.mark.parametrize("C,heads,ws,kw", [
    (96, 3, 7, {}), (96, 3, 7, dict(layer=0, post_norm=False)), (128, 4, 8, dict(layer_scale=None)),
    (128, 4, 8, dict(dropout=0.0)), (128, 4, 8, dict(hidden_dropout=0.0, residual_scale=1.0)),
])
def test_block_trains_as_the_oracle(dev, monkeypatch, C, heads, ws, kw, hand_over):
    H, W = 2 * ws, 3 * ws
    blocks = _blocks(C, heads, ws, H, W, **kw)
    x = torch.randn(2, H * W, C, generator=torch.Generator().manual_seed(8))
    y_ref, g_ref, dy = _oracle(blocks, x, True, hand_over)
    blocks = [b.to(dev).train() for b in blocks]
    _seeds(monkeypatch, dev)
    y, g = _run(blocks, x, dy, dev, hand_over)
    assert _rel(y, y_ref) <= 2e-5
    _check_gradients(g, g_ref, 1e-4)
    # in evaluation the ends stay and dropout goes
    y_ref, _, _ = _oracle(blocks, x, False, hand_over)
    blocks = [b.eval() for b in blocks]
    with torch.no_grad():
        y = blocks[1](blocks[0](x.to(dev)))
    assert _rel(y, y_ref) <= 2e-5


def test_slab_with_padding_and_partial_windows(dev, monkeypatch):
    """A rank's slab: padding rows, window rows left out, pad windows; tokens that no window holds keep alpha x."""
    ws, H, W, C = 8, 24, 16, 96
    torch.manual_seed(3)
    attn = SequentialSwinTransformer(1, H, W, C, window_size=ws, num_heads=3, init_seed_base=5, pad=(0, 8, 0, 0),
                                     win_row_begin=1, win_rows=2, valid_windows=(1, 4), **OPTIONS)
    blocks = [attn, SequentialMlp(C, 4 * C, init_seed_base=6, hidden_dropout=0.2, **OPTIONS)]
    x = torch.randn(2, H * W, C, generator=torch.Generator().manual_seed(8))
    y_ref, g_ref, dy = _oracle(blocks, x, True, False)
    blocks = [b.to(dev).train() for b in blocks]
    _seeds(monkeypatch, dev)
    y, g = _run(blocks, x, dy, dev, False)
    assert _rel(y, y_ref) <= 2e-5
    _check_gradients(g, g_ref, 1e-4)


@pytest.mark.parametrize("hand_over", [False, True])
def test_block_under_autocast(dev, monkeypatch, hand_over):
    C, heads, ws = 192, 6, 8
    H, W = 16, 24
    blocks = _blocks(C, heads, ws, H, W)
    x = torch.randn(2, H * W, C, generator=torch.Generator().manual_seed(8))
    y_ref, g_ref, dy = _oracle(blocks, x, True, hand_over)
    blocks = [b.to(dev).train() for b in blocks]
    _seeds(monkeypatch, dev)
    with torch.amp.autocast("cuda", dtype=torch.bfloat16):
        y, g = _run(blocks, x, dy, dev, hand_over)
    assert y.dtype == torch.float32
    base = x.double() * 0.81
    assert _rel(y.cpu() - base, y_ref - base) <= 2e-2
    assert all(t.dtype == torch.float32 for t in g.values())
    _check_gradients(g, g_ref, 4e-2)


def test_off_by_default(dev):
    """Without the options nothing changes: parameter names, and results bit for bit whatever the mode."""
    torch.manual_seed(0)
    attn = SequentialSwinTransformer(1, 16, 16, 96, window_size=8, num_heads=3, init_seed_base=5)
    mlp = SequentialMlp(96, 384, init_seed_base=6, drop=0.5)
    assert not any("post_norm" in n or "layer_scale" in n for b in (attn, mlp) for n in b.state_dict())
    attn, mlp = attn.to(dev), mlp.to(dev)
    x = torch.randn(1, 256, 96, device=dev)
    outs = []
    for train in (True, False):
        with torch.no_grad():
            outs.append(mlp.train(train)(attn.train(train)(x)))
    assert torch.equal(*outs)
    quiet = SequentialSwinTransformer(1, 16, 16, 96, window_size=8, num_heads=3, init_seed_base=5, dropout=0.5).to(dev).eval()
    with torch.no_grad():
        assert torch.equal(quiet(x), attn(x))


def test_dropout_of_the_modules(dev):
    """torch's seed fixes the masks; calls differ; the rate is p."""
    attn, mlp = (b.to(dev).train() for b in _blocks(96, 3, 7, 14, 14, layer_scale=None, post_norm=False, dropout=0.3))
    x = torch.randn(1, 196, 96, device=dev)
    for b in (attn, mlp):
        with torch.no_grad():
            torch.manual_seed(4)
            first = b(x)
            second = b(x)
            torch.manual_seed(4)
            assert torch.equal(b(x), first) and not torch.equal(first, second)
            dropped = (first == b.residual_scale * x).float().mean().item()
        # 18816 draws: a rate of 0.3 is off by more than 5 sigma = 0.017 once in 1.7 million
        assert abs(dropped - 0.3) < 0.017


def test_bad_options():
    for kw in (dict(dropout=-0.1), dict(dropout=1.5), dict(dropout=float("nan"))):
        with pytest.raises(ValueError, match="dropout"):
            SequentialSwinTransformer(0, 16, 16, 96, window_size=8, num_heads=3, **kw)
        with pytest.raises(ValueError, match="dropout"):
            SequentialMlp(96, 384, **kw)
    with pytest.raises(ValueError, match="hidden_dropout"):
        SequentialMlp(96, 384, hidden_dropout=2.0)


def test_empty_batch_and_out(dev):
    attn, mlp = (b.to(dev).train() for b in _blocks(96, 3, 7, 14, 14))
    y, z = attn(torch.empty(0, 196, 96, device=dev), next_norm=mlp.norm2)
    assert y.shape == z.shape == (0, 196, 96)
    assert mlp(y, normed=z).shape == (0, 196, 96) and mlp(y).shape == (0, 196, 96)
    x = torch.randn(1, 196, 96, device=dev)
    with pytest.raises(ValueError, match="out is for"):
        mlp(x, out=torch.empty_like(x))


def test_layers_of_another_kind_are_called(dev):
    """A hook on a layer sees and may change its output, and a layer of another class runs its own forward,
    in the regularised path as in the others."""
    _, mlp = _blocks(96, 3, 7, 14, 14, dropout=0.0, hidden_dropout=0.25)
    mlp = mlp.to(dev).train()
    x = torch.randn(1, 196, 96, device=dev)
    with torch.no_grad():
        torch.manual_seed(4)
        want = mlp(x)
        for name in ("fc1", "fc2", "act"):
            seen = []
            handle = getattr(mlp, name).register_forward_hook(lambda m, i, o: seen.append(o.shape))
            torch.manual_seed(4)
            assert (mlp(x) - want).norm() <= 2e-5 * want.norm() and len(seen) == 1
            handle.remove()

        class Halved(torch.nn.Linear):
            def forward(self, v):
                return super().forward(v) / 2

        fc2 = Halved(384, 96).to(dev)
        fc2.load_state_dict({k: 2 * v for k, v in mlp.fc2.state_dict().items()})
        mlp.fc2 = fc2
        torch.manual_seed(4)
        assert (mlp(x) - want).norm() <= 2e-5 * want.norm()


def test_checkpointing_repeats_the_masks(dev):
    from torch.utils.checkpoint import checkpoint

    blocks = [b.to(dev).train() for b in _blocks(96, 3, 7, 14, 14)]
    x = torch.randn(1, 196, 96, device=dev, requires_grad=True)
    for b in blocks:
        torch.manual_seed(8)
        y = b(x)
        want, = torch.autograd.grad(y.sum(), x)
        torch.manual_seed(8)
        again = checkpoint(b, x, use_reentrant=False)
        got, = torch.autograd.grad(again.sum(), x)
        # bit for bit but for the LayerNorm gather's sums, which do not reach x's gradient
        assert torch.equal(again, y) and torch.equal(got, want)


def test_frozen_parameters_and_inference(dev):
    """A gradient for a gate or for the input alone, and calls in inference mode."""
    blocks = [b.to(dev).train() for b in _blocks(96, 3, 7, 14, 14)]
    x = torch.randn(1, 196, 96, device=dev)
    for b, gate in zip(blocks, (blocks[0].layer_scale1, blocks[1].layer_scale2)):
        torch.manual_seed(9)
        want = torch.autograd.grad(b(x.requires_grad_()).sum(), (x, gate))
        x.requires_grad_(False)
        b.requires_grad_(False)
        gate.requires_grad_(True)
        torch.manual_seed(9)
        assert torch.equal(torch.autograd.grad(b(x).sum(), gate)[0], want[1])
        gate.requires_grad_(False)
        torch.manual_seed(9)
        assert torch.equal(torch.autograd.grad(b(x.requires_grad_()).sum(), x)[0], want[0])
        torch.manual_seed(9)
        y = b(x)
        x.requires_grad_(False)
        torch.manual_seed(9)
        with torch.inference_mode():
            assert (b(x) - y.detach()).norm() <= 2e-5 * y.detach().norm()


def _captured(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


def _step_of(attn, mlp, x, dy):
    params = [p for b in (attn, mlp) for p in b.parameters()]

    def step():
        y, z = attn(x, next_norm=mlp.norm2)
        y = mlp(y, normed=z)
        return y.detach(), torch.autograd.grad(y, params, dy)

    return step


def test_captured_step_draws_new_masks(dev):
    attn, mlp = (b.to(dev).train() for b in _blocks(96, 3, 7, 14, 14))
    x, dy = torch.randn(2, 196, 96, device=dev), torch.randn(2, 196, 96, device=dev)
    graph, (y, grads) = _captured(_step_of(attn, mlp, x, dy))
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(y.clone())
        assert all(bool(torch.isfinite(g).all()) for g in grads)
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_captured_step_gives_the_eager_results(dev, monkeypatch):
    """With seeds from buffers: every replay, with new inputs and seeds, against the
    eager pass (y bit for bit; gradients to 1e-5, since the LayerNorm gather's backward
    sums its parameters' with atomics)."""
    attn, mlp = (b.to(dev).train() for b in _blocks(96, 3, 7, 14, 14))
    seeds = [torch.tensor([s], device=dev) for s in SEEDS]
    calls = iter(range(1 << 30))
    monkeypatch.setattr(kernels, "dropout_seed", lambda *a, **k: seeds[next(calls) % 2])
    x, dy = torch.randn(2, 196, 96, device=dev), torch.randn(2, 196, 96, device=dev)
    step = _step_of(attn, mlp, x, dy)
    graph, (y, grads) = _captured(step)
    for i in range(3):
        for s in seeds:
            s.add_(i)
        x.add_(0.1 * i)
        graph.replay()
        torch.cuda.synchronize()
        y_ref, g_ref = step()
        assert torch.equal(y, y_ref)
        for a, b in zip(grads, g_ref):
            assert (a - b).norm() <= 1e-5 * b.norm() + 1e-4  # 1e-4: the key bias's, which is 0 and rounding
