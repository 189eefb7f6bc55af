"""The block operators together, as a causal layer over the frames of every site uses them - trained on whole clips and then
run one frame at a time - and the 8-bit checkpoints inside the training backend's ResnetBlocks.

Tolerances, set before the first run; u = 2^-8 (half a step of bfloat16), v = 2^-4 (of an e4m3 code).
Layer: an output passes through six roundings to bfloat16 in a row (norm, qkv, attention core twice, projection, sum), each u / sqrt(3)
in the 2-norm of what it rounds, the sums adding what they do not share: sqrt(6) u / sqrt(3) of the branch, under 2 u.  A
gradient passes as many again: 4 u.  A weight's gradient from kept rows adds v / sqrt(3).
ResnetBlock: the kept rows enter a gradient through both norms (twice each: the normalised row and the slope of SiLU) and
once as the convolution's input, each v / sqrt(3): under 4 v / sqrt(3)."""
import pytest
import torch

from tests.helpers import new_graph, record, rel_err

gpu = pytest.mark.gpu
DEV = "cuda:0"
U, V = 2.0 ** -8, 2.0 ** -4


class Layer(torch.nn.Module):
    def __init__(self, c, heads, d):
        super().__init__()
        self.heads, self.d = heads, d
        g = torch.Generator().manual_seed(c)
        rnd = lambda *s: torch.randn(*s, generator=g)
        P = torch.nn.Parameter
        self.wqkv, self.bqkv = P(rnd(3 * heads * d, c) * c ** -0.5), P(0.1 * rnd(3 * heads * d))
        self.wout, self.bout = P(rnd(c, heads * d) * (heads * d) ** -0.5), P(0.1 * rnd(c))
        self.norm, self.post, self.next = P(1 + 0.1 * rnd(c)), P(1 + 0.1 * rnd(c)), P(1 + 0.1 * rnd(c))
        self.register_buffer("log_decay", torch.log1p(-torch.exp2(-torch.linspace(2, 6, heads))))

    def forward(self, x, mod, state=None, lengths=None):
        """x [b, frames, sites, c]; mod [b, 5, c] (scale, shift, gate, and scale, shift of the norm that follows)."""
        from video_diffusion_amd import block_hip as B
        b, f, s, c = x.shape
        scale, shift, gate, scale2, shift2 = (m.contiguous() for m in mod.unbind(1))
        y = B.norm_before(x, self.norm, scale, shift, kind="layer")
        qkv = B.linear_rows8(y, self.wqkv, self.bqkv).view(b, f, s, 3, self.heads, self.d)
        q, k, v = (t.permute(0, 2, 1, 3, 4) for t in qkv.unbind(3))
        if f == 1 and state is not None:
            o = B.decay_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], self.log_decay, state).unsqueeze(2)
            last = state
        else:
            o, last = B.decay_attention(q, k, v, self.log_decay, initial_state=state, lengths=lengths, return_state=True)
        o = o.permute(0, 2, 1, 3, 4).reshape(b, f, s, self.heads * self.d)
        h = B.linear_rows8(o, self.wout, self.bout)
        out, nxt = B.norm_between(x, h, self.post, gate, self.next, scale2, shift2, alpha=0.9, kind="rms", post_kind="rms")
        return out, nxt, last

    def exact(self, x, mod):
        """The layer in float64 from its float32 parameters."""
        p = {k: v.double() for k, v in self.named_parameters()} | {"log_decay": self.log_decay.double()}
        return self.exact_of(x, mod, p)

    def exact_of(self, x, mod, p):
        b, f, s, c = x.shape
        row = lambda i: mod[:, i, None, None]
        m = x - x.mean(-1, keepdim=True)
        y = m / torch.sqrt((m * m).mean(-1, keepdim=True) + 1e-5) * p["norm"] * (1 + row(0)) + row(1)
        qkv = (y @ p["wqkv"].t() + p["bqkv"]).view(b, f, s, 3, self.heads, self.d)
        q, k, v = (t.permute(0, 2, 3, 1, 4) for t in qkv.unbind(3))                     # [b, s, heads, f, d]
        t = torch.arange(f, device=x.device, dtype=torch.float64)
        gap = t[:, None] - t[None, :]
        D = torch.where(gap >= 0, torch.exp(p["log_decay"].view(-1, 1, 1) * gap.clamp(min=0)), torch.zeros((), dtype=torch.float64, device=x.device))
        o = self.d ** -0.5 * ((q @ k.mT) * D) @ v
        h = o.permute(0, 3, 1, 2, 4).reshape(b, f, s, -1) @ p["wout"].t() + p["bout"]
        h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5) * p["post"]
        out = 0.9 * x + row(2) * h
        nxt = out / torch.sqrt((out * out).mean(-1, keepdim=True) + 1e-5) * p["next"] * (1 + row(3)) + row(4)
        return out, nxt


def setup(b, f, s, c, heads, d):
    layer = Layer(c, heads, d).to(DEV)
    g = torch.Generator(device=DEV).manual_seed(f)
    x = torch.randn(b, f, s, c, generator=g, device=DEV).to(torch.bfloat16)
    mod = 0.3 * torch.randn(b, 5, c, generator=g, device=DEV)
    ups = [torch.randn(b, f, s, c, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]
    return layer, x, mod, ups


@gpu
@pytest.mark.parametrize("b,f,s,c,heads,d", [(2, 10, 16, 64, 8, 32), (1, 70, 5, 128, 2, 64), (3, 1, 9, 96, 2, 32)])
def test_layer_trains(b, f, s, c, heads, d):
    layer, x, mod, ups = setup(b, f, s, c, heads, d)
    xr, mr = x.clone().requires_grad_(), mod.clone().requires_grad_()
    out, nxt, _ = layer(xr, mr)
    names = [n for n, _ in layer.named_parameters()]
    grads = torch.autograd.grad((out, nxt), (xr, mr, *layer.parameters()), ups)
    x64, m64 = x.double().requires_grad_(), mod.double().requires_grad_()
    p64 = {k: v.detach().double().requires_grad_() for k, v in layer.named_parameters()} | {"log_decay": layer.log_decay.double()}
    want = layer.exact_of(x64, m64, p64)
    refs = torch.autograd.grad(want, (x64, m64, *(p64[n] for n in names)), [t.double() for t in ups])
    for name, a, r in (("out", out, want[0]), ("next", nxt, want[1])):
        assert record(f"layer.{f}.{name}", rel_err(a.detach(), r.detach()), 2 * U) < 2 * U, name
    for name, a, r in zip(("x", "mod", *names), grads, refs):
        bar = 4 * U + (V / 3 ** 0.5 if name in ("wqkv", "wout") else 0)
        assert record(f"layer.{f}.d{name}", rel_err(a, r), bar) < bar, name


@gpu
def test_layer_runs_frame_by_frame():
    """A clip at once, a prompt and then single frames, and a clip handed over in two pieces agree."""
    layer, x, mod, _ = setup(2, 12, 6, 64, 2, 32)
    with torch.no_grad():
        out, nxt, last = layer(x, mod)
        first, _, state = layer(x[:, :8], mod)
        assert torch.equal(first, out[:, :8])
        rest, _, end = layer(x[:, 8:], mod, state.clone())
        frames = [layer(x[:, t:t + 1], mod, state)[0] for t in range(8, 12)]
    for got in (rest, torch.cat(frames, 1)):
        assert rel_err(got, out[:, 8:]) < 2 * U
    assert rel_err(end, last) < 1e-5 and rel_err(state, last) < 1e-5


@gpu
def test_layer_in_a_graph():
    """Forward and backward captured; replays against eager runs.  (Every eager graph over these leaves has ended before the
    capture: while one lives, torch's engine ties the captured backward to the stream of its leaves' accumulators, which
    invalidates the capture and ends the process.)"""
    layer, x, mod, ups = setup(1, 10, 4, 64, 2, 32)
    x.requires_grad_()
    mod.requires_grad_()
    leaves = (x, mod, *layer.parameters())

    def run():
        out, nxt, _ = layer(x, mod)
        return [out.detach(), nxt.detach(), *torch.autograd.grad((out, nxt), leaves, ups)]

    run()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = new_graph()
    with torch.cuda.graph(graph):
        outs = run()
    g = torch.Generator(device=DEV).manual_seed(3)
    for _ in range(3):
        with torch.no_grad():
            for t in (x, mod, *ups):
                t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, run()))


def _block(cin, cout, seed=0):
    from video_diffusion_amd.modules import ResnetBlock
    torch.manual_seed(seed)
    return ResnetBlock(cin, cout, time_emb_dim=32).to(DEV)


@gpu
@pytest.mark.parametrize("cin,cout", [(64, 64), (64, 128), (128, 64)])
def test_resnet_block_with_rows8_checkpoints(cin, cout):
    """Same output bits; gradients that see the kept rows rounded to 8 bits."""
    from video_diffusion_amd import train_hip as T
    rb = _block(cin, cout)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(2, cin, 3, 16, 16, generator=g, device=DEV).to(torch.bfloat16).requires_grad_()
    temb = torch.randn(2, 32, generator=g, device=DEV)
    dout = torch.randn(2, cout, 3, 16, 16, generator=g, device=DEV).to(torch.bfloat16)
    leaves = [x, *rb.parameters()]
    names = ["x", *(n for n, _ in rb.named_parameters())]
    plain = T.resnet_block(rb, x, temb)
    want = torch.autograd.grad(plain, leaves, dout)
    with T.rows8_checkpoints():
        kept = T.resnet_block(rb, x, temb)
    got = torch.autograd.grad(kept, leaves, dout)            # outside the block: the choice was made in the forward
    assert torch.equal(plain, kept)
    bar = 4 * V / 3 ** 0.5
    for n, a, b in zip(names, got, want):
        assert record(f"rows8_resnet.{cin}.{cout}.{n}", rel_err(a, b), bar) < bar, n
    with T.rows8_checkpoints(False):
        again = torch.autograd.grad(T.resnet_block(rb, x, temb), leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    # an input gradient alone
    with T.rows8_checkpoints():
        (dx,) = torch.autograd.grad(T.resnet_block(rb, x, temb), x, dout)
    assert torch.equal(dx, got[0])


@gpu
def test_rows8_checkpoints_hold_less():
    from video_diffusion_amd import train_hip as T
    rb = _block(128, 128)
    x = torch.randn(2, 128, 8, 64, 64, device=DEV).to(torch.bfloat16).requires_grad_()
    temb = torch.randn(2, 32, device=DEV)

    def held(on):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with T.rows8_checkpoints(on):
            out = T.resnet_block(rb, x, temb)
        torch.cuda.synchronize()
        n = torch.cuda.memory_allocated() - before - out.numel() * 2
        out.backward(torch.ones_like(out))
        rb.zero_grad()
        x.grad = None
        return n

    held(False)
    rows = x.numel()
    full, small = held(False), held(True)
    # y1, h1, y2 as rows (the input is the caller's; a permuted copy of it is kept too) against codes and exponents
    assert full >= 3 * 2 * rows and small <= 4 * rows * (1 + 1 / 32) + (1 << 22)


@gpu
def test_unet_trains_with_rows8_checkpoints():
    """A whole denoiser on the hip backend: every gradient there, finite and near the one without (the roundings of the
    layers' kept rows add up along the way back: the bar is on their direction)."""
    from video_diffusion_amd import Unet3D
    from video_diffusion_amd import train_hip as T
    torch.manual_seed(0)
    unet = Unet3D(dim=64, dim_mults=(1, 2), channels=3).to(DEV)
    unet.train_backend = "hip"
    x, t = torch.randn(1, 3, 4, 16, 16, device=DEV), torch.tensor([7], device=DEV)

    def grads(on):
        unet.zero_grad(set_to_none=True)
        with T.rows8_checkpoints(on):
            loss = unet(x, t).square().mean()
        loss.backward()
        return float(loss), {n: p.grad.clone() for n, p in unet.named_parameters() if p.grad is not None}

    l0, a = grads(False)
    l1, b = grads(True)
    assert l0 == l1 and a.keys() == b.keys()
    assert all(torch.isfinite(g).all() for g in b.values())
    dot = sum(float((a[n].double() * b[n].double()).sum()) for n in a)
    na, nb = (sum(float(g.double().square().sum()) for g in z.values()) ** 0.5 for z in (a, b))
    assert record("rows8_unet.direction", 1 - dot / (na * nb), 4 * V / 3 ** 0.5) < 4 * V / 3 ** 0.5


def test_rows8_checkpoints_nest():
    from video_diffusion_amd import train_hip as T
    assert T._ROWS8 is False
    with T.rows8_checkpoints():
        assert T._ROWS8 is True
        with T.rows8_checkpoints(False):
            assert T._ROWS8 is False
        assert T._ROWS8 is True
    assert T._ROWS8 is False


@gpu
def test_trainer_keeps_rows_in_8_bits(tmp_path, monkeypatch):
    """Trainer.rows8_checkpoints: the blocks of every micro-step pack their rows, the first loss is the one without."""
    from tests.test_training import _write_gifs
    from video_diffusion_amd import GaussianDiffusion, Trainer, Unet3D, VAE, block_hip
    folder = str(tmp_path / "gifs")
    _write_gifs(folder, n=4, frames=6, size=36)
    packs = []
    real = block_hip.pack_rows8
    monkeypatch.setattr(block_hip, "pack_rows8", lambda x: packs.append(tuple(x.shape)) or real(x))

    def run(on):
        packs.clear()
        torch.manual_seed(0)
        gd = GaussianDiffusion(Unet3D(dim=64, dim_mults=(1, 2), channels=4), VAE(channels=3, latent_dim=4, base_dim=64),
                               image_size=32, num_frames=4, channels=3, timesteps=50).to(DEV)
        tr = Trainer(gd, folder, num_prev_frames=2, train_batch_size=2, train_num_steps=2, gradient_accumulate_every=1,
                     step_start_ema=0, update_ema_every=1, save_and_sample_every=10 ** 6, results_folder=str(tmp_path / f"r{on}"))
        tr.train_backend = "hip"
        tr.rows8_checkpoints = on
        torch.manual_seed(1)
        logs = []
        tr.train(log_fn=logs.append)
        return [l["loss"] for l in logs], len(packs)

    (a, none), (b, some) = run(False), run(True)
    assert none == 0 and some > 0 and some % 8 == 0          # four row sets a block, the same blocks in both steps
    assert a[0] == b[0] and all(x == x and abs(x) < 1e30 for x in b)


@gpu
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_a_block_packs_nothing_where_no_backward_can_follow(mode, monkeypatch):
    """Sampling inside a rows8_checkpoints block, with parameters that ask for gradients."""
    from video_diffusion_amd import block_hip, train_hip as T
    rb = _block(64, 128)
    x, temb = torch.randn(1, 64, 2, 8, 8, device=DEV).to(torch.bfloat16), torch.randn(1, 32, device=DEV)
    packs = []
    real = block_hip.pack_rows8
    monkeypatch.setattr(block_hip, "pack_rows8", lambda t: packs.append(t.shape) or real(t))
    with T.rows8_checkpoints():
        want = T.resnet_block(rb, x, temb)
        assert len(packs) == 4
        with mode():
            got = T.resnet_block(rb, x, temb)
        assert len(packs) == 4 and torch.equal(got, want)


def test_rows8_checkpoints_belong_to_their_thread():
    """The switch holds for the forward of the thread that set it."""
    import threading
    from video_diffusion_amd import train_hip as T
    seen, inside, done = [], threading.Event(), threading.Event()

    def other():
        inside.wait(10)
        seen.append(T._ROWS8)
        with T.rows8_checkpoints(False):
            seen.append(T._ROWS8)
        with T.rows8_checkpoints():
            seen.append(T._ROWS8)
            done.set()

    t = threading.Thread(target=other)
    t.start()
    with T.rows8_checkpoints():
        inside.set()
        done.wait(10)
        assert T._ROWS8 is True
    t.join(10)
    assert T._ROWS8 is False and seen == [False, False, True]


@gpu
def test_rows8_checkpoints_and_recomputation():
    """torch.utils.checkpoint around a block: its context_fn sets the switch for the recomputation too, which runs during the
    backward, outside the `with` of the forward; gradients are those without recomputation."""
    from torch.utils.checkpoint import checkpoint
    from video_diffusion_amd import train_hip as T
    rb = _block(64, 64)
    x = torch.randn(1, 64, 2, 16, 16, device=DEV).to(torch.bfloat16).requires_grad_()
    temb = torch.randn(1, 32, device=DEV)
    leaves = [x, *rb.parameters()]
    with T.rows8_checkpoints():
        want = T.resnet_block(rb, x, temb)
    dout = torch.randn_like(want)
    grads = torch.autograd.grad(want, leaves, dout)
    got = checkpoint(lambda x: T.resnet_block(rb, x, temb), x, use_reentrant=False,
                     context_fn=lambda: (T.rows8_checkpoints(), T.rows8_checkpoints()))
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, dout), grads))
