"""The AdamW class: against adamw_step_ bit for bit, against torch.optim.AdamW, its states and state
dicts, captured steps, and a training step of blocks, loss, clipping and AdamW together."""

import copy
import io
import math

import pytest
import torch

import fussim_b200 as fb
from fussim_b200 import synthetic

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
SHAPES = [(7, 33), (300,), (1,), (4, 5, 3, 3), (2048,)]


def parameters(dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(s, generator=g) * 0.1).to(dtype).cuda()) for s in SHAPES]


def give_grads(params, step, dtype=None, skip=()):
    g = torch.Generator().manual_seed(1000 + step)
    for i, p in enumerate(params):
        t = (torch.randn(p.shape, generator=g) * 0.01).to(p.dtype).cuda()
        p.grad = None if i in skip else t


def equal(a, b):
    return all(torch.equal(x.detach().view(torch.uint8) if x.dtype == F8 else x.detach(),
                           y.detach().view(torch.uint8) if y.dtype == F8 else y.detach()) for x, y in zip(a, b))


@pytest.mark.parametrize("amsgrad_free", [dict(), dict(maximize=True), dict(weight_decay=0.0, betas=(0.5, 0.9), eps=1e-3)])
def test_like_torch(amsgrad_free):
    """Ten steps of 32 bits. Each step's two sides are off from the definition by some 20 u of the
    change (both moments, root, quotient and constants) and 4 u of the parameter; a change is at most
    10 rates (|m| / sqrt(v) with b1 = 0.9, b2 = 0.999), and what a step is off stays in the moments."""
    a = parameters()
    b = [torch.nn.Parameter(p.detach().double()) for p in a]
    lr = 1e-2
    ours = fb.AdamW(a, lr=lr, **amsgrad_free)
    ref = torch.optim.AdamW(b, lr=lr, **amsgrad_free)
    for step in range(10):
        skip = (1,) if step in (2, 3) else ()
        give_grads(a, step, skip=skip)
        for p, q in zip(a, b):
            q.grad = None if p.grad is None else p.grad.double()
        ours.step()
        ref.step()
    for p, q in zip(a, b):
        tol = 10 * (20 * U * 10 * lr + 4 * U * q.detach().abs().max())
        assert (p.detach().double() - q.detach()).abs().max() <= tol
        assert int(ours.state[p]["step"]) == int(ref.state[q]["step"])


@pytest.mark.parametrize("bits", [32, 8])
def test_like_the_function(bits):
    """Groups of different settings and counts of steps: the calls of adamw_step_ that they stand for."""
    a, b = parameters(), parameters()
    groups = lambda p: [dict(params=p[:2], lr=1e-3), dict(params=p[2:], weight_decay=0.1)]  # noqa: E731
    opt = fb.AdamW(groups(a), lr=3e-3, state_bits=bits, max_norm=0.05, seed=9)
    moments = [fb.adamw_moments(p, bits) for p in b]
    counts = [0] * 5
    for step in range(5):
        skip = (0, 3) if step == 1 else ()
        give_grads(a, step, skip=skip)
        give_grads(b, step, skip=skip)
        opt.step()
        norm = fb.grad_norm([p.grad for p in b if p.grad is not None])
        assert torch.equal(norm, opt.grad_norm)
        calls = 0
        for indices, kw in (((0, 1), dict(lr=1e-3)), ((2, 3, 4), dict(lr=3e-3, weight_decay=0.1))):
            batches = {}
            for i in indices:
                if b[i].grad is not None:
                    counts[i] += 1
                    batches.setdefault(counts[i], []).append(i)
            for t, batch in batches.items():
                fb.adamw_step_([b[i].detach() for i in batch], [b[i].grad for i in batch],
                               [moments[i][0] for i in batch], [moments[i][1] for i in batch],
                               [moments[i][2] for i in batch] if bits == 8 else None, step=t,
                               max_norm=0.05, norm=norm, seed=(9 + 0x9E3779B1 * calls) & 0xFFFFFFFF, **kw)
                calls += 1
    assert equal(a, b)
    for p, (first, second, scales) in zip(a, moments):
        assert equal([opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq"]], [first, second])


def test_master_weights():
    """16-bit parameters follow a 32-bit copy, which takes the steps of 32-bit parameters."""
    for bits in (32, 8):
        a = parameters(BF16)
        b = [torch.nn.Parameter(p.detach().float()) for p in a]
        opt = fb.AdamW(a, lr=1e-3, master_weights=True, state_bits=bits, seed=3)
        ref = fb.AdamW(b, lr=1e-3, state_bits=bits, seed=3)
        for step in range(4):
            give_grads(a, step)
            for p, q in zip(a, b):
                q.grad = p.grad.float()
            opt.step()
            ref.step()
        assert equal([opt.state[p]["master"] for p in a], b)
        assert equal(a, [q.detach().to(BF16) for q in b])


@pytest.mark.parametrize("kw", [dict(), dict(state_bits=8), dict(master_weights=True), dict(capturable=True),
                                dict(state_bits=8, master_weights=True, capturable=True)], ids=str)
def test_state_dict(kw):
    """A saved and loaded optimiser goes on with the same bits; so do a deep and a saved copy."""
    a = parameters(BF16)
    opt = fb.AdamW(a, lr=1e-3, **kw)
    for step in range(3):
        give_grads(a, step)
        opt.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    again = fb.AdamW(b, lr=5.0, **kw)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    c, third = copy.deepcopy((a, opt))
    file = io.BytesIO()  # (torch's own pickling: Python's alone does not know 8-bit floats)
    torch.save((a, opt), file)
    file.seek(0)
    d, fourth = torch.load(file, weights_only=False)
    for p in a:
        for k, v in opt.state[p].items():
            if isinstance(v, torch.Tensor):
                w = again.state[b[[x is p for x in a].index(True)]][k]
                assert v.dtype == w.dtype and v.stride() == w.stride()
    for step in range(3, 6):
        for params, o in ((a, opt), (b, again), (c, third), (d, fourth)):
            give_grads(params, step)
            o.step()
        assert equal(a, b) and equal(a, c) and equal(a, d)


def test_torch_state_dicts():
    """32-bit states from torch's optimiser and back into it."""
    a = parameters()
    ref = torch.optim.AdamW(a, lr=1e-2)
    for step in range(3):
        give_grads(a, step)
        ref.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ours = fb.AdamW(b)
    ours.load_state_dict(ref.state_dict())
    assert ours.param_groups[0]["lr"] == 1e-2 and ours.state[b[0]]["step"] == 3
    give_grads(a, 3)
    give_grads(b, 3)
    ref.step()
    ours.step()
    for p, q in zip(a, b):  # one step's roundings on both sides
        assert (p - q).abs().max() <= 2 * (20 * U * 10 * 1e-2 + 4 * U * p.detach().abs().max())
    back = torch.optim.AdamW([torch.nn.Parameter(q.detach().clone()) for q in b])
    back.load_state_dict(ours.state_dict())
    for q, r in zip(b, back.param_groups[0]["params"]):
        assert torch.equal(ours.state[q]["exp_avg"], back.state[r]["exp_avg"]) and int(back.state[r]["step"]) == 4
    with pytest.raises(ValueError, match="not of 8 bits"):
        fb.AdamW(parameters(), state_bits=8).load_state_dict(ref.state_dict())
    with pytest.raises(ValueError, match="amsgrad"):
        odd = fb.AdamW(b)
        state = torch.optim.AdamW(a, amsgrad=True).state_dict()
        odd.load_state_dict(state)
        odd.step()


def test_codes_and_strides():
    p = torch.nn.Parameter(torch.randn(4, 5, 3, 3, device="cuda").to(memory_format=torch.channels_last))
    opt = fb.AdamW([p], state_bits=8)
    p.grad = torch.randn_like(p)
    opt.step()
    q = torch.nn.Parameter(p.detach().contiguous())
    with pytest.raises(ValueError, match="strides"):
        fb.AdamW([q], state_bits=8).load_state_dict(opt.state_dict())


def test_captured_steps():
    a, b = parameters(), parameters()
    lr = torch.tensor(1e-2, device="cuda")
    opt = fb.AdamW(a, lr=lr, capturable=True, max_norm=0.05, state_bits=8)
    ref = fb.AdamW(b, lr=1e-2, max_norm=0.05, state_bits=8)
    give_grads(a, 0)
    give_grads(b, 0)
    opt.step()
    ref.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for step in range(1, 4):
        lr.fill_(1e-2 / step)
        ref.param_groups[0]["lr"] = lr.item()
        g = [torch.randn(p.shape, device="cuda") * 0.01 for p in a]
        for p, q, t in zip(a, b, g):
            p.grad.copy_(t)
            q.grad = t
        graph.replay()
        ref.step()
        assert torch.equal(opt.grad_norm, ref.grad_norm)
        assert equal(a, b)
    assert int(opt.state[a[0]]["step"]) == 4


def test_no_gradients_and_closure():
    a = parameters()
    opt = fb.AdamW(a, max_norm=1.0)
    before = [p.detach().clone() for p in a]
    assert opt.step() is None and equal(a, before) and opt.grad_norm is None

    def closure():
        opt.zero_grad()
        loss = sum((p * p).sum() for p in a)
        loss.backward()
        return loss

    first = opt.step(closure).item()
    assert opt.step(closure).item() < first


def test_loss_scaling():
    """torch's GradScaler: steps with infinite gradients are left out."""
    a = parameters()
    opt = fb.AdamW(a)
    scaler = torch.amp.GradScaler("cuda", init_scale=4.0)
    for bad in (False, True):
        before = [p.detach().clone() for p in a]
        loss = scaler.scale(sum((p * p).sum() for p in a))
        opt.zero_grad()
        loss.backward()
        if bad:
            a[0].grad[0, 0] = math.inf
        scaler.step(opt)
        scaler.update()
        assert equal(a, before) == bad


# ---- blocks, loss, clipping and AdamW together ----
class Block(torch.nn.Module):
    """A residual block over tokens: a modulated norm, two products, and a norm and gate behind them."""

    def __init__(self, c, plain):
        super().__init__()
        self.up, self.down = torch.nn.Linear(c, 2 * c), torch.nn.Linear(2 * c, c)
        self.weight, self.after = (torch.nn.Parameter(torch.ones(c)) for _ in range(2))
        self.bias = torch.nn.Parameter(torch.zeros(c))
        self.gate = torch.nn.Parameter(torch.full((c,), 0.3))
        self.plain = plain

    def forward(self, x, z, scale, shift):
        """(x, its norm z) to those of the next block."""
        y = self.down(torch.nn.functional.silu(self.up(z)))
        if not self.plain:
            return fb.gated_residual_norm(x, y, self.gate, self.weight, self.bias, scale=scale, shift=shift,
                                          kind="layer", branch_kind="rms", branch_weight=self.after, residual_scale=0.5)
        h = y * (y.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * self.after
        r = x + 0.5 * self.gate * h
        n = torch.nn.functional.layer_norm(r, r.shape[-1:], self.weight, self.bias, 1e-6)
        return r, n * (1 + scale[:, None]) + shift[:, None]


class Network(torch.nn.Module):
    """Patches of an image through blocks and back to an image."""

    def __init__(self, plain, c=48, depth=2):
        super().__init__()
        torch.manual_seed(5)
        self.inward, self.outward = torch.nn.Linear(48, c), torch.nn.Linear(c, 48)
        self.condition = torch.nn.Linear(3, 2 * c)
        self.blocks = torch.nn.ModuleList(Block(c, plain) for _ in range(depth))
        self.first = fb.BlockNorm(c)
        self.plain = plain

    def forward(self, image):
        b, _, h, w = image.shape
        t = image.view(b, 3, h // 4, 4, w // 4, 4).permute(0, 2, 4, 1, 3, 5).reshape(b, h * w // 16, 48)
        scale, shift = self.condition(image.mean((2, 3))).chunk(2, -1)
        x = self.inward(t)
        if self.plain:
            z = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * self.first.weight
        else:
            z = self.first(x)
        for block in self.blocks:
            x, z = block(x, z, scale, shift)
        t = self.outward(z).sigmoid().view(b, h // 4, w // 4, 3, 4, 4).permute(0, 3, 1, 4, 2, 5)
        return t.reshape(b, 3, h, w)


def test_training_steps():
    """Three steps of our operators beside torch's: the losses and parameters stay together. A step's
    differences are a few roundings (some 1e-6 of a gradient); AdamW turns that into at most a change of
    a rate where a gradient is itself rounding, and else into the same fraction of one."""
    kept = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        a, b = (t.cuda() for t in synthetic.pair_noise((2, 3, 64, 80), 0.1, seed=3))
        ours, ref = Network(False).cuda(), Network(True).cuda()
        lr = 1e-3
        opt = fb.AdamW(ours.parameters(), lr=lr, max_norm=0.5)
        other = torch.optim.AdamW(ref.parameters(), lr=lr)
        for _ in range(3):
            opt.zero_grad()
            other.zero_grad()
            loss, want = fb.l1_dssim_loss(ours(a).contiguous(), b), fb.l1_dssim_loss(ref(a).contiguous(), b)
            loss.backward()
            want.backward()
            assert abs(loss.item() - want.item()) <= 1e-5
            opt.step()
            norm = torch.nn.utils.clip_grad_norm_(ref.parameters(), 0.5)
            other.step()
            assert abs(opt.grad_norm.item() - norm.item()) <= 1e-3 * norm.item()
        worst = [((p - q).abs() > 0.05 * lr).float().mean().item() for p, q in zip(ours.parameters(), ref.parameters())]
        assert max(worst) <= 0.02
        assert all((p - q).abs().max() <= 2 * 3 * lr for p, q in zip(ours.parameters(), ref.parameters()))
    finally:
        torch.backends.cuda.matmul.allow_tf32 = kept


def test_captured_training_step():
    """A whole step in a graph: blocks, loss, backward pass, clipping and AdamW. Replays go as eager steps."""
    a, b = (t.cuda() for t in synthetic.pair_noise((1, 3, 32, 48), 0.1, seed=4))
    nets = [Network(False).cuda() for _ in range(2)]
    opts = [fb.AdamW(n.parameters(), lr=1e-3, capturable=True, max_norm=0.5, state_bits=8) for n in nets]

    def body(net, opt):
        params = list(net.parameters())
        loss = fb.l1_dssim_loss(net(a).contiguous(), b)
        for p, g in zip(params, torch.autograd.grad(loss, params)):
            p.grad = g
        opt.step()
        return loss.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for net, opt in zip(nets, opts):
            for _ in range(2):
                body(net, opt)
    torch.cuda.synchronize()
    assert equal(nets[0].parameters(), nets[1].parameters())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss = body(nets[0], opts[0])
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(side):
            want = body(nets[1], opts[1])
        torch.cuda.synchronize()
        # (the products of the blocks may go to other library kernels in a graph)
        assert abs(loss.item() - want.item()) <= 1e-5
    assert int(opts[0].state[next(nets[0].parameters())]["step"]) == 5
