"""The operators together: the ViT that takes images of any size, against plain torch in
64 bits, packed against one by one, and trained by the Trainer with AdamW."""

import math

import pytest
import torch

from npairloss_amd import NPairLossConfig, NPairMultiClassLoss
from npairloss_amd.config.params import SolverConfig
from npairloss_amd.engine import AdamW, Trainer
from npairloss_amd.models import RotaryViTB16, build_embedding_model
from npairloss_amd.models.embedding import EmbeddingNet
from transformer_util import DEVICES, U

SMALL = dict(patch=4, dim=48, depth=2, heads=3, embed_dim=24, softcap=8.0)
SIZES = [(8, 12), (4, 4), (20, 16), (12, 8), (28, 4), (16, 16), (8, 8)]
# Six products a block sum at most 192 terms, each off by 192 U of its terms' magnitudes,
# which are some 14 times the sum (random signs): 6 * 192 * 14 U = 1e-3 of the largest
# value a block, two blocks, and as much again for the norms and softmax between them.
FORWARD = 4 * 6 * 192 * 14 * U
# A gradient passes all of it twice.
BACKWARD = 2 * FORWARD


def model_of(device, seed=0, **more):
    torch.manual_seed(seed)
    m = RotaryViTB16(**{**SMALL, **more})
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() == 1:
                p.add_(0.1 * torch.randn(p.shape))
    return m.to(device)


def plain(params, image, cfg, amplitude=1.0):
    """One image's embedding, fp64, written out."""
    p, dim, H = cfg["patch"], cfg["dim"], cfg["heads"]
    D = dim // H
    rows, cols = image.shape[1] // p, image.shape[2] // p
    x = torch.stack([image[:, r * p:(r + 1) * p, c * p:(c + 1) * p].reshape(-1) for r in range(rows) for c in range(cols)])
    x = torch.cat([params["cls"][None], x @ params["patch_embed.weight"].T + params["patch_embed.bias"]])
    pos = torch.tensor([[0, 0]] + [[r + 1, c + 1] for r in range(rows) for c in range(cols)], dtype=torch.float64)
    f = 100.0 ** (-torch.arange(D // 4, dtype=torch.float64) / (D // 4))
    angle = torch.cat([pos[:, :1] * f, pos[:, 1:] * f], 1)[:, None]

    def norm(t, w):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w

    def turn(t):
        a, b = t[..., :D // 2], t[..., D // 2:]
        c, s = torch.cos(angle) * amplitude, torch.sin(angle) * amplitude
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    for i in range(cfg["depth"]):
        g = lambda n: params[f"blocks.{i}.{n}"]  # noqa: E731,B023
        h = norm(x, g("norm1"))
        q, k, v = (h @ g("qkv.weight").T + g("qkv.bias")).view(-1, 3, H, D).unbind(1)
        s = torch.einsum("ihd,jhd->hij", turn(q), turn(k)) / math.sqrt(D)
        if cfg["softcap"]:
            s = cfg["softcap"] * torch.tanh(s / cfg["softcap"])
        a = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(-1, dim)
        x = x + a @ g("out.weight").T + g("out.bias")
        h = norm(x, g("norm2")) @ g("mlp.0.weight").T + g("mlp.0.bias")
        x = x + torch.nn.functional.gelu(h) @ g("mlp.2.weight").T + g("mlp.2.bias")
    return norm(x[0], params["norm"]) @ params["proj.weight"].T + params["proj.bias"]


def images_of(device, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(3, h, w, generator=g).to(device) for h, w in SIZES]


def doubled(m):
    return {n: p.detach().double().cpu().requires_grad_() for n, p in m.named_parameters()}


def near(got, want, part, what):
    got, want = got.detach().double().cpu(), want.detach()
    assert float((got - want).abs().max()) <= part * float(want.abs().max()), what


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("row_length", [0, 40, 71])
def test_packed_with_gradients(row_length, device):
    """Rows of several images, of one, with padding behind."""
    m, images = model_of(device), images_of(device)
    out = m.forward_packed(images, row_length)
    params = doubled(m)
    want = torch.stack([plain(params, im.double().cpu(), SMALL) for im in images])
    near(out, want, FORWARD, "embeddings")
    dy = torch.randn(want.shape, generator=torch.Generator().manual_seed(2))
    out.backward(dy.to(device))
    want.backward(dy.double())
    for n, p in m.named_parameters():
        near(p.grad, params[n].grad, BACKWARD, n)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scaling", [None, "ramp"])
def test_batch(device, scaling):
    more = {} if scaling is None else dict(scaling=scaling, factor=2.0, original_length=10 ** 9)  # every pair turns often: kept, amplitude alone
    m = model_of(device, **more)
    x = torch.randn(3, 3, 12, 20, generator=torch.Generator().manual_seed(3)).to(device)
    want = torch.stack([plain(doubled(m), im.double().cpu(), SMALL, m.amplitude) for im in x])
    near(m(x), want, FORWARD, "embeddings")
    near(m.forward_packed(list(x)), want, FORWARD, "packed")


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    m = model_of(device)
    with pytest.raises(ValueError):
        m(torch.zeros(1, 3, 10, 12, device=device))
    with pytest.raises(ValueError):
        m.forward_packed([])
    with pytest.raises(ValueError):
        m.forward_packed([torch.zeros(3, 40, 40, device=device)], row_length=100)
    with pytest.raises(ValueError):
        RotaryViTB16(dim=30, heads=3)


def test_by_name():
    net = build_embedding_model("vit-rotary")
    assert isinstance(net.backbone, RotaryViTB16) and net.embed_dim == 768 and len(net.backbone.blocks) == 12


def trainer_of(device, graph, solver, **more):
    torch.manual_seed(0)
    net = EmbeddingNet(RotaryViTB16(**{**SMALL, "dim": 64, "heads": 2}))
    t = Trainer(net, NPairMultiClassLoss(NPairLossConfig()), solver, [], device=torch.device(device), hip_graph=graph, log_fn=lambda s: None, **more)
    t.graph_warmup = 2
    return t


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [8, 32])
def test_trainer_steps_and_goes_on(device, bits, tmp_path):
    """Steps by AdamW, a snapshot, and the same steps from it."""
    solver = SolverConfig(type="AdamW", base_lr=1e-3, momentum=0.9, weight_decay=0.01, state_bits=bits, max_iter=10)
    t = trainer_of(device, False, solver)
    assert isinstance(t.optimizer, AdamW)
    g = torch.Generator().manual_seed(5)
    batches = [(torch.randn(8, 3, 16, 16, generator=g), torch.arange(4).repeat(2)) for _ in range(4)]
    for x, y in batches[:2]:
        assert math.isfinite(float(t.train_step(x, y)["loss"]))
    path = t.snapshot(str(tmp_path / "s_"))
    for x, y in batches[2:]:
        t.train_step(x, y)
    other = trainer_of(device, False, solver)
    other.restore(path)
    for x, y in batches[2:]:
        other.train_step(x, y)
    for (n, a), b in zip(t.model.named_parameters(), other.model.parameters()):
        # equal inputs, states and random bits; a library's products may sum in another order: some U of a step's magnitudes
        assert float((a - b).detach().abs().max()) <= 1e-5, n
    assert int(next(iter(other.optimizer.state.values()))["step"]) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("pure", [False, True])
def test_trainer_graph(pure):
    """A captured step of norm, rotary, attention, loss and AdamW, replayed: as many steps
    as iterations, and the losses of the eager trainer."""
    solver = SolverConfig(type="AdamW", base_lr=1e-3, momentum=0.9, weight_decay=0.01, max_iter=10)
    g = torch.Generator().manual_seed(6)
    batches = [(torch.randn(8, 3, 16, 16, generator=g), torch.arange(4).repeat(2)) for _ in range(7)]
    eager, graph = (trainer_of("cuda", flag, solver, pure_bf16=pure) for flag in (False, True))
    for x, y in batches:
        a = float(eager.train_step(x, y)["loss"])
        b = float(graph._graph_step(x, y)["loss"])
        torch.cuda.synchronize()
        if graph.iter != graph.graph_warmup + 1:  # that iteration captured: its loss is a replay's first
            assert math.isfinite(b) and abs(a - b) <= (0.05 if pure else 1e-3) * (1 + abs(a))
        (torch.randn(256, 256, device="cuda") @ torch.randn(256, 256, device="cuda")).sum().item()
    assert graph._graph_state is not None
    steps = {int(s["step"]) for s in graph.optimizer.state.values()}
    assert steps == {len(batches)}


@pytest.mark.gpu
def test_bf16_autocast():
    """Under autocast the stream is bf16, the weights fp32: a row of packed images against
    the fp32 model, to bf16's rounding through two blocks (30 roundings of 2^-8, random signs)."""
    m, images = model_of("cuda"), images_of("cuda")
    want = m.forward_packed(images)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = m.forward_packed(images)
    assert got.dtype == torch.bfloat16
    near(got, want.detach().double().cpu(), 30 * 2.0 ** -8, "autocast")
    got.float().square().mean().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() and p.grad.dtype == torch.float32 for p in m.parameters())


@pytest.mark.parametrize("device", DEVICES)
def test_training_after_inference_mode(device):
    """What a model keeps of its first pass, in inference mode, serves a training pass."""
    m, other = model_of(device), model_of(device)
    x = torch.randn(2, 3, 8, 12, generator=torch.Generator().manual_seed(4)).to(device)
    with torch.inference_mode():
        first = m(x).clone()
    out = m(x)
    assert torch.equal(out, first)
    out.sum().backward()
    other(x).sum().backward()
    for (n, p), q in zip(m.named_parameters(), other.named_parameters()):
        near(p.grad, q[1].grad.double().cpu(), BACKWARD, n)
