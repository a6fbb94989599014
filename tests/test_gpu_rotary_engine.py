"""LinearEngine.full_attention with a rotary plan and with caches that have
scales of blocks, on the GPU: against its parts, in serving steps, captured."""
import math

import pytest
import torch

import paged_oracle as PO
from test_gpu_paged import _Server

pytestmark = pytest.mark.gpu

YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32}


class Server(_Server):
    """A _Server whose layer rotates by a plan (or by the config's parameters) over a cache of either kind."""

    def __init__(self, F, dev, requests, kind, plan=True, neighbours=False, block=16):
        super().__init__(F, dev, requests, kind != "bf16")
        self.kind = kind
        if kind == "blocks":
            shape = (self.caches[0].size(0), self.PAGE // block, self.HK)
            self.scales = {n: torch.full(shape, 255, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu) for n in ("k_scale", "v_scale")}
        if plan:
            self.ROPE = F.rotary_plan(16, 10000.0, YARN, neighbours=neighbours, sections=_Server.ROPE["mrope_section"], device=dev)

    def bits(self):
        return [c.view(torch.uint8 if c.element_size() == 1 else torch.int16) for c in (*self.caches, *self.scales.values()) if c.dtype != torch.float32]


@pytest.mark.parametrize("plan", [True, False])
@pytest.mark.parametrize("kind", ["bf16", "heads", "blocks"])
def test_full_attention_is_its_parts(fp8lin, gpu, kind, plan):
    """Prompts, then drafted tokens with rows of no request: the operators one by one, on copies of the projection's parts."""
    a, b = [Server(fp8lin, gpu, 3, kind, plan) for _ in range(2)]
    H, HK, D, P = a.H, a.HK, a.D, a.P
    g = torch.Generator().manual_seed(3)
    for step, (counts, extra) in enumerate((([40, 17, 5], 0), ([3, 1, 4], 6), ([0, 1, 30], 2))):
        tokens = torch.randint(0, a.V, (sum(counts) + extra,), generator=g).to(gpu)
        counts_t = torch.tensor(counts, dtype=torch.int32, device=gpu)
        lays = []
        for s in (a, b):
            lays.append(fp8lin.paged_layout(s.lengths, counts_t, s.table, s.free, tokens.numel(), s.PAGE, cursor=s.cursor, out=s.table))
            s.cursor.copy_(lays[-1].cursor)
        x = a.embed[tokens]
        positions = None if step else torch.stack([lays[0].positions, lays[0].positions // 2, lays[0].positions % 9])
        y = a.eng.full_attention(x, P, lays[0], *a.caches, *a.norms, H, HK, D, a.ROPE, 1e-6, max_count=max(counts), positions=positions, **a.scales)
        at = lays[1].positions if positions is None else positions
        t = tokens.numel()
        projected = b.eng.linear(x, P + ".qkv_gate")
        qg = projected[:, :2 * H * D].reshape(t, H, 2 * D)
        k, v = [projected[:, lo:lo + HK * D].reshape(t, HK, D).contiguous() for lo in (2 * H * D, (2 * H + HK) * D)]
        if plan:
            q = fp8lin.paged_rotate_append(qg[..., :D].contiguous(), k, v, at, lays[1].slots, *b.caches, b.ROPE, q_norm=b.norms[0], k_norm=b.norms[1],
                                           eps=1e-6, **b.scales)
        else:
            sections = b.ROPE["mrope_section"]
            q, k = fp8lin.qk_norm_rope(projected, *b.norms, at if at.dim() == 2 else at.expand(3, t), H, HK, D, 16, b.ROPE["rope_theta"],
                                       sections[1], sections[2], 1e-6)
            fp8lin.paged_append(k, v, lays[1].slots, *b.caches, **b.scales)
        core = fp8lin.paged_attention(q, *b.caches, lays[1].block_table, lays[1].offsets, lays[1].lengths, max_count=max(counts),
                                      gate=qg[..., D:].contiguous(), out=torch.zeros_like(q), **b.scales)
        want = b.eng.linear(core.view(t, H * D), P + ".o_proj")
        assert torch.equal(y.view(torch.int16), want.view(torch.int16)), step
        assert all(torch.equal(m, n) for m, n in zip(a.bits(), b.bits()))
        assert (y[sum(counts):] == 0).all()
        # a mistake in the positions would show
        assert not torch.equal(q[:, 0], q[:, 1])
        for s, lay in zip((a, b), lays):
            s.lengths.copy_(lay.lengths)


def test_plan_is_full_attentions_alone(fp8lin, gpu):
    s = Server(fp8lin, gpu, 1, "bf16")
    with pytest.raises(fp8lin.Fp8linError):
        s.eng.full_attention_inputs(s.embed[:3], s.P, torch.zeros(3, 3, dtype=torch.int64, device=gpu), *s.norms, s.H, s.HK, s.D, s.ROPE, 1e-6)


def test_unscaled_plan_is_near_the_reference_form(fp8lin, gpu):
    """The same layer by the config's parameters and by an unscaled plan: apart by the reference's BF16 roundings of the cosines and
    sines, of the norms, of the products and sums (6 half steps of the pair's values), through the layer."""
    a, b = Server(fp8lin, gpu, 2, "bf16", plan=False), Server(fp8lin, gpu, 2, "bf16")
    b.ROPE = fp8lin.rotary_plan(16, 10000.0, a.ROPE, sections=a.ROPE["mrope_section"], device=gpu)
    tokens = torch.randint(0, a.V, (50,), generator=torch.Generator().manual_seed(4)).to(gpu)
    counts = torch.tensor([30, 20], dtype=torch.int32, device=gpu)
    lay = [s.step(tokens, counts, 30)[1] for s in (a, b)]
    slots = lay[0].slots.cpu()
    assert torch.equal(slots, lay[1].slots.cpu())
    ka, kb = [s.caches[0].flatten(0, 1)[slots.to(gpu)].double().cpu() for s in (a, b)]
    # a pair's length is kept by the rotation, so its reach is at most sqrt(2) of that
    size = kb.abs()
    pair = (kb[..., :8] ** 2 + kb[..., 8:16] ** 2).sqrt() * 2 ** 0.5
    size[..., :8], size[..., 8:16] = pair, pair
    assert float(((ka - kb).abs() - 7 * PO.BF16_HALF * size * 1.05).max()) <= 0
    assert torch.equal(a.caches[1].flatten(0, 1)[slots.to(gpu)], b.caches[1].flatten(0, 1)[slots.to(gpu)])


@pytest.mark.parametrize("kind", ["bf16", "blocks"])
def test_serving_step_captured(fp8lin, gpu, kind):
    """Decode steps with a plan as one HIP graph: layout, projection, rotated append, attention, head and verification; every replay
    equals the eager step from the same state."""
    state = []
    for form in ("eager", "graph"):
        s = Server(fp8lin, gpu, 3, kind, neighbours=True)
        ints = dict(dtype=torch.int32, device=gpu)
        g = torch.Generator().manual_seed(4)
        _, lay = s.step(torch.randint(0, s.V, (60,), generator=g).to(gpu), torch.tensor([33, 16, 11], **ints), 33)
        s.lengths.copy_(lay.lengths)
        tokens = torch.randint(0, s.V, (9,), generator=g).to(gpu)
        counts, u = torch.full((3,), 3, **ints), torch.empty(9, device=gpu)
        heads = torch.arange(0, 9, 3, device=gpu)

        def one():
            y, lay = s.step(tokens, counts, 3)
            logits = s.eng.linear(y, "lm_head")
            accepted, out = fp8lin.verify_drafts(logits, tokens, u, lay.offsets)
            s.lengths.add_(1 + accepted)
            tokens[heads] = out[heads + accepted]
            return logits, accepted, out

        held = (s.lengths, s.cursor, s.table, tokens, *s.bits())
        saved = [x.clone() for x in held]
        if form == "graph":
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                u.fill_(0.5)
                one()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                res = one()
            for x, y in zip(held, saved):
                x.copy_(y)
        got = []
        for i in range(8):
            u.copy_(torch.rand(9, generator=torch.Generator().manual_seed(i)))
            torch.cuda.synchronize()
            if form == "graph":
                graph.replay()
            else:
                res = one()
            torch.cuda.synchronize()
            got += [x.clone().cpu() for x in (*res, s.lengths, s.cursor, s.table)]
        assert math.isfinite(float(res[0].float().sum()))
        state.append(got)
    for x, y in zip(*state):
        assert torch.equal(x, y)
