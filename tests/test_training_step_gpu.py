"""The operators around the layer as they are used together: embedding, residual block of norm and MoE layer, norm, linear cross
entropy with the layer's losses, AdamW. Every operator is held to its own definition in 64 bits at the tensors that it sees."""

import pytest
import torch

import test_adamw_gpu as adamw
import test_layer_norm_gpu as norm
import test_linear_cross_entropy_gpu as entropy

VOCAB, WIDTH, EXPERTS = 1003, 128, 4


class Model(torch.nn.Module):
    def __init__(self, layers=2):
        from flashfusedmoe_b200 import LayerNorm, MoELayer
        super().__init__()
        torch.manual_seed(5)
        self.embed = torch.nn.Embedding(VOCAB, WIDTH)
        self.blocks = torch.nn.ModuleList(MoELayer(WIDTH, 256, EXPERTS, top_k=2, num_shared_experts=1, aux_loss_coeff=0.01,
                                                   z_loss_coeff=0.001, pre_norm=True) for _ in range(layers))
        self.norm = LayerNorm(WIDTH)
        self.head = torch.nn.Parameter(torch.randn(VOCAB, WIDTH) * WIDTH ** -0.5)
        self.seen = {}

    def forward(self, tokens, target, **options):
        from flashfusedmoe_b200 import linear_cross_entropy
        x, extra = self.embed(tokens), 0.0
        for block in self.blocks:
            y, losses = block(x)
            x = x + y
            extra = extra + losses["aux_loss"] + losses["z_loss"]
        hidden = self.norm(x)
        self.seen = {"x": x, "hidden": hidden}
        return linear_cross_entropy(hidden, self.head, target, z_loss_coeff=1e-4, **options), extra


def batch(seed, rows=3, length=41):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = torch.randint(0, VOCAB, (rows, length), device="cuda", generator=g)
    target = tokens.roll(-1, dims=1)
    target[:, -1] = -100
    target[0, 20:] = -100   # a padded sequence
    return tokens, target


def make(state_bits, master=True):
    from flashfusedmoe_b200 import AdamW
    model = Model().cuda().bfloat16()
    dense = [p for p in model.parameters() if p.dim() < 2]
    wide = [p for p in model.parameters() if p.dim() >= 2]
    opt = AdamW([{"params": wide, "weight_decay": 0.1}, {"params": dense, "weight_decay": 0.0}], lr=3e-3, betas=(0.9, 0.95),
                state_bits=state_bits, master_weights=master)
    return model, opt


@pytest.mark.gpu
@pytest.mark.parametrize("state_bits", [32, 8])
def test_every_operator_of_a_step(state_bits):
    from flashfusedmoe_b200 import ops
    model, opt = make(state_bits)
    for k in range(3):
        tokens, target = batch(k)
        opt.zero_grad()
        loss, extra = model(tokens, target)
        x, hidden = model.seen["x"], model.seen["hidden"]
        x.retain_grad()
        hidden.retain_grad()
        (loss + extra).backward()
        ops.check_status()
        # the loss at the hidden rows that it saw
        flat = hidden.detach().view(-1, WIDTH)
        out, bound = entropy.reference(flat, model.head.detach(), target.view(-1), 1e-4)
        entropy.check(loss.detach(), out, bound, "loss")
        entropy.check(hidden.grad.view(-1, WIDTH), out, bound, "dh")
        entropy.check(model.head.grad, out, bound, "dw")
        # the last norm at the rows and gradients that it saw
        rows = x.detach().view(-1, WIDTH)
        out, bound = norm.reference(rows, model.norm.weight.detach(), model.norm.bias.detach(), model.norm.eps, hidden.grad.view(-1, WIDTH))
        norm.check(flat, out, bound, "y")
        norm.check(model.norm.weight.grad, out, bound, "dw")
        norm.check(model.norm.bias.grad, out, bound, "db")
        # the update at the gradients that it saw
        for group in opt.param_groups:
            for p in group["params"]:
                opt._state_of(p, group)
            t = adamw.Tensors([], torch.float32, 32)
            states = [opt.state[p] for p in group["params"]]
            eight = ["exp_avg_scale" in s for s in states]
            assert any(eight) == (state_bits == 8 and group["weight_decay"] > 0)
            before, found = [s["step"].item() for s in states], []
            for p, s in zip(group["params"], states):
                t.params, t.grads, t.steps, t.masters = [p.detach().clone()], [p.grad], [s["step"]], [s["master"]]
                t.m, t.v = [s["exp_avg"]], [s["exp_avg_sq"]]
                t.m_scale, t.v_scale = ([s["exp_avg_scale"]], [s["exp_avg_sq_scale"]]) if "exp_avg_scale" in s else (None, None)
                found += t.exact(lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"])
            group["checked"] = (before, found)
        opt.step()
        for group in opt.param_groups:
            before, found = group.pop("checked")
            for p, step, (m, v, exact, m_off, v_off, p_off) in zip(group["params"], before, found):
                s = opt.state[p]
                assert s["step"].item() == step + 1
                assert ((s["master"].double() - exact).abs() <= p_off).all()
                assert torch.equal(p.detach(), s["master"].bfloat16())
                if "exp_avg_scale" not in s:
                    assert ((s["exp_avg"].double() - m).abs() <= m_off).all() and ((s["exp_avg_sq"].double() - v).abs() <= v_off).all()


@pytest.mark.gpu
@pytest.mark.parametrize("state_bits,master", [(32, True), (8, True), (8, False)])
def test_a_captured_step_replays_to_the_eager_bits(state_bits, master):
    def step(model, opt, tokens, target):
        loss, extra = model(tokens, target)
        (loss + extra).backward()
        opt.step()
        return loss.detach()

    model, opt = make(state_bits, master)
    twin, eager = make(state_bits, master)
    tokens, target = batch(100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for k in range(2):   # states and workspaces come into being
            opt.zero_grad(set_to_none=True)
            step(model, opt, tokens, target)
    torch.cuda.current_stream().wait_stream(side)
    opt.zero_grad(set_to_none=True)
    model.seen = {}   # no eager graph of these leaves is left
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss = step(model, opt, tokens, target)
    model.seen = {}
    for k in range(2):
        eager.zero_grad(set_to_none=True)
        step(twin, eager, *batch(100))
    for k in range(4):
        a, b = batch(200 + k)
        tokens.copy_(a)
        target.copy_(b)
        graph.replay()
        eager.zero_grad(set_to_none=True)
        other = step(twin, eager, a, b)
        torch.cuda.synchronize()
        assert torch.equal(loss, other)
    for p, q in zip(model.parameters(), twin.parameters()):
        assert torch.equal(p, q)
        for name, value in opt.state[p].items():
            assert torch.equal(value.view(torch.uint8) if value.dim() else value, eager.state[q][name].view(torch.uint8) if value.dim() else eager.state[q][name]), name


@pytest.mark.gpu
def test_scoring_after_training():
    """Log-probabilities of single tokens and of the whole batch agree with the training loss's rows."""
    model, opt = make(32)
    tokens, target = batch(7)
    model(tokens, target)[0].backward()
    opt.step()
    with torch.no_grad():
        nll, _ = model(tokens, target, reduction="none")
        mean, _ = model(tokens, target)
        hidden = model.seen["hidden"]
        out, bound = entropy.reference(hidden.reshape(-1, WIDTH), model.head, target.reshape(-1), 1e-4)
        entropy.check(nll.reshape(-1), out, bound, "nll")
        entropy.check(mean, out, bound, "loss")
        from flashfusedmoe_b200 import linear_cross_entropy
        one = linear_cross_entropy(hidden[1, 5:6], model.head, target[1, 5:6], reduction="none", z_loss_coeff=1e-4)
        row = tokens.shape[1] + 5
        entropy.check(one, {"nll": out["nll"][row:row + 1]}, {"nll": bound["nll"][row:row + 1]}, "nll")


@pytest.mark.gpu
def test_a_compiled_model_breaks_its_graph_around_them():
    model, _ = make(32)
    tokens, target = batch(11)

    def run(m):
        model.zero_grad(set_to_none=True)
        loss, extra = m(tokens, target)
        (loss + extra).backward()
        return loss.detach(), [p.grad.clone() for p in model.parameters()]

    loss, grads = run(model)
    other, others = run(torch.compile(model, backend="aot_eager"))
    assert torch.equal(loss, other) and all(torch.equal(a, b) for a, b in zip(grads, others))


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [True, False])
def test_recomputed_and_moved_operands_give_the_same_bits(reentrant):
    """Checkpointing runs the forward calls again in the backward pass (and leaves them at the last saved tensor); hooks that move
    saved tensors to the host hand back others."""
    from torch.utils.checkpoint import checkpoint
    from flashfusedmoe_b200 import layer_norm, linear_cross_entropy
    torch.manual_seed(3)
    x = torch.randn(40, WIDTH, device="cuda").bfloat16().requires_grad_()
    w, b = (torch.randn(WIDTH, device="cuda", requires_grad=True) for _ in range(2))
    head = torch.randn(VOCAB, WIDTH, device="cuda").bfloat16().requires_grad_()
    target = torch.randint(0, VOCAB, (40,), device="cuda")

    def normed(x):
        return layer_norm(x, w, b)

    def scored(x):
        return linear_cross_entropy(normed(x), head, target)

    for call, leaves in ((normed, (x, w, b)), (scored, (x, w, b, head))):
        want = torch.autograd.grad(call(x).float().sum(), leaves)
        x.grad = w.grad = b.grad = head.grad = None
        checkpoint(call, x, use_reentrant=reentrant).float().sum().backward()
        assert all(torch.equal(leaf.grad, g) for leaf, g in zip(leaves, want))
        with torch.autograd.graph.save_on_cpu():
            out = call(x)
        assert all(torch.equal(p, g) for p, g in zip(torch.autograd.grad(out.float().sum(), leaves), want))


@pytest.mark.gpu
def test_steps_of_several_threads_at_once(monkeypatch):
    """Each thread on a stream of its own, against the same steps one after the other; the first calls of all."""
    import threading
    from flashfusedmoe_b200 import adamw_step, layer_norm, linear_cross_entropy, ops
    monkeypatch.setattr(ops, "_status", {})
    monkeypatch.setattr(ops, "_reported", {})

    def steps(seed, found):
        g = torch.Generator(device="cuda").manual_seed(seed)
        with torch.cuda.stream(torch.cuda.Stream()):
            x = torch.randn(700, WIDTH, device="cuda", generator=g).bfloat16().requires_grad_()
            w = torch.randn(WIDTH, device="cuda", generator=g).requires_grad_()
            head = torch.randn(VOCAB, WIDTH, device="cuda", generator=g).bfloat16().requires_grad_()
            target = torch.randint(0, VOCAB, (700,), device="cuda", generator=g)
            moments = [torch.zeros(VOCAB, WIDTH, device="cuda") for _ in range(2)]
            count = torch.zeros((), dtype=torch.int32, device="cuda")
            for _ in range(40):
                x.grad = w.grad = head.grad = None
                linear_cross_entropy(layer_norm(x, w), head, target).backward()
                adamw_step([head.detach()], [head.grad], moments[:1], moments[1:], [count], lr=1e-3)
            torch.cuda.current_stream().synchronize()
            found[seed] = [t.clone() for t in (x.grad, w.grad, head.detach(), *moments, count)]
            torch.cuda.current_stream().synchronize()

    at_once, alone = {}, {}
    threads = [threading.Thread(target=steps, args=(seed, at_once)) for seed in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for seed in range(3):
        steps(seed, alone)
    assert len(at_once) == 3
    for seed in range(3):
        assert all(torch.equal(a, b) for a, b in zip(at_once[seed], alone[seed]))
