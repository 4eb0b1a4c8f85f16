"""Calls of the token operators that have to be refused, or that must not lose anything: each of these once gave a wrong
result, or grew, in silence."""
import copy

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

from reid_gan_amd import attention, optim, rinet

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
GRAPHS = []            # captured graphs stay until the process ends
SECTIONS = (8, 12, 12)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(seed, *shape, to=F32):
    return torch.randn(*shape, generator=gen(seed), device=DEV).to(to)


class Sub(torch.Tensor):
    """A subclass keeps a call from going straight to the kernels: the checks in Python see it."""


def calls():
    """name, function of its tensors, the tensors"""
    x, w, b = normal(1, 5, 64), normal(2, 64), normal(3, 64)
    r, pos, freqs = normal(4, 1, 3, 2, 64), normal(5, 1, 3, 3), attention.rotary_frequencies(SECTIONS)
    q, k, v = normal(6, 1, 3, 2, 64, to=BF16), normal(7, 1, 9, 2, 64, to=BF16), normal(8, 1, 9, 2, 64, to=BF16)
    return {"layer_norm": (attention.layer_norm, (x, w, b)),
            "rotary": (lambda t, p, f: attention.rotary(t, p, f, SECTIONS), (r, pos, freqs)),
            "cross_attention": (attention.cross_attention, (q, k, v))}


# --------------------------------------------------------------------------- AdamW: the group's parameters
def ones(n):
    p = torch.nn.Parameter(torch.ones(n, device=DEV))
    p.grad = torch.ones(n, device=DEV)
    return p


def test_adamw_refuses_parameters_that_were_replaced():
    a, b, new = ones(300), ones(7), ones(300)
    opt = optim.AdamW([a, b])
    opt.step()
    before = [t.detach().clone() for t in (a, b, new)]
    for params in ([new, b], [a, new], [b, new]):
        opt.param_groups[0]["params"] = params
        with pytest.raises(RuntimeError, match="add_param_group"):
            opt.step()
        with pytest.raises(RuntimeError, match="add_param_group"):
            opt.flat_state()
    opt.param_groups[0]["params"] = [a, b]
    opt.param_groups[0]["params"][0] = new                                  # in the list itself
    with pytest.raises(RuntimeError, match="add_param_group"):
        opt.step()
    assert all(torch.equal(t, o) for t, o in zip((a, b, new), before))
    opt.param_groups[0]["params"] = [b, a]                                  # the same ones in another order
    opt.step()
    assert not torch.equal(a, before[0]) and not torch.equal(b, before[1])
    assert int(opt.state[a]["step"]) == int(opt.state[b]["step"]) == 2


def test_adamw_refuses_a_parameter_that_was_transposed_where_it_lies():
    p = torch.nn.Parameter(normal(20, 16, 16))
    opt = optim.AdamW([p])
    p.grad = normal(21, 16, 16)
    opt.step()
    p.data = p.data.t()
    p.grad = normal(21, 16, 16)
    before = p.detach().clone()
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    assert torch.equal(p, before)
    p.data = p.data.t()
    opt.step()


def test_adamw_parameters_that_move_at_every_step_cost_no_memory():
    ps = [ones(3) for _ in range(900)]                                      # (a job table of 43 KB)
    opt = optim.AdamW(ps)
    homes = [[p.data for p in ps], [p.data.clone() for p in ps]]
    for i in range(40):
        for p, t in zip(ps, homes[i & 1]):
            p.data = t
        opt.step()
        if i == 3:
            base = torch.cuda.memory_allocated()
    assert torch.cuda.memory_allocated() <= base + 8192


def test_adamw_a_captured_step_keeps_its_table_when_parameters_move():
    """Parameters move away after a capture and come back: the replays go on where the capture found them."""
    a, b = ones(700), ones(700)
    one, two = optim.AdamW([a], lr=1e-2), optim.AdamW([b], lr=1e-2)
    one.step(), two.step()
    graph = torch.cuda.CUDAGraph()
    GRAPHS.append(graph)
    with torch.cuda.graph(graph):
        one.step()
    home = a.data
    for i in range(3):
        a.data = home.clone()
        for _ in range(3):                                                  # (and tables are made for other places)
            a.data = a.data.clone()
            one.step(), two.step()
        home.copy_(a.data)
        a.data = home
        graph.replay(), two.step()
        torch.cuda.synchronize()
        assert torch.equal(a, b), i
        one.step(), two.step()
        assert torch.equal(a, b), i


# --------------------------------------------------------------------------- AdamW: state dicts
def test_adamw_load_state_dict_runs_its_hooks():
    a, b = ones(5), ones(5)
    one, two = optim.AdamW([a], lr=1e-3), optim.AdamW([b], lr=1e-3)
    one.step()
    seen = []

    def before(opt, state):
        seen.append("before")
        state = copy.deepcopy(state)
        state["param_groups"][0]["lr"] = 0.5
        return state
    two.register_load_state_dict_pre_hook(before)
    two.register_load_state_dict_pre_hook(lambda opt, state: seen.append("second") or None)
    two.register_load_state_dict_post_hook(lambda opt: seen.append(("after", opt is two, int(opt.state[b]["step"]))))
    saved = one.state_dict()
    two.load_state_dict(saved)
    assert seen == ["before", "second", ("after", True, 1)]
    assert two.param_groups[0]["lr"] == 0.5 and saved["param_groups"][0]["lr"] == 1e-3
    handle = two.register_load_state_dict_pre_hook(lambda opt, state: state.update(mark=1))
    two.load_state_dict(saved)
    assert "mark" not in saved                                              # (a hook gets a dict of its own)
    handle.remove()
    assert torch.equal(two.state[b]["exp_avg"], one.state[a]["exp_avg"])


def test_adamw_group_entries_travel():
    """What a schedule or a caller keeps in the groups comes back with them, as with every torch optimizer."""
    a, b = ones(5), ones(5)
    one = optim.AdamW([{"params": [a], "name": "decoder"}])
    sched = torch.optim.lr_scheduler.OneCycleLR(one, max_lr=0.1, total_steps=50)
    for _ in range(7):
        one.step(), sched.step()
    saved = copy.deepcopy(one.state_dict())
    two = optim.AdamW([{"params": [b], "name": "?"}])
    torch.optim.lr_scheduler.OneCycleLR(two, max_lr=9.0, total_steps=50)
    two.load_state_dict(saved)
    mine = two.param_groups[0]
    assert mine["params"][0] is b
    assert {k: v for k, v in mine.items() if k != "params"} == {k: v for k, v in saved["param_groups"][0].items() if k != "params"}
    assert mine["name"] == "decoder" and mine["max_lr"] == 0.1
    saved["param_groups"][0]["name"] = "other"                              # (nothing is shared with what was loaded)
    assert mine["name"] == "decoder"


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_a_refused_state_changes_nothing(bits):
    a, b = ones(300), ones(40)
    opt = optim.AdamW([{"params": [a]}, {"params": [b], "lr": 0.25}], state_bits=bits)
    opt.step()
    good = copy.deepcopy(opt.state_dict())
    a.grad.mul_(3), opt.step()
    held = copy.deepcopy(opt.state_dict())
    shape, names, kind, value, group = (copy.deepcopy(good) for _ in range(5))
    shape["state"][1]["exp_avg"] = shape["state"][1]["exp_avg"][:3]
    names["state"][1]["max_exp_avg_sq"] = names["state"][1]["exp_avg"]
    kind["state"][1]["exp_avg"] = torch.zeros(40, device=DEV, dtype=F32 if bits == 8 else torch.float8_e4m3fn)
    value["param_groups"][1]["lr"] = -1.0
    group["param_groups"][1]["maximize"] = True
    for i, bad in enumerate((shape, names, kind, value, group)):
        bad["param_groups"][0]["lr"] = 77.0
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
        now = opt.state_dict()
        assert now["param_groups"] == held["param_groups"], i
        for s in (0, 1):
            for name, t in held["state"][s].items():
                assert torch.equal(now["state"][s][name].float(), t.float()), (i, s, name)


def test_adamw_on_the_generators_own_parameters():
    """The drop-in generator's parameters, as they are (222 tensors), against the formula in 64 bits: each step is off by
    at most 3 e of p and 12 e of its update, which lr bounds while the moments are those of equal gradients."""
    net = rinet.RIGAN().cuda()
    ps = list(net.parameters())
    start = [p.detach().double() for p in ps]
    opt = optim.AdamW(ps, lr=1e-3, weight_decay=0.1)
    grads = [normal(100 + i, *p.shape) for i, p in enumerate(ps)]
    for p, g in zip(ps, grads):
        p.grad = g
    for _ in range(2):
        opt.step()
    e = 2.0 ** -24
    for p, s, g in zip(ps, start, grads):
        g, want = g.double(), s
        for t in (1, 2):                                                    # m / (1 - b1^t) = g, v / (1 - b2^t) = g^2
            want = want * (1 - 1e-4) - 1e-3 * g / (g.abs() + 1e-8)
        assert bool(((p.detach().double() - want).abs() <= 2 * (4 * e * (s.abs() + 1e-3) + 12 * e * 1e-3)).all())


# --------------------------------------------------------------------------- derivatives and traces that would be lost
@pytest.mark.parametrize("name", ["layer_norm", "rotary", "cross_attention"])
@pytest.mark.parametrize("plain", [True, False])
def test_forward_mode_derivatives_are_refused(name, plain):
    call, args = calls()[name]
    wrap = (lambda t: t) if plain else (lambda t: t.as_subclass(Sub))
    with forward_ad.dual_level():
        for i, t in enumerate(args):
            dual = [forward_ad.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate(args)]
            for grad in (False, True):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    call(*map(wrap, dual))
        call(*map(wrap, args))                                              # (tensors without a tangent are none of its business)
        with forward_ad._set_fwd_grad_enabled(False):
            call(*map(wrap, dual))
        leaf = args[0].detach().clone().requires_grad_()                    # and the incoming gradient of a backward pass
        out = call(*map(wrap, (leaf, *args[1:])))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, leaf, forward_ad.make_dual(torch.ones_like(args[0]), torch.ones_like(args[0])))


@pytest.mark.parametrize("name", ["layer_norm", "rotary", "cross_attention"])
@pytest.mark.parametrize("plain", [True, False])
def test_traces_are_refused(name, plain):
    """A trace would hold the allocation of the result and not the kernel that writes it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    call, args = calls()[name]
    wrap = (lambda t: t) if plain else (lambda t: t.as_subclass(Sub))
    function = lambda *ts: call(*map(wrap, ts)).as_subclass(torch.Tensor)
    want = function(*args)
    for grad in (False, True):
        leaves = [a.detach().requires_grad_(grad and i == 0) for i, a in enumerate(args)]
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(function, tuple(leaves), check_trace=False)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(function)(*leaves)
    assert torch.equal(function(*args), want)
    if name == "layer_norm":
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(attention.LayerNorm(64).to(DEV), args[0], check_trace=False)


@pytest.mark.parametrize("plain", [True, False])
def test_rotary_refuses_gradients_of_its_tables(plain):
    call, (x, pos, freqs) = calls()["rotary"]
    wrap = (lambda t: t) if plain else (lambda t: t.as_subclass(Sub))
    for leaf in (pos, freqs):
        leaf.requires_grad_()
        for first in (x, x.clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="positions and freqs have no gradient"):
                call(wrap(first), pos, freqs)
        with torch.no_grad():
            got = call(wrap(x), pos, freqs)
        leaf.requires_grad_(False)
        assert torch.equal(got.as_subclass(torch.Tensor), call(x, pos, freqs))


def test_function_transforms_are_refused():
    """torch.func's wrappers have no memory of their own to launch on."""
    call, args = calls()["layer_norm"]
    x = args[0]
    for wrong in (lambda: torch.func.grad(lambda t: call(t).sum())(x), lambda: torch.func.vmap(call)(x[None]),
                  lambda: torch.func.jvp(call, (x,), (torch.ones_like(x),)), lambda: torch.func.vjp(call, x)):
        with pytest.raises(RuntimeError):
            wrong()


def test_cross_attention_small_scales_keep_hidden_keys_out():
    """A scale close to nothing: the result is the mean of the values that count."""
    _, (q, k, v) = calls()["cross_attention"]
    mask = torch.tensor([[True, False] * 4 + [True]], device=DEV)
    want = v[:, ::2].double().mean(1, keepdim=True)
    for rows in (3, 90):
        got = attention.cross_attention(q.repeat(1, rows // 3, 1, 1), k, v, key_mask=mask, scale=2e-37)
        assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -8 * v.double().abs().mean(1, keepdim=True)).all())
    for scale in (1e-46, 1e30):
        with pytest.raises(ValueError, match="scale"):
            attention.cross_attention(q, k, v, key_mask=mask, scale=scale)


# --------------------------------------------------------------------------- functions on buffers
@pytest.mark.parametrize("name", ["layer_norm_fwd", "layer_norm_bwd", "rotary", "xattn_fwd", "xattn_bwd"])
def test_functions_on_buffers_refuse_what_the_kernels_could_not_read(name):
    """Refused before any launch: one tensor in host memory, scratch and statistics of another type."""
    from test_tokens_guards_cpu import buffer_calls
    call, tensors = buffer_calls(DEV)[name]
    call(**tensors)
    for one in tensors:
        with pytest.raises(AssertionError):
            call(**{**tensors, one: tensors[one].cpu()})
    for one in set(tensors) & {"stats", "scratch", "lse"}:
        with pytest.raises(AssertionError):
            call(**{**tensors, one: tensors[one].to(BF16)})
    torch.cuda.synchronize()


@pytest.mark.parametrize("plain", [True, False])
def test_cross_attention_gradients_where_queries_lie_far_apart(plain):
    """Views of q and of the incoming gradient that span over 2^31 bytes: the kernels of the gradients get copies."""
    wrap = (lambda t: t) if plain else (lambda t: t.as_subclass(Sub))
    big = torch.empty(600 << 22, dtype=BF16, device=DEV)
    q, d = (big.as_strided((1, 600, 4, 64), (0, 1 << 22, 64, 1), at) for at in (0, 4096))
    q.copy_(normal(30, 1, 600, 4, 64)), d.copy_(normal(31, 1, 600, 4, 64))
    k, v = normal(32, 1, 77, 2, 64, to=BF16), normal(33, 1, 77, 2, 64, to=BF16)
    results = []
    for a, g in ((q, d), (q, d.contiguous()), (q.contiguous(), d), (q.contiguous(), d.contiguous())):
        leaves = [t.detach().requires_grad_() for t in (a, k, v)]
        out = attention.cross_attention(*map(wrap, leaves))
        results.append([out.detach().as_subclass(torch.Tensor), *torch.autograd.grad(out, leaves, g)])
    for got in results[:3]:
        assert all(torch.equal(a, b.as_subclass(torch.Tensor)) for a, b in zip(results[3], got))


def test_adamw_a_refused_step_changes_nothing():
    """A second group's parameter, gradient or rate that cannot be taken: the first group is not stepped either."""
    def moved(p, q):
        q.data = q.data.new_zeros(9)

    def wrong(p, q):
        q.grad = torch.sparse_coo_tensor([[0]], [1.0], (7,), device=DEV)

    def replaced(p, q):
        opt.param_groups[1]["params"] = [ones(7)]

    def negative(p, q):
        opt.param_groups[1]["lr"] = -1.0
    for break_it in (moved, wrong, replaced, negative):
        p, q = ones(300), ones(7)
        opt = optim.AdamW([{"params": [p]}, {"params": [q]}])
        opt.step()
        before, count = p.detach().clone(), int(opt.state[p]["step"])
        break_it(p, q)
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            opt.step()
        assert torch.equal(p, before) and int(opt.state[p]["step"]) == count == 1
