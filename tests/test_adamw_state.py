"""What AdamW keeps: master copies beside parameters that others write to, roots of the second moment for any eps, and states that come back from a dict."""
import pytest
import torch

from test_adamw import _bits, _codes


def _trained(dtype, bits, steps=3, lr=1e-2):
    import gelib_b200 as G
    gen = torch.Generator().manual_seed(5)
    p = torch.nn.Parameter(torch.randn(700, generator=gen).to(dtype).cuda())
    grads = [torch.randn(700, generator=gen).to(dtype).cuda() for _ in range(8)]
    opt = G.AdamW([p], lr=lr, weight_decay=0.0, state_bits=bits)
    for g in grads[:steps]:
        p.grad = g
        opt.step()
    return p, opt, grads[steps:]


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("how", ["data", "no_grad", "load_state_dict", "some"])
def test_what_is_written_to_a_parameter_stays(how, dtype, bits, native, monkeypatch):
    """A parameter that was written between two steps takes the next one from what it holds; a rate of zero leaves that as it is."""
    import gelib_b200 as G
    if not native:
        monkeypatch.setattr(G._lib, "_native", G._lib._Declines())
    p, opt, grads = _trained(dtype, bits)
    old = p.detach().clone()
    want = torch.linspace(-2, 2, 700, device="cuda").to(dtype)
    if how == "data":
        p.data.copy_(want)
    elif how == "no_grad":
        with torch.no_grad():
            p.copy_(want)
    elif how == "load_state_dict":
        holder = torch.nn.Module()
        holder.w = p
        holder.load_state_dict({"w": want})
    else:   # a clamp writes some elements only
        p.data.clamp_(-0.5, 0.5)
        want = old.clamp(-0.5, 0.5)
        assert 0 < int((want != old).sum()) < 700
    kept = opt.state[p].get("master", p.detach()).clone()
    opt.param_groups[0]["lr"] = 0.0
    p.grad = grads[0]
    opt.step()
    assert torch.equal(p.detach(), want)
    if "master" in opt.state[p]:   # an element that was not written keeps its copy's further digits
        same = want == old
        master = opt.state[p]["master"]
        assert torch.equal(master[same], kept[same]) and torch.equal(master[~same], want[~same].float())
    opt.param_groups[0]["lr"] = 1e-1
    p.grad = grads[1]
    opt.step()
    assert ((p.detach() - want).abs().float() < 0.5).all() and not torch.equal(p.detach(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_steps_below_a_parameters_last_place_add_up(dtype):
    p, opt, _ = _trained(dtype, 32, steps=0, lr=1e-6)
    first = p.detach().float()
    for _ in range(200):
        p.grad = torch.ones_like(p)
        opt.step()
    moved = first - opt.state[p]["master"]
    assert ((moved - 200e-6).abs() <= 200 * 16 * 2.0 ** -24 * (first.abs() + 1e-6)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("offset", [0, 1])
def test_refreshing_master_copies(offset, native, monkeypatch):
    """adamw_step takes the step from the master copies; where it is told to, first from what the parameters hold where that is not their rounding."""
    import gelib_b200 as G
    if not native:
        monkeypatch.setattr(G._lib, "_native", G._lib._Declines())
    gen = torch.Generator().manual_seed(2)
    for dtype in (torch.bfloat16, torch.float16):
        copy = torch.randn(999 + offset, generator=gen).cuda()[offset:]
        p = copy.to(dtype) if not offset else torch.cat([copy[:1], copy]).to(dtype)[1:]
        p[::7] = 3.0
        p[5], p[6] = float("nan"), -0.0
        copy[6] = 0.0
        for refresh in (False, True):
            q, master = torch.cat([p[:offset], p])[offset:], torch.cat([copy[:offset], copy])[offset:]
            m, v = (torch.zeros(999, device="cuda") for _ in range(2))
            G.adamw_step([q], [torch.zeros_like(q)], [m], [v], step=1, lr=0.0, master=[master], refresh_master=refresh)
            want = torch.where(p.view(torch.int16) == copy.to(dtype).view(torch.int16), copy, p.float()) if refresh else copy
            assert torch.equal(master.view(torch.int32)[torch.arange(999) != 5], want.view(torch.int32)[torch.arange(999) != 5])
            assert bool(master[5].isnan()) == refresh and torch.equal(q[7:], want[7:].to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("size,eps", [(1e-2, 1e-2), (1e-2, 1e2), (1e-9, 1e-8), (1e-13, 1e-8), (1e-13, 0.0), (1e12, 1e-8)])
def test_codes_of_the_root_whatever_eps_is(size, eps):
    """The root that is held does not depend on eps.  Rounded to nearest it has the codes of torch's root, all of 2^24 elements."""
    import gelib_b200 as G
    n, b1, b2, seed = 1 << 24, 0.9, 0.999, 31
    gen = torch.Generator(device="cuda").manual_seed(3)
    sizes = torch.exp(torch.randn(n // 256, generator=gen, device="cuda")).repeat_interleave(256) * size
    g = torch.randn(n, generator=gen, device="cuda") * sizes
    code, scale = _codes((0.3 + torch.rand(n, generator=gen, device="cuda")) * sizes)
    r = code.float() * scale.repeat_interleave(256)
    root = torch.sqrt(r * r * b2 + g * (1 - b2) * g)
    m, ms = torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), torch.ones(n // 256, device="cuda")
    G.adamw_step([torch.zeros(n, device="cuda")], [g], [m], [code], step=1000, lr=1e-3, betas=(b1, b2), eps=eps, weight_decay=0.0,
                 exp_avg_scale=[ms], exp_avg_sq_scale=[scale], seed=seed)
    b = root.view(-1, 256).double()
    power = torch.exp2((torch.floor(torch.log2(b.amax(1))) - 7).clamp(min=-100))
    assert torch.equal(power, scale.double())
    y = (b / power[:, None]).view(-1)
    step = torch.exp2((torch.floor(torch.log2(y)) - 3).clamp(min=-9))
    q = torch.floor(y / step + ((_bits(seed, n).cuda() >> 16).double() * 16 + 8) / 2 ** 20) * step
    q = torch.where((y > 0) & (q == 0), 2.0 ** -9, q)
    assert torch.equal(code.double(), q), (code.double() != q).sum().item()


def _with_state(value=2.0):
    import gelib_b200 as G
    p = torch.nn.Parameter(torch.ones(300, dtype=torch.bfloat16))
    opt = G.AdamW([p], state_bits=8)
    state = opt._state_of(p, 8)
    state["step"] = 4
    state["master"].fill_(value + 2.0 ** -12)
    state["exp_avg"].view(torch.uint8).fill_(9)
    state["exp_avg_scale"].fill_(0.25)
    return p, opt


def test_hooks_see_the_state_that_is_loaded():
    _, opt = _with_state()
    p, other = _with_state(1.0)
    seen = {}

    def before(o, d):
        seen["before"] = {k: dict(v) for k, v in d["state"].items()}

    def after(o):
        seen["after"] = dict(o.state[p])

    other.register_load_state_dict_pre_hook(before)
    other.register_load_state_dict_post_hook(after)
    for _ in range(2):   # nothing of the first call is left for the second
        seen.clear()
        other.load_state_dict(opt.state_dict())
        assert seen["before"][0]["step"] == 4 and float(seen["before"][0]["master"][0]) == 2.0 + 2.0 ** -12
        assert seen["after"]["step"] == 4 and seen["after"]["exp_avg"].dtype == torch.float8_e4m3fn
        assert seen["after"]["master"].dtype == torch.float32 and float(seen["after"]["master"][7]) == 2.0 + 2.0 ** -12
        assert (seen["after"]["exp_avg"].view(torch.uint8) == 9).all() and (seen["after"]["exp_avg_scale"] == 0.25).all()
    assert seen["after"]["master"] is not opt.state[opt.param_groups[0]["params"][0]]["master"]
    assert len(other._optimizer_load_state_dict_pre_hooks) == 1 and len(other._optimizer_load_state_dict_post_hooks) == 1


def test_a_hook_may_give_another_state():
    _, opt = _with_state()
    p, other = _with_state(1.0)

    def before(o, d):
        new = dict(d)
        new["state"] = {0: dict(d["state"][0], step=11)}
        return new

    other.register_load_state_dict_pre_hook(before)
    other.load_state_dict(opt.state_dict())
    assert other.state[p]["step"] == 11


def test_a_state_that_does_not_fit_changes_nothing():
    import gelib_b200 as G
    _, opt = _with_state()
    p, q = (torch.nn.Parameter(torch.ones(3)) for _ in range(2))
    other = G.AdamW([p, q])
    other._state_of(p, 32)
    with pytest.raises(ValueError):
        other.load_state_dict(opt.state_dict())
    assert p in other.state and not other._optimizer_load_state_dict_pre_hooks and not other._optimizer_load_state_dict_post_hooks
