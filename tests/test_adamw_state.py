"""What AdamW's state holds and takes back: layouts, captures, dicts that are refused. On the CPU where no step is taken."""
import copy

import pytest
import torch

from oracle import head as orc


def coded(p, seed=1):
    """An optimizer with moments in 8 bits for p, as if it had stepped: codes and exponents at random."""
    import kernels
    g = torch.Generator().manual_seed(seed)
    opt = kernels.AdamW([p], state_bits=8)
    s = opt._new_state(p, 8)
    for name, top in (("exp_avg", 120), ("exp_avg_sq", 249)):
        s[name].view(-1)[:p.numel()] = torch.randint(0, top, (p.numel(),), generator=g).to(torch.uint8)
        s[name + "_exps"].copy_(torch.randint(100, 140, s[name + "_exps"].shape, generator=g))
    s["step"] += 3
    opt.state[p] = s
    return opt


def leaf(shape, order=None, device="cpu"):
    """A parameter of that shape; order: its axes from the outermost in memory to the innermost."""
    order = order or tuple(range(len(shape)))
    x = torch.randn([shape[i] for i in order], generator=torch.Generator().manual_seed(5))
    back = [order.index(i) for i in range(len(shape))]
    return x.to(device).permute(back).requires_grad_(True)


LAYOUTS = [((5, 300), (1, 0), (0, 1)), ((5, 300), (0, 1), (1, 0)), ((4, 3, 50), (1, 0, 2), (0, 1, 2)), ((4, 3, 50), (2, 0, 1), (1, 0, 2)),
           ((2, 8, 3, 3), (0, 2, 3, 1), (0, 1, 2, 3))]


@pytest.mark.parametrize("shape,was,becomes", LAYOUTS)
def test_codes_do_not_go_into_another_layout(shape, was, becomes):
    """Codes lie as their parameter does: one that lies otherwise would take them for other elements."""
    import kernels
    saved = coded(leaf(shape, was)).state_dict()
    p = leaf(shape, becomes)
    opt = kernels.AdamW([p], lr=0.5, state_bits=8)
    with pytest.raises(ValueError, match="laid out"):
        opt.load_state_dict(saved)
    assert not opt.state.get(p) and opt.param_groups[0]["lr"] == 0.5


@pytest.mark.parametrize("shape,order", [((5, 300), (1, 0)), ((5, 300), (0, 1)), ((4, 3, 50), (2, 0, 1)), ((300,), (0,)), ((), ())])
def test_codes_go_into_the_same_layout(shape, order, tmp_path):
    import kernels
    a = leaf(shape, order)
    opt = coded(a)
    torch.save(opt.state_dict(), tmp_path / "state.pt")
    for saved in (copy.deepcopy(opt.state_dict()), torch.load(tmp_path / "state.pt", weights_only=True), copy.deepcopy(opt).state_dict()):
        b = leaf(shape, order)
        other = kernels.AdamW([b], state_bits=8)
        other.load_state_dict(saved)
        again = kernels.AdamW([leaf(shape, order)], state_bits=8)
        again.load_state_dict(other.state_dict())
        for o, p in ((other, b), (again, again.param_groups[0]["params"][0])):
            assert set(o.state[p]) == set(opt.state[a])
            for name in ("exp_avg", "exp_avg_exps", "exp_avg_sq", "exp_avg_sq_exps", "step"):
                assert torch.equal(o.state[p][name], opt.state[a][name])


def test_axes_of_one_element_have_no_place_in_a_layout():
    """The strides of such axes say nothing: a column and a row of one are alike."""
    import kernels
    a = torch.zeros(7, 40).t().unsqueeze(1).requires_grad_(True)                       # [40, 1, 7], strides (1, 280, 40) or the like
    b = torch.empty_strided((40, 1, 7), (1, 1, 40)).zero_().requires_grad_(True)
    assert a.stride() != b.stride()
    kernels.AdamW([b], state_bits=8).load_state_dict(coded(a).state_dict())


def test_moments_of_32_bits_go_by_element():
    import kernels
    a, b = leaf((5, 300), (1, 0)), leaf((5, 300), (0, 1))
    opt, other = kernels.AdamW([a]), kernels.AdamW([b])
    opt.state[a] = opt._new_state(a, 32)
    opt.state[a]["exp_avg"].copy_(torch.randn(5, 300))
    other.load_state_dict(opt.state_dict())
    assert torch.equal(other.state[b]["exp_avg"], opt.state[a]["exp_avg"]) and other.state[b]["exp_avg"].stride() == b.stride()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_that_changes_its_layout_is_refused(bits):
    import kernels
    p = leaf((5, 300), (0, 1), "cuda").detach().requires_grad_(True)
    opt = kernels.AdamW([p], state_bits=bits)
    p.grad = torch.ones_like(p)
    opt.step()
    kept, was = p.data, p.detach().clone()
    p.grad = None
    p.data = kept.t().contiguous().t()
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="laid out"):
        opt.step()
    if bits == 8:
        with pytest.raises(ValueError, match="laid out"):
            opt.moments()
    assert torch.equal(p, was) and int(opt.state[p]["step"]) == 1
    p.grad = None
    p.data = kept
    p.grad = torch.ones_like(p)
    opt.step()
    assert int(opt.state[p]["step"]) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("order", [(1, 0), (0, 1)])
def test_a_loaded_transposed_parameter_steps_on(order):
    """Saved, loaded and stepped: the moments by element are those of the optimizer that went on."""
    import kernels
    g = torch.Generator().manual_seed(2)
    a, b = (leaf((33, 40), order, "cuda").detach().requires_grad_(True) for _ in range(2))
    one, two = (kernels.AdamW([p], lr=0.1, state_bits=8) for p in (a, b))
    a.grad = torch.randn(33, 40, generator=g).cuda()
    one.step()
    two.load_state_dict(one.state_dict())
    b.data.copy_(a.data)
    a.grad = torch.randn(33, 40, generator=g).cuda()
    b.grad = a.grad.clone()
    one.step(), two.step()
    assert torch.equal(a, b)
    for x, y in zip(one.moments()[0], two.moments()[0]):
        assert torch.equal(x, y) and x.stride() == a.stride()
    flat = a.t() if order == (1, 0) else a
    m = orc.moment_values(one.state[a]["exp_avg"], one.state[a]["exp_avg_exps"], 14, False, a.numel()).view(flat.shape)
    assert torch.equal(one.moments()[0][0].cpu().double(), m.t() if order == (1, 0) else m)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["loaded", "copied"])
def test_a_capture_is_the_first_step_of_loaded_state(how, bits):
    """Captured first, then stepped eagerly before any replay, then replayed and stepped again: as many eager steps."""
    import kernels
    g = torch.Generator().manual_seed(3)
    shapes = [(70000,), (129, 3)]  # more blocks than one
    start = [torch.randn(s, generator=g).cuda().requires_grad_(True) for s in shapes]
    first = kernels.AdamW(start, lr=0.1, state_bits=bits)
    for p in start:
        p.grad = torch.randn(p.shape, generator=g).cuda()
    first.step()
    if how == "copied":
        opt, twin = copy.deepcopy(first), copy.deepcopy(first)
    else:
        opt, twin = (kernels.AdamW([p.detach().clone().requires_grad_(True) for p in start], state_bits=bits) for _ in range(2))
        opt.load_state_dict(first.state_dict()), twin.load_state_dict(first.state_dict())
    pairs = list(zip(opt.param_groups[0]["params"], twin.param_groups[0]["params"], start))
    for p, q, s in pairs:
        p.grad, q.grad = s.grad.clone(), s.grad.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for n, do in enumerate((opt.step, graph.replay, graph.replay, opt.step, graph.replay), 2):
        do()
        twin.step()
        for p, q, _ in pairs:
            assert int(opt.state[p]["step"]) == n and int(twin.state[q]["step"]) == n and torch.equal(p, q)
    for x, y in zip(opt.moments(), twin.moments()):
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


@pytest.mark.gpu
def test_a_capture_does_not_make_the_kernels_word():
    """State put in place by hand: there is no word yet, and a capture cannot make one. The step itself is refused, and one outside goes on."""
    import kernels
    p = torch.zeros(500, device="cuda", requires_grad=True)
    p.grad = torch.ones_like(p)
    opt = kernels.AdamW([p])
    opt.state[p] = opt._new_state(p, 32)
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert not opt._counters
    opt.step()
    assert int(opt.state[p]["step"]) == 1 and (p < 0).all()


def torch_dict(p, **kw):
    """A dict of torch's optimizer after a step of a parameter like p."""
    q = p.detach().clone().requires_grad_(True)
    opt = torch.optim.AdamW([q], lr=0.25, **kw)
    q.grad = torch.ones_like(q)
    opt.step()
    return opt.state_dict()


def spoiled(saved, group=None, **state):
    """The dict with other options of its group, or other entries of its state (None: without)."""
    saved = copy.deepcopy(saved)
    saved["param_groups"][0].update(group or {})
    for name, value in state.items():
        if value is None:
            del saved["state"][0][name]
        else:
            saved["state"][0][name] = value
    return saved


def refuses(opt, saved, match):
    """ValueError, with the optimizer as it was, its groups and its state."""
    before = copy.deepcopy(opt.state_dict())
    with pytest.raises(ValueError, match=match):
        opt.load_state_dict(saved)
    after = opt.state_dict()
    assert after["param_groups"] == before["param_groups"] and list(after["state"]) == list(before["state"])
    for key, s in before["state"].items():
        assert set(s) == set(after["state"][key])
        for name, x in s.items():
            assert torch.equal(x, after["state"][key][name]) if isinstance(x, torch.Tensor) else x == after["state"][key][name]


def test_options_that_there_are_not_are_refused():
    import kernels
    p = leaf((4, 6))
    for opt in (kernels.AdamW([p], lr=0.5), coded(p)):
        for kw in ({"maximize": True}, {"amsgrad": True}):
            refuses(opt, torch_dict(p, **kw), next(iter(kw)))
        # torch.optim.Adam's decay goes through the moments
        refuses(opt, spoiled(torch_dict(p), {"decoupled_weight_decay": False}), "decoupled")
    for kw in ({"maximize": True}, {"amsgrad": True}):
        with pytest.raises(ValueError, match=next(iter(kw))):
            kernels.AdamW([{"params": [p], **kw}])
    opt = kernels.AdamW([p])
    for saved in (torch_dict(p), spoiled(torch_dict(p), {"decoupled_weight_decay": False, "weight_decay": 0.0})):
        opt.load_state_dict(saved)
        assert opt.param_groups[0]["lr"] == 0.25 and torch.equal(opt.state[p]["exp_avg"], saved["state"][0]["exp_avg"])


def test_values_out_of_range_are_refused():
    import kernels
    p = leaf((4, 6))
    for opt in (kernels.AdamW([p], lr=0.5), coded(p)):
        for bad, match in (({"lr": -1.0}, "lr"), ({"betas": (1.0, 0.9)}, "betas"), ({"eps": -1.0}, "eps"), ({"weight_decay": -1.0}, "weight_decay")):
            refuses(opt, spoiled(torch_dict(p), bad), match)


@pytest.mark.parametrize("shape", [(1,), (1, 6), (4, 1), (6, 4), (4, 6, 1), ()])
def test_moments_of_another_shape_are_refused(shape):
    """Also where they could be repeated to fill the parameter's."""
    import kernels
    p = leaf((4, 6))
    for name in ("exp_avg", "exp_avg_sq"):
        refuses(kernels.AdamW([p], lr=0.5), spoiled(torch_dict(p), **{name: torch.ones(shape)}), name)
    refuses(kernels.AdamW([p]), spoiled(torch_dict(p), exp_avg=None), "exp_avg")
    refuses(kernels.AdamW([p]), spoiled(torch_dict(p), step=torch.zeros(2)), "step")


def test_codes_of_another_shape_or_type_are_refused():
    p, q = leaf((4, 60)), leaf((3, 100))
    saved = coded(q).state_dict()
    for bad, match in (({"exp_avg": torch.ones(1, 128, dtype=torch.uint8)}, "exp_avg"), ({"exp_avg_sq": torch.ones(3, 1, dtype=torch.uint8)}, "exp_avg_sq"),
                       ({"exp_avg_exps": torch.ones(1, dtype=torch.uint8)}, "exp_avg_exps"), ({"exp_avg_sq": torch.ones(3, 128)}, "exp_avg_sq"),
                       ({"exp_avg_sq_exps": None}, "exp_avg_sq_exps"), ({"step": torch.zeros(3)}, "step")):
        refuses(coded(q, 7), spoiled(saved, **bad), match)
    refuses(coded(p), saved, "exp_avg")  # 300 elements' for 240


def test_a_step_count_of_any_kind_is_taken():
    import kernels
    p = leaf((4, 6))
    opt = kernels.AdamW([p])
    for step in (7, 7.0, torch.tensor(7.0), torch.tensor([7])):
        opt.load_state_dict(spoiled(torch_dict(p), step=step))
        assert int(opt.state[p]["step"]) == 7 and opt.state[p]["step"].dtype == torch.int64 and opt.state[p]["step"].shape == ()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [lambda: torch.tensor(0.1, dtype=torch.float64), lambda: torch.tensor(0.1, dtype=torch.bfloat16), lambda: torch.zeros(0),
                                 lambda: torch.zeros(2), lambda: torch.tensor(1)], ids=["f64", "bf16", "none", "two", "int"])
def test_another_lr_on_the_device_is_checked(bad):
    """The kernel reads one float32: what a schedule puts in lr's place has to be one."""
    import kernels
    p = torch.ones(100, device="cuda", requires_grad=True)
    opt = kernels.AdamW([p], lr=torch.tensor(0.1, device="cuda"))
    p.grad = torch.ones_like(p)
    opt.step()
    was = p.detach().clone()
    opt.param_groups[0]["lr"] = bad().cuda()
    with pytest.raises(ValueError, match="one float32"):
        opt.step()
    assert torch.equal(p, was) and int(opt.state[p]["step"]) == 1


def test_the_lr_that_a_kernel_would_read():
    import flb_ops
    for bad in (torch.tensor(0.1, dtype=torch.float64), torch.zeros(0), torch.zeros(3)):
        with pytest.raises(ValueError, match="one float32"):
            flb_ops.adamw([], {}, 32, 0.0, bad, 0.9, 0.999, 1e-8, 0.0, 0, {})
    for good in (None, torch.tensor(0.1), torch.tensor([0.1])):
        assert flb_ops.adamw([], {}, 32, 0.0, good, 0.9, 0.999, 1e-8, 0.0, 0, {}) == []


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_first_step_leaves_no_state(bits):
    import kernels
    good = torch.ones(300, device="cuda", requires_grad=True)
    good.grad = torch.ones_like(good)
    gaps = torch.ones(40, 8, device="cuda")[:, :3].requires_grad_(True)
    gaps.grad = torch.ones_like(gaps)
    sparse = torch.ones(40, 8, device="cuda", requires_grad=True)
    sparse.grad = torch.ones(40, 8, device="cuda").to_sparse()
    for bad, match in ((gaps, "gaps"), (sparse, "sparse")):
        opt = kernels.AdamW([good, bad], state_bits=bits)
        with pytest.raises(ValueError, match=match):
            opt.step()
        assert not opt.state and opt.moments() == [] and (good == 1).all() and (bad == 1).all()
    sparse.grad = torch.ones_like(sparse)
    opt.step()
    assert [int(opt.state[p]["step"]) for p in (good, sparse)] == [1, 1] and (good < 1).all() and (sparse < 1).all()


def test_hooks_of_a_load():
    """What a hook before the load returns is what is loaded, and checked; one after it sees the state as it stays."""
    import kernels
    p = leaf((4, 6))
    saved = torch_dict(p)
    opt, seen = kernels.AdamW([p], lr=0.5), []

    def before(o, d):
        return spoiled(d, {"lr": 0.75}, exp_avg=2 * d["state"][0]["exp_avg"])

    handle = opt.register_load_state_dict_pre_hook(before)
    opt.register_load_state_dict_post_hook(lambda o: seen.append({k: t.dtype for k, t in o.state[p].items()}))
    for _ in range(2):
        opt.load_state_dict(saved)
        assert opt.param_groups[0]["lr"] == 0.75 and torch.equal(opt.state[p]["exp_avg"], 2 * saved["state"][0]["exp_avg"])
    assert seen == [{"step": torch.int64, "exp_avg": torch.float32, "exp_avg_sq": torch.float32}] * 2
    handle.remove()
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == 0.25 and torch.equal(opt.state[p]["exp_avg"], saved["state"][0]["exp_avg"])
    opt.register_load_state_dict_pre_hook(lambda o, d: spoiled(d, {"maximize": True}))
    refuses(opt, saved, "maximize")
