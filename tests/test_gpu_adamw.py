"""AdapterAdamW on the GPU against the numpy oracle: the moments bit for bit, the
parameters within the roundings of the update."""

import copy

import numpy as np
import pytest
import torch

from mirai_amd import AdapterAdamW, CompressedGroupedExperts, route_topk
from mirai_amd import workloads as wl
from oracle import adamw as oadam
from oracle import layer as olayer
from oracle import mxfp4 as omx

from helpers import build_module

pytestmark = pytest.mark.gpu

HYPER = {"lr": 1e-2, "betas": (0.9, 0.99), "eps": 1e-8, "weight_decay": 0.1}


class Model:
    """The oracle's state of one parameter group: float64 parameters of the types'
    values, fp32 or coded moments."""

    def __init__(self, params, bits, seed=0, group=0, **hyper):
        self.bits, self.seed, self.group = bits, seed, group
        self.h = {**HYPER, **hyper}
        self.p = [t.detach().double().cpu().numpy().reshape(-1) for t in params]
        self.bf16 = [t.dtype == torch.bfloat16 for t in params]
        self.slack = [np.zeros(p.size) for p in self.p]
        self.m = [np.zeros(p.size, dtype=np.float32) for p in self.p]
        self.v = [np.zeros(p.size, dtype=np.float32) for p in self.p]
        self.t = [0] * len(self.p)
        self.at = np.cumsum([0] + [-(-p.size // 128) * 128 for p in self.p])

    def step(self, grads):
        b1, b2 = self.h["betas"]
        for i, g in enumerate(grads):
            if g is None:
                continue
            g = g.detach().float().cpu().numpy().reshape(-1)
            self.t[i] += 1
            m, v = oadam.averages(g, self.m[i], self.v[i], b1, b2)
            new = oadam.update(self.p[i], m, v, lr=self.h["lr"], beta1=b1, beta2=b2, eps=self.h["eps"],
                               weight_decay=self.h["weight_decay"], step=self.t[i])
            # p (1 - lr wd): the factor and the product rounded; the update: its eight
            # constants and operations; the difference; half a step each, with the square
            # root allowed a whole one. bf16: its rounding on top.
            moved = new - self.p[i] * (1 - self.h["lr"] * self.h["weight_decay"])
            self.slack[i] += 2.0 ** -24 * (3 * np.abs(self.p[i]) + 10 * np.abs(moved) + np.abs(new)) + 1e-37
            if self.bf16[i]:
                self.slack[i] += 2.0 ** -8 * (np.abs(new) + self.slack[i])
            self.p[i] = new
            if self.bits == 8:
                n, at = m.size, int(self.at[i])
                low, high = oadam.noise(n, self.seed, self.t[i], self.group, at)
                m = oadam.decode(*oadam.encode(m, 4, True, low), 4, True).astype(np.float32)
                v = oadam.decode(*oadam.encode(v, 5, False, high), 5, False).astype(np.float32)
            self.m[i], self.v[i] = m, v

    def check(self, params, opt, group=0):
        fm, fv = (t.cpu().numpy() for t in opt.flat_moments(group))
        for i, p in enumerate(params):
            at, n = int(self.at[i]), self.p[i].size
            for flat, want in ((fm, self.m[i]), (fv, self.v[i])):
                assert np.array_equal(flat[at:at + n], want, equal_nan=True), i
                assert not flat[at + n:int(self.at[i + 1])].any()
            err = np.abs(p.detach().double().cpu().numpy().reshape(-1) - self.p[i])
            assert (err <= self.slack[i]).all(), (i, float((err - self.slack[i]).max()))


def _params(shapes, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(s, generator=g) * 0.1).to(dtype).cuda()) for s in shapes]


def _set_grads(params, seed, zero=()):
    g = torch.Generator().manual_seed(100 + seed)
    for i, p in enumerate(params):
        scale = 10.0 ** ((i % 5) - 3)
        grad = torch.randn(p.shape, generator=g) * scale
        grad[grad.abs() < 0.1 * scale] = 0
        p.grad = None if i in zero else grad.to(p.dtype).cuda()


SHAPES = [(1,), (7,), (128,), (129,), (3, 43), (8, 16, 64), (4096,), (4097,), (5, 1000), (2, 31, 130), (0,),
          (12289,)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps(bits, dtype):
    params = _params(SHAPES, dtype)
    opt = AdapterAdamW(params, **HYPER, state_bits=bits, seed=9)
    model = Model(params, bits, seed=9)
    for step in range(4):
        _set_grads(params, step)
        opt.step()
        model.step([p.grad for p in params])
        model.check(params, opt)
        if dtype == torch.bfloat16:  # the rounded parameters go on
            model.p = [p.detach().double().cpu().numpy().reshape(-1) for p in params]
            model.slack = [np.zeros(p.numel()) for p in params]


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_takes(bits):
    params = _params([(i % 9 + 1, 37) for i in range(200)])
    opt = AdapterAdamW(params, **HYPER, state_bits=bits)
    model = Model(params, bits)
    for step in range(2):
        _set_grads(params, step)
        opt.step()
        model.step([p.grad for p in params])
    model.check(params, opt)


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_without_gradients_are_left_alone(bits):
    params = _params([(300,), (40, 5), (129,)])
    opt = AdapterAdamW(params, **HYPER, state_bits=bits)
    model = Model(params, bits)
    for step, zero in enumerate(((1,), (), (0, 2), (0, 1, 2))):
        _set_grads(params, step, zero)
        opt.step()
        model.step([p.grad for p in params])
        model.check(params, opt)
    assert [opt.state[p]["step"] for p in params] == [2, 2, 2]


@pytest.mark.parametrize("bits", [32, 8])
def test_parameter_groups(bits):
    a, b = _params([(300,), (77,)]), _params([(5, 64)], torch.bfloat16, seed=1)
    opt = AdapterAdamW([{"params": a}, {"params": b, "lr": 1e-3, "weight_decay": 0.0}], **HYPER,
                       state_bits=bits, seed=3)
    models = [Model(a, bits, 3, 0), Model(b, bits, 3, 1, lr=1e-3, weight_decay=0.0)]
    _set_grads(a + b, 0)
    opt.step()
    for gi, (params, model) in enumerate(zip((a, b), models)):
        model.step([p.grad for p in params])
        model.check(params, opt, gi)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_gradients_stay_in_their_block(bits, bad):
    params = _params([(400,)])
    opt = AdapterAdamW(params, **HYPER, state_bits=bits)
    model = Model(params, bits)
    _set_grads(params, 0)
    params[0].grad[200] = bad
    opt.step()
    model.step([p.grad for p in params])
    fm, fv = (t.cpu().numpy() for t in opt.flat_moments())
    assert np.array_equal(fm[:400], model.m[0], equal_nan=True)
    assert np.array_equal(fv[:400], model.v[0], equal_nan=True)
    got = params[0].detach().cpu().numpy()
    assert np.isfinite(np.delete(got, 200)).all() and not np.isfinite(got[200])


@pytest.mark.parametrize("bits", [32, 8])
def test_tiny_and_huge_gradients(bits):
    g = np.concatenate([np.full(128, 1e-30), np.full(128, 1e18), [1e-22, 1e-3] * 64]).astype(np.float32)
    params = _params([(384,)])
    opt = AdapterAdamW(params, **HYPER, state_bits=bits)
    model = Model(params, bits)
    for _ in range(2):
        params[0].grad = torch.from_numpy(g).cuda()
        opt.step()
        model.step([params[0].grad])
        model.check(params, opt)


@pytest.mark.parametrize("bits", [32, 8])
def test_strides_and_alignment(bits):
    base = torch.randn(64, 48, device="cuda")
    flat = torch.randn(1001, device="cuda")
    params = [torch.nn.Parameter(base.t()), torch.nn.Parameter(flat[1:]),
              torch.nn.Parameter(torch.randn(6, 5, 4, device="cuda").permute(2, 0, 1))]
    twins = [torch.nn.Parameter(p.detach().clone(memory_format=torch.contiguous_format)) for p in params]
    opt = AdapterAdamW(params, **HYPER, state_bits=bits)
    ref = AdapterAdamW(twins, **HYPER, state_bits=32)
    for step in range(2):
        for p, q in zip(params, twins):
            grad = torch.randn(p.shape, generator=torch.Generator(device="cuda").manual_seed(step), device="cuda")
            p.grad, q.grad = grad, grad.clone()
        params[0].grad = params[0].grad.t().contiguous().t()  # the parameter's own order
        opt.step()
        ref.step()
    if bits == 32:
        for p, q in zip(params, twins):
            assert torch.equal(p, q)
            assert torch.equal(opt.state[p]["exp_avg"], ref.state[q]["exp_avg"])
    assert flat[0] == flat[0].clone()


@pytest.mark.parametrize("bits", [32, 8])
def test_saved_state_goes_on_bit_for_bit(bits):
    params = _params([(300,), (3, 50)], torch.bfloat16)
    opt = AdapterAdamW(params, **HYPER, state_bits=bits, seed=5)
    _set_grads(params, 0)
    opt.step()
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = AdapterAdamW(twins, **HYPER, state_bits=bits, seed=5)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    third_params = copy.deepcopy(params)
    third = copy.deepcopy(opt)
    third.param_groups[0]["params"], old = third_params, third.param_groups[0]["params"]
    third.state = type(third.state)(dict, {n: third.state[o] for n, o in zip(third_params, old)})
    for step in (1, 2):
        _set_grads(params, step)
        for p, q, r in zip(params, twins, third_params):
            q.grad, r.grad = p.grad.clone(), p.grad.clone()
        opt.step()
        other.step()
        third.step()
        for p, q, r in zip(params, twins, third_params):
            assert torch.equal(p, q) and torch.equal(p, r)
        for x, y in zip(opt.flat_moments(), other.flat_moments()):
            assert torch.equal(x, y)


def test_saved_state_is_checked():
    params = _params([(300,)])
    opt = AdapterAdamW(params, state_bits=8)
    _set_grads(params, 0)
    opt.step()
    with pytest.raises(ValueError, match="state_bits"):
        AdapterAdamW(_params([(300,)]), state_bits=32).load_state_dict(opt.state_dict())
    bad = copy.deepcopy(opt.state_dict())
    bad["state"][0]["exp_avg_e"] = bad["state"][0]["exp_avg_e"][:1]
    with pytest.raises(ValueError, match="exp_avg_e"):
        AdapterAdamW(_params([(300,)]), state_bits=8).load_state_dict(bad)
    del bad["state"][0]["exp_avg_e"]
    with pytest.raises(ValueError, match="lacks"):
        AdapterAdamW(_params([(300,)]), state_bits=8).load_state_dict(bad)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(bits):
    params, twins = _params([(300,), (64, 65)]), _params([(300,), (64, 65)])
    lr = torch.tensor(1e-2, device="cuda")
    opt = AdapterAdamW(params, **{**HYPER, "lr": lr}, state_bits=bits, capturable=True)
    ref = AdapterAdamW(twins, **HYPER, state_bits=bits)
    _set_grads(params, 0)
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    opt.step()
    ref.step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for step in range(1, 5):
        rate = 1e-2 / step
        lr.fill_(rate)
        ref.param_groups[0]["lr"] = float(lr)
        for p, q in zip(params, twins):
            q.grad = torch.randn(p.shape, generator=torch.Generator(device="cuda").manual_seed(step),
                                 device="cuda")
            p.grad.copy_(q.grad)
        graph.replay()
        torch.cuda.synchronize()
        ref.step()
        for p, q in zip(params, twins):
            assert torch.equal(p, q), step
        for x, y in zip(opt.flat_moments(), ref.flat_moments()):
            assert torch.equal(x, y), step
    assert int(opt.state[params[0]]["step"]) == 5
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ref.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_goes_on_after_a_load(bits):
    params, twins = _params([(300,), (64, 65)]), _params([(300,), (64, 65)])
    opt = AdapterAdamW(params, **HYPER, state_bits=bits, capturable=True)
    ref = AdapterAdamW(twins, **HYPER, state_bits=bits)
    for p, q in zip(params, twins):
        q.grad = torch.randn(p.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
        p.grad = q.grad.clone()
    opt.step()
    ref.step()
    saved, kept = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in params]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    graph.replay()
    held = opt._groups[0]
    opt.load_state_dict(saved)
    assert opt._groups[0] is held
    with torch.no_grad():
        for p, k in zip(params, kept):
            p.copy_(k)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        ref.step()
        for p, q in zip(params, twins):
            assert torch.equal(p, q)
    # Its own state: nothing changes.
    before = [t.clone() for t in opt.flat_moments()]
    opt.load_state_dict(opt.state_dict())
    for a, b in zip(before, opt.flat_moments()):
        assert torch.equal(a, b)
    assert int(opt.state[params[0]]["step"]) == 3


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_state_taken_away_or_replaced(bits, capturable):
    params, twins = _params([(300,), (64, 65)]), _params([(300,), (64, 65)])
    opt = AdapterAdamW(params, **HYPER, state_bits=bits, capturable=capturable)
    for s in range(2):
        _set_grads(params, s)
        opt.step()
    saved = {k: copy.deepcopy(dict(v)) for k, v in zip("ab", opt.state.values())}
    values = [p.detach().clone() for p in params]

    def again():
        for s in range(2):
            for ps, o in ((params, opt), (twins, ref)):
                _set_grads(ps, s)
                o.step()
            for p, q in zip(params, twins):
                assert torch.equal(p, q)

    # Emptied: from the first step again.
    with torch.no_grad():
        for p, q in zip(params, twins):
            q.copy_(p)
    opt.state.clear()
    ref = AdapterAdamW(twins, **HYPER, state_bits=bits)
    again()
    assert int(opt.state[params[1]]["step"]) == 2

    # Replaced: from what the new entries hold.
    ref = AdapterAdamW(twins, **HYPER, state_bits=bits)
    with torch.no_grad():
        for p, q, v in zip(params, twins, values):
            p.copy_(v)
            q.copy_(v)
    for o, ps in ((opt, params), (ref, twins)):
        for k, p in zip("ab", ps):
            o.state[p] = copy.deepcopy(saved[k])
    again()
    assert int(opt.state[params[1]]["step"]) == 4 == int(ref.state[twins[1]]["step"])


def test_learning_rates_after_construction():
    params = _params([(300,)])
    opt = AdapterAdamW(params)
    _set_grads(params, 0)
    before = params[0].detach().clone()
    for lr in (torch.tensor(1e-3, device="cuda"), -1.0, float("nan")):
        opt.param_groups[0]["lr"] = lr
        with pytest.raises(ValueError, match="lr|learning rate"):
            opt.step()
        with pytest.raises(ValueError, match="lr|learning rate"):
            opt.add_param_group({"params": _params([(5,)]), "lr": lr})
    assert torch.equal(params[0], before) and len(opt.param_groups) == 1

    # Between optimisers with a learning rate on the GPU and ones without: the tensor
    # stays, its value and the numbers go over.
    rate = torch.tensor(0.5, device="cuda")
    a = AdapterAdamW(params, lr=rate, capturable=True)
    b = AdapterAdamW(params, lr=0.25)
    saved = copy.deepcopy(a.state_dict())
    a.load_state_dict(b.state_dict())
    assert a.param_groups[0]["lr"] is rate and float(rate) == 0.25
    b.load_state_dict(saved)
    assert b.param_groups[0]["lr"] == 0.5
    a.load_state_dict(saved)
    assert a.param_groups[0]["lr"] is rate and float(rate) == 0.5


def test_state_of_the_plain_optimiser():
    """torch.optim.AdamW's state goes on here: the same formula, a few roundings of
    fp32 apart (at most 8 per step and value: the update is lr long, the parameter's own
    roundings 2 more)."""
    params, twins = _params([(300,), (64, 65)]), _params([(300,), (64, 65)])
    ref = torch.optim.AdamW(twins, lr=1e-3, weight_decay=0.1)
    for s in range(3):
        _set_grads(twins, s)
        ref.step()
    opt = AdapterAdamW(params)
    opt.load_state_dict(copy.deepcopy(ref.state_dict()))
    with torch.no_grad():
        for p, q in zip(params, twins):
            p.copy_(q)
    assert opt.param_groups[0]["weight_decay"] == 0.1
    for s in range(3, 5):
        _set_grads(params, s)
        _set_grads(twins, s)
        opt.step()
        ref.step()
    eps = torch.finfo(torch.float32).eps / 2
    for p, q in zip(params, twins):
        # |m| / sqrt(v) is at most (1 - b1) / sqrt(1 - b2) / (1 - b1 / sqrt(b2)) < 33.
        assert float((p - q).abs().max()) <= 2 * (8 * eps * 33e-3 + 4 * eps * float(q.abs().max()))
    assert int(opt.state[params[0]]["step"]) == 5
    for other in (torch.optim.AdamW(twins, amsgrad=True), torch.optim.AdamW(twins, maximize=True)):
        with pytest.raises(ValueError, match="amsgrad|maximize"):
            opt.load_state_dict(other.state_dict())


def test_positions_past_32_bits():
    """8-bit moments behind (and within) a parameter of more than 2^32 elements."""
    big = torch.nn.Parameter(torch.zeros(2 ** 32 + 77, dtype=torch.bfloat16, device="cuda"))
    (small,) = _params([(4097,)], torch.bfloat16)
    opt = AdapterAdamW([big, small], **HYPER, state_bits=8, seed=5)
    big.grad = torch.zeros_like(big)
    big.grad[-1] = 3.0
    _set_grads([small], 2)
    tail = torch.zeros(77 + 128, dtype=torch.float32, device="cuda")
    tail[-1] = 3.0
    opt.step()
    b1, b2 = HYPER["betas"]
    for p, g, n, at in ((big, tail, 205, 2 ** 32 - 128), (small, small.grad, 4097, 2 ** 32 + 128)):
        zero = np.zeros(n, dtype=np.float32)
        m, v = oadam.averages(g.float().cpu().numpy(), zero, zero, b1, b2)
        low, high = oadam.noise(n, 5, 1, 0, at)
        for name, x, noise, ebits, signed in (("exp_avg", m, low, 4, True), ("exp_avg_sq", v, high, 5, False)):
            codes, exps = oadam.encode(x, ebits, signed, noise)
            entry = opt.state[p]
            assert np.array_equal(entry[name + "_q"][-n:].cpu().numpy(), codes)
            assert np.array_equal(entry[name + "_e"][-exps.size:].cpu().numpy(), exps)
    assert not opt.state[big]["exp_avg_q"][:-1].any() and not big.detach()[:-1].any() and float(big.detach()[-1]) < 0
    for flat, entry in zip(opt.flat_moments(), ("exp_avg", "exp_avg_sq")):
        q, e = opt.state[small][entry + "_q"].cpu().numpy(), opt.state[small][entry + "_e"].cpu().numpy()
        want = oadam.decode(q, e, 4 if entry == "exp_avg" else 5, entry == "exp_avg")
        at = 2 ** 32 + 128
        assert np.array_equal(flat[at:at + 4097].double().cpu().numpy(), want)


def test_parameters_without_elements():
    params = _params([(0,), (3, 0)])
    opt = AdapterAdamW(params)
    _set_grads(params, 0)
    opt.step()
    assert all(t.numel() == 0 for t in opt.flat_moments())


def test_parameters_whose_storage_changed_are_refused():
    for swap in (lambda p: torch.zeros(100, device="cuda"), lambda p: torch.zeros(300, 2, device="cuda")[:, 0]):
        params = _params([(300,)])
        opt = AdapterAdamW(params)
        _set_grads(params, 0)
        opt.step()
        params[0].grad = None
        params[0].data = swap(params[0])
        params[0].grad = torch.ones_like(params[0])
        with pytest.raises(ValueError, match="storage changed|shape"):
            opt.step()


def test_refusals():
    params = _params([(300,)])
    opt = AdapterAdamW(params)
    opt.step()  # no gradients: nothing to do
    assert not opt.state[params[0]]
    params[0].grad = torch.zeros(300, device="cuda").to_sparse()
    with pytest.raises(ValueError, match="dense"):
        opt.step()
    with pytest.raises(ValueError, match="GPU|ROCm|device"):
        p = torch.nn.Parameter(torch.zeros(4))
        p.grad = torch.zeros(4)
        AdapterAdamW([p]).step()


def test_the_closure_and_the_version():
    params = _params([(300,)])
    opt = AdapterAdamW(params, **HYPER)
    before = params[0]._version

    def closure():
        opt.zero_grad()
        loss = (params[0] ** 2).sum()
        loss.backward()
        return loss

    loss = opt.step(closure)
    assert float(loss.detach()) > 0 and params[0]._version > before


@pytest.mark.parametrize("bits", [32, 8])
def test_an_adapter_training_step_over_mxfp4_experts(bits):
    """Experts quantised to MXFP4, routed layer forward and backward, AdamW step:
    against autograd through the oracle layer and the oracle step; the next forward
    runs with the new factors."""
    w = wl.Workload("mxtrain", 15, 64, 256, 192, 8, 2, 8, 16.0, "mxfp4", torch.bfloat16)
    dense, lora = wl.dense_weights(w), wl.lora_factors(w)
    m = build_module(w, dense, lora)
    factors = [t for k in ("w1", "w3", "w2") for t in (m.expert_lora[k].lora_a, m.expert_lora[k].lora_b)]
    opt = AdapterAdamW(m.expert_lora.parameters(), **HYPER, state_bits=bits)
    idx, scores = route_topk(wl.router_logits(w).cuda(), w.top_k)
    x, dy = wl.tokens(w), wl.upstream_grad(w)
    m.run_direct_routed(x.cuda(), scores, idx).backward(dy.cuda())
    order = list(m.expert_lora.parameters())
    model = Model(order, bits)
    model.step([p.grad for p in order])
    opt.step()
    model.check(order, opt)
    with torch.no_grad():
        after = m.run_direct_routed(x.cuda(), scores, idx)
    ow = {k: torch.from_numpy(omx.roundtrip(t.float().numpy())).bfloat16() for k, t in dense.items()}
    new = {k: (m.expert_lora[k].lora_a.detach().cpu(), m.expert_lora[k].lora_b.detach().cpu(),
               float(w.alpha) / w.rank) for k in ("w1", "w3", "w2")}
    ref = olayer.layer_forward(x, scores.cpu(), idx.cpu(), ow, new, w.experts)
    rel = float((after.float().cpu() - ref.float()).abs().sum() / ref.float().abs().sum())
    assert rel <= 5e-3 and len(factors) == 6
    assert isinstance(m, CompressedGroupedExperts)
