"""The optimizer without a GPU: checkpoints, copies and refused steps.  The step itself is the kernel's and is replaced or refused here."""

import copy
import io
import pickle

import pytest
import torch

import fp8_gmm_amd as pkg
from fp8_gmm_amd import backend


def make(n=2, **options):
    return pkg.AdamW([torch.nn.Parameter(torch.full((3,), i + 1.0, dtype=torch.bfloat16)) for i in range(n)], **options)


def stepped(value=7.0, **options):
    """An optimizer whose states are there, as a step on the GPU leaves them."""
    opt = make(**options)
    for p in opt.param_groups[0]["params"]:
        opt._init_state(p, opt.state[p])
        opt.state[p]["exp_avg"].fill_(value)
        if not opt.capturable:
            opt.state[p]["step"] = 5
    if opt.capturable:
        opt.param_groups[0]["steps"] = torch.tensor(5)
    return opt


@pytest.mark.parametrize("options", [dict(), dict(state_bits=8, master_weights=True), dict(capturable=True)])
def test_hooks_of_a_load_have_their_way(options):
    saved = stepped(**options).state_dict()

    def zeroed(_, state_dict):
        return {**state_dict, "state": {k: {**v, "exp_avg": torch.zeros_like(v["exp_avg"])} for k, v in state_dict["state"].items()}}

    opt = make(**options)
    opt.register_load_state_dict_pre_hook(zeroed)
    opt.load_state_dict(saved)
    for p in opt.param_groups[0]["params"]:
        assert not opt.state[p]["exp_avg"].float().any() and opt.state[p]["exp_avg"].dtype == saved["state"][0]["exp_avg"].dtype
        assert opt.state[p]["exp_avg"] is not saved["state"][0]["exp_avg"]

    opt = make(**options)
    opt.register_load_state_dict_pre_hook(lambda _, state_dict: {**state_dict, "state": {}})
    opt.load_state_dict(saved)
    assert not opt.state

    def renamed(_, state_dict):   # a checkpoint of another layout, put right by its hook
        return {"state": state_dict["moments"], "param_groups": state_dict["groups"]}

    opt = make(**options)
    opt.register_load_state_dict_pre_hook(renamed)
    opt.load_state_dict({"moments": saved["state"], "groups": saved["param_groups"]})
    assert all((opt.state[p]["exp_avg"].float() == 7).all() for p in opt.param_groups[0]["params"])

    def behind(optimizer):
        for p in optimizer.param_groups[0]["params"]:
            assert optimizer.state[p]["exp_avg"].dtype == saved["state"][0]["exp_avg"].dtype
            optimizer.state[p]["exp_avg"].fill_(2.0)

    opt = make(**options)
    opt.register_load_state_dict_post_hook(behind)
    opt.load_state_dict(saved)
    assert all((opt.state[p]["exp_avg"].float() == 2).all() for p in opt.param_groups[0]["params"])


def test_a_load_leaves_no_hook_behind():
    opt = make()
    opt.load_state_dict(stepped().state_dict())
    for other in (stepped(state_bits=8), stepped()):
        hooks = [len(h) for h in (opt._optimizer_load_state_dict_pre_hooks, opt._optimizer_load_state_dict_post_hooks)]
        assert hooks == [0, 0]
        before = {p: dict(opt.state[p]) for p in opt.param_groups[0]["params"]}
        if other.state_bits == 8:
            with pytest.raises(ValueError, match="not a checkpoint"):
                opt.load_state_dict(other.state_dict())
            assert all(opt.state[p][k] is v for p, s in before.items() for k, v in s.items())


@pytest.mark.parametrize("options", [dict(), dict(state_bits=8, master_weights=True, max_norm=0.5), dict(capturable=True, lr=torch.tensor(0.5))])
def test_copies_step_as_their_original_does(options, monkeypatch):
    opt = stepped(**options)
    calls = []
    monkeypatch.setattr(backend, "multi_adamw", lambda *args: calls.append(args))
    monkeypatch.setattr(backend, "multi_norm", lambda grads: torch.tensor(2.0))
    file = io.BytesIO()
    torch.save(opt, file)
    file.seek(0)
    copies = [copy.deepcopy(opt), torch.load(file, weights_only=False)]
    if opt.state_bits == 32:   # (pickle alone takes no tensor of 8-bit floats, whoever holds it)
        copies.append(pickle.loads(pickle.dumps(opt)))
    copies.append(copy.copy(opt))   # last: it shares the states
    for copied in copies:
        for name in ("state_bits", "master_weights", "max_norm", "capturable", "grad_norm"):
            assert getattr(copied, name) == getattr(opt, name)
        for p, q in zip(opt.param_groups[0]["params"], copied.param_groups[0]["params"]):
            assert {k: getattr(v, "dtype", v) for k, v in opt.state[p].items()} == {k: getattr(v, "dtype", v) for k, v in copied.state[q].items()}
            q.grad = torch.ones_like(q)
        copied.step()
        assert len(calls.pop()[0]) == 2 and not calls
        again = make(**options)
        again.load_state_dict(copied.state_dict())
        if "max_norm" in options:
            assert copied.grad_norm == 2.0


@pytest.mark.parametrize("capturable", [True, False])
def test_a_refused_step_does_not_count(capturable, monkeypatch):
    opt = stepped(capturable=capturable)
    group = opt.param_groups[0]

    def steps():
        return [int(group["steps"])] if capturable else [opt.state[p]["step"] for p in group["params"]]

    for p in group["params"]:
        p.grad = torch.ones_like(p)
    for _ in range(3):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            opt.step()
    assert set(steps()) == {5}
    monkeypatch.setattr(backend, "multi_adamw", lambda *args: None)
    opt.step()
    assert set(steps()) == {6}

    calls = []

    def second_refused(*args):   # of a group whose parameters have masters and have none
        calls.append(args)
        if len(calls) == 2:
            raise RuntimeError("refused")

    mixed = pkg.AdamW([torch.nn.Parameter(torch.ones(3, dtype=t)) for t in (torch.bfloat16, torch.float32)], master_weights=True,
                      capturable=capturable)
    for p in mixed.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    monkeypatch.setattr(backend, "multi_adamw", second_refused)
    with pytest.raises(RuntimeError, match="refused"):
        mixed.step()
    assert len(calls) == 2 and (int(mixed.param_groups[0]["steps"]) == 1 if capturable else
                                [mixed.state[p]["step"] for p in mixed.param_groups[0]["params"]] == [1, 0])


@pytest.mark.parametrize("capturable", [True, False])
def test_groups_without_parameters_load(capturable):
    lr = torch.tensor(0.25) if capturable else 0.25

    def with_empty(params):
        return pkg.AdamW([{"params": params}, {"params": [], "lr": lr}], capturable=capturable)

    opt = with_empty([torch.nn.Parameter(torch.ones(3))])
    p, = opt.param_groups[0]["params"]
    opt._init_state(p, opt.state[p])
    opt.step()   # nothing to do
    other = with_empty([torch.nn.Parameter(torch.ones(3))])
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[1]["params"] == [] and float(other.param_groups[1]["lr"]) == 0.25
    assert set(other.state[other.param_groups[0]["params"][0]]) == set(opt.state[p])


def test_arguments_that_torchs_users_give():
    p = [torch.nn.Parameter(torch.ones(3))]
    theirs = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1, amsgrad=False, maximize=False, foreach=None, capturable=False,
                  differentiable=False, fused=None)
    torch.optim.AdamW(p, **theirs)
    for options in (theirs, {**theirs, "foreach": True}, {**theirs, "fused": True}):
        assert pkg.AdamW(p, **options).param_groups[0]["betas"] == (0.9, 0.99)
    for name in ("amsgrad", "maximize", "differentiable"):
        with pytest.raises(ValueError, match=name):
            pkg.AdamW(p, **{**theirs, name: True})
        with pytest.raises(ValueError, match=name):
            pkg.AdamW([{"params": p, name: True}])
    with pytest.raises(ValueError, match="amsgrad"):
        pkg.AdamW(p, 1e-3, (0.9, 0.99), 1e-8, 0.1, True)
    with pytest.raises(TypeError, match="dict"):
        pkg.AdamW(p).add_param_group(p)
