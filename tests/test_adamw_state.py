"""AdamW's state as it is loaded, without a GPU: its own types, torch's hooks, entries that are no tensors."""
import copy

import pytest
import torch

from tgengine_amd import ops

F, B, E = torch.float32, torch.bfloat16, torch.float8_e4m3fn


def _new(dtype=B):
    params = [torch.nn.Parameter(torch.zeros(n, dtype=dtype)) for n in (300, 5)]
    return params, ops.AdamW(params, lr=1e-2, bits=8)


def _saved(seed=0):
    """A state dict of an 8-bit and a 32-bit tensor, 7 steps on."""
    g = torch.Generator().manual_seed(seed)
    first = {"step": torch.tensor(7), "exp_avg": torch.randn(300, generator=g).to(E), "exp_avg_sq": torch.rand(300, generator=g).to(E),
             "scales": torch.full((2, 2), 2.0 ** -100)}
    second = {"step": torch.tensor(7), "exp_avg": torch.randn(5, generator=g) / 3, "exp_avg_sq": torch.rand(5, generator=g) / 3}
    out = _new()[1].state_dict()
    out["state"] = {0: first, 1: second}
    return out


def _same(a, b):
    return set(a) == set(b) and all(a[k].dtype == b[k].dtype and torch.equal(a[k].float(), b[k].float()) for k in a)


@pytest.mark.parametrize("dtype", [F, B])
def test_types_and_copies(dtype):
    params, adam = _new(dtype)
    saved = _saved()
    kept = copy.deepcopy(saved["state"])
    adam.load_state_dict(saved)
    for i, p in enumerate(params):
        assert _same(adam.state[p], kept[i])
        for k, v in adam.state[p].items():
            assert v.data_ptr() != saved["state"][i][k].data_ptr()
            v.zero_()
    assert all(_same(saved["state"][i], kept[i]) for i in kept)  # what was loaded stays
    assert not adam._optimizer_load_state_dict_pre_hooks and not adam._optimizer_load_state_dict_post_hooks


@pytest.mark.parametrize("in_place", [False, True])
def test_pre_hooks(in_place):
    """A hook that changes the dictionary, or gives another one, decides what is loaded."""
    params, adam = _new()
    other = _saved(1)

    def hook(_, given):
        if in_place:
            given["state"] = other["state"]
            return None
        return other

    adam.register_load_state_dict_pre_hook(hook)
    adam.load_state_dict(_saved())
    assert all(_same(adam.state[p], other["state"][i]) for i, p in enumerate(params))


def test_post_hooks():
    """A hook sees the loaded state, in its types, and what it writes stays."""
    params, adam = _new()
    seen = []

    def hook(o):
        seen.append([{k: v.clone() for k, v in o.state[p].items()} for p in params])
        o.state[params[1]]["exp_avg"].fill_(0.7)
        o.state[params[0]]["step"] = torch.tensor(99)

    adam.register_load_state_dict_post_hook(hook)
    saved = _saved()
    adam.load_state_dict(saved)
    assert all(_same(s, saved["state"][i]) for i, s in enumerate(seen[0]))
    assert bool((adam.state[params[1]]["exp_avg"] == 0.7).all()) and int(adam.state[params[0]]["step"]) == 99


def test_entries_that_are_no_tensors():
    params, adam = _new()
    saved = _saved()
    saved["state"][1]["note"] = "warm"
    saved["state"][1]["seen"] = [3, 4]
    adam.load_state_dict(saved)
    assert adam.state[params[1]]["note"] == "warm" and adam.state[params[1]]["seen"] == [3, 4]
    assert torch.equal(adam.state[params[1]]["exp_avg"], saved["state"][1]["exp_avg"])


def test_a_refused_state_leaves_no_hooks():
    _, adam = _new()
    saved = _saved()
    saved["param_groups"][0]["params"] = [0]
    with pytest.raises(ValueError, match="size of optimizer's group"):
        adam.load_state_dict(saved)
    assert not adam.state and not adam._optimizer_load_state_dict_pre_hooks and not adam._optimizer_load_state_dict_post_hooks


def test_states_of_some_parameters_only():
    params, adam = _new()
    saved = _saved()
    del saved["state"][0]
    adam.load_state_dict(saved)
    assert params[0] not in adam.state and _same(adam.state[params[1]], saved["state"][1])
