"""Argument checks of the choices by rules and of the update over many tensors, without a GPU: every refusal comes before any device work."""
import ctypes

import pytest
import torch

FAKE = ctypes.c_void_p(0x1000)      # never dereferenced: every call below fails validation first
BIG = 1 << 32
OK, TOO_LARGE, BAD, WORKSPACE = 0, 2, 3, 4
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def lib():
    from snntc_amd import _lib
    return _lib.load()


def _rules(**how):
    from snntc_amd import _lib
    r = _lib.Rules(history=FAKE, history_rows=2, history_len=5, repetition_all=1.5, presence_all=0.0, frequency_all=0.0, delay_rows=1,
                   allowed_rows=1)
    for k, v in how.items():
        setattr(r, k, v)
    return ctypes.byref(r)


@pytest.mark.parametrize("entry", ["times", "backward", "choose"])
def test_rules_argument_errors(lib, entry):
    def call(r=4, j=70000, ty=0, t=FAKE, out=FAKE, rules=None, ws=FAKE, have=1 << 20):
        rules = _rules() if rules is None else rules
        if entry == "times":
            return lib.snntc_rule_times(t, ty, rules, out, r, j, None)
        if entry == "backward":
            return lib.snntc_rule_times_backward(FAKE, t, ty, rules, out, r, j, None)
        return lib.snntc_choose(t, ty, FAKE, None, 1.0, rules, out, FAKE, r, j, ws, have, None)
    assert call(t=None) == call(out=None) == call(ty=3) == call(ty=-1) == call(r=-1) == call(j=-1) == call(j=0) == BAD
    assert call(r=1 << 24) == call(j=BIG) == call(rules=_rules(history_len=BIG)) == TOO_LARGE
    assert call(rules=_rules(history_len=-1)) == call(rules=_rules(history_rows=-1)) == call(rules=_rules(history_rows=0)) == BAD
    assert call(rules=_rules(history_rows=3)) == BAD and b"do not divide" in lib.snntc_last_error()
    assert call(rules=_rules(delay=FAKE, delay_rows=2)) == call(rules=_rules(allowed=FAKE, allowed_rows=3)) == BAD
    for bad in (0.0, -1.0, NAN, INF):
        assert call(rules=_rules(repetition_all=bad)) == BAD
    for bad in (NAN, INF):
        assert call(rules=_rules(presence_all=bad)) == call(rules=_rules(frequency_all=bad)) == BAD
    assert call(r=0) == call(r=0, j=0) == call(r=0, t=None, out=None) == OK


def test_rules_that_read_no_times_need_none(lib):
    """Without a history, or a repetition other than 1, the gradient does not read the times: only its own tensors are missing here."""
    for rules in (_rules(history=None), _rules(repetition_all=1.0), None):
        assert lib.snntc_rule_times_backward(None, None, 0, rules, FAKE, 4, 5, None) == BAD
        assert lib.snntc_rule_times_backward(FAKE, None, 0, rules, None, 4, 5, None) == BAD


def test_choose_argument_errors(lib):
    need = ctypes.c_size_t()
    assert lib.snntc_choose_workspace_bytes(100, 64, ctypes.byref(need)) == OK and need.value == 0
    assert lib.snntc_choose_workspace_bytes(100, 200000, ctypes.byref(need)) == OK and need.value > 0
    assert lib.snntc_choose_workspace_bytes(100, 10, None) == lib.snntc_choose_workspace_bytes(-1, 10, ctypes.byref(need)) == BAD
    f = lambda u=FAKE, heat=None, all_=1.0, lp=FAKE, ws=FAKE, have=1 << 20: lib.snntc_choose(
        FAKE, 0, u, heat, all_, None, FAKE, lp, 4, 200000, ws, have, None)
    assert f(u=None) == f(u=None, heat=FAKE, all_=0.0) == f(lp=None) == BAD
    assert f(all_=-0.1) == f(all_=NAN) == f(all_=INF) == BAD
    assert f(ws=None) == f(have=16) == f(ws=ctypes.c_void_p(0x1010)) == f(u=None, all_=0.0, ws=None) == WORKSPACE


def _array(*values):
    return (ctypes.c_void_p * len(values))(*values)


def test_adamw_argument_errors(lib):
    from snntc_amd import _lib
    one = _array(0x1000, 0x2000)
    hole = _array(0x1000, None)
    n = (ctypes.c_int64 * 2)(4, 300)
    types = (ctypes.c_int * 2)(0, 1)

    def numbers(**how):
        a = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1, max_norm=1.0)
        return ctypes.byref(_lib.AdamW(**{**a, **how}))

    def f(w=one, g=one, m=one, v=one, ms=None, vs=None, ty=types, sizes=n, count=2, how=None, ws=None, have=0):
        return lib.snntc_adamw_update(w, g, m, v, ms, vs, ty, sizes, count, numbers() if how is None else how, ws, have, None)
    assert f(count=-1) == f(sizes=(ctypes.c_int64 * 2)(4, -1)) == f(ty=(ctypes.c_int * 2)(0, 7)) == f(ty=None) == f(sizes=None) == BAD
    assert f(sizes=(ctypes.c_int64 * 2)(4, (1 << 34) + 1)) == TOO_LARGE
    for k in "wgmv":
        assert f(**{k: hole}) == f(**{k: None}) == BAD
    assert f(ms=one) == f(vs=one) == f(ms=hole, vs=one) == f(ms=one, vs=hole) == BAD
    for how in (dict(lr=-1.0), dict(lr=NAN), dict(lr=INF), dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0), dict(beta2=NAN), dict(eps=0.0),
                dict(eps=1e-45), dict(eps=NAN), dict(eps=INF), dict(weight_decay=-0.1), dict(weight_decay=INF), dict(step=0), dict(step=-3),
                dict(norm=FAKE, max_norm=0.0), dict(norm=FAKE, max_norm=NAN)):
        assert f(how=numbers(**how)) == BAD, how
    assert f(how=numbers(steps=FAKE)) == f(how=numbers(steps=FAKE), ws=FAKE, have=8) == WORKSPACE
    assert f(count=0) == OK and f(sizes=(ctypes.c_int64 * 2)(0, 0), w=_array(None, None)) == OK
    assert lib.snntc_adamw_update(one, one, one, one, None, None, types, n, 2, None, None, 0, None) == BAD

    need = ctypes.c_size_t()
    assert lib.snntc_grad_norm_workspace_bytes(n, 2, ctypes.byref(need)) == OK and need.value >= 16
    assert lib.snntc_grad_norm_workspace_bytes(n, 2, None) == lib.snntc_grad_norm_workspace_bytes(n, -1, ctypes.byref(need)) == BAD
    g = lambda g=one, ty=types, sizes=n, norm=FAKE, ws=FAKE, have=1 << 20: lib.snntc_grad_norm(g, ty, sizes, 2, norm, ws, have, None)
    assert g(g=None) == g(g=hole) == g(ty=None) == g(ty=(ctypes.c_int * 2)(0, 3)) == g(sizes=None) == g(norm=None) == BAD
    assert g(sizes=(ctypes.c_int64 * 2)(4, 1 << 35)) == TOO_LARGE and g(ws=None) == g(have=8) == WORKSPACE
    h = lambda *at: lib.snntc_adamw_moments(*[hole if i in at else one for i in range(6)], n, 2, None)
    assert all(h(i) == BAD for i in range(6))


def test_host_tensors_are_refused():
    import snntc_amd as snn
    x, k = torch.rand(2, 3), torch.zeros(2, 3, dtype=torch.int64)
    for call in (lambda: snn.rule_times(x), lambda: snn.rule_times_grad(x, x), lambda: snn.choose_tokens(x, x[:, 0]), lambda: snn.grad_norm([x]),
                 lambda: snn.adamw_update([x], [x], [x], [x], 1), lambda: snn.adamw_moments([x], [x], [x], [x])):
        with pytest.raises(snn.SnntcLibraryError, match="no CPU fallback"):
            call()
    with pytest.raises(TypeError, match="times must be a torch.Tensor"):
        snn.rule_times([1.0, 2.0])
    with pytest.raises(TypeError, match="must be a list|iterable"):
        snn.grad_norm(3)
    with pytest.raises(ValueError, match="no gradients"):
        snn.grad_norm([])
    snn.adamw_update([], [], [], [], 1)
    with pytest.raises(ValueError, match="8 or 32"):
        snn.optim.AdamW([torch.nn.Parameter(x)], state_bits=16)
    with pytest.raises(ValueError, match="at least one token"):
        snn.train.answer(snn.networks.build([("dense", 3, 2)]), k, x)


@pytest.mark.parametrize("J", [1, 31, 32, 33, 100])
def test_packed_masks(J):
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(J)
    mask = torch.rand(3, 2, J, generator=gen) < 0.5
    words = snn.pack_allowed(mask)
    assert words.dtype == torch.int32 and words.shape == (3, 2, (J + 31) // 32)
    for j in range(J):
        assert torch.equal((words[..., j // 32] >> (j % 32) & 1).bool(), mask[..., j])


def test_the_optimizer_refuses_numbers_that_mean_nothing():
    import torch
    import snntc_amd as snn
    w = [torch.nn.Parameter(torch.ones(3))]
    for wrong in ({"max_norm": 0}, {"max_norm": -1.0}, {"max_norm": float("nan")}, {"seed": -1}, {"seed": 1 << 32}, {"state_bits": 16}):
        with pytest.raises(ValueError):
            snn.optim.AdamW(w, **wrong)


def test_a_copied_optimizer_keeps_its_numbers():
    import copy
    import pickle
    import snntc_amd as snn
    opt = snn.optim.AdamW([torch.nn.Parameter(torch.ones(3))], state_bits=8, max_norm=0.5, seed=9, capturable=True)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert (other.state_bits, other.max_norm, other.seed, other.capturable, other.norm) == (8, 0.5, 9, True, None)
        assert other.step(lambda: 3) == 3
        other.load_state_dict(opt.state_dict())


@pytest.mark.parametrize("ty,size", [(0, 4), (1, 2), (2, 2)])
def test_results_in_place_of_an_input_are_refused(lib, ty, size):
    """Several lanes or workgroups share the ends of rows, so a call in place would rule them twice."""
    at = lambda n: ctypes.c_void_p((1 << 30) + n)                                       # noqa: E731
    far, whole = at(1 << 33), 4 * 70000 * size
    for shift in (0, 2, -2, whole - 2, 2 - whole):
        assert lib.snntc_rule_times(at(0), ty, _rules(), at(shift), 4, 70000, None) == BAD
        assert b"overlaps" in lib.snntc_last_error()
        for grad, times in ((at(0), far), (far, at(0))):
            assert lib.snntc_rule_times_backward(grad, times, ty, _rules(), at(shift), 4, 70000, None) == BAD
            assert b"overlaps" in lib.snntc_last_error()
