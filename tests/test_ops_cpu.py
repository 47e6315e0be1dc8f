"""CPU tests of the step operators: refusals of their Python and C entries and
the rotary frequencies."""

import ctypes as C
import math

import pytest
import torch

import stickykv_b200 as skv
from stickykv_b200 import _lib
from stickykv_b200._lib import RotaryArgs, SampleArgs, WindowArgs


# -- Python entries -----------------------------------------------------------------------

def _rotary(**kw):
    a = dict(query=torch.zeros(2, 4, 3, 16), key=torch.zeros(2, 2, 3, 16),
             positions=torch.arange(3), inv_freq=torch.ones(8))
    extra = {k: kw.pop(k) for k in ("out", "interleaved", "inverse") if k in kw}
    a.update(kw)
    return skv.apply_rotary(a["query"], a["key"], a["positions"], a["inv_freq"], **extra)


@pytest.mark.parametrize("kw, error", [
    (dict(query=torch.zeros(4, 3, 16)), ValueError),
    (dict(key=torch.zeros(2, 2, 4, 16)), ValueError),
    (dict(key=torch.zeros(1, 2, 3, 16)), ValueError),
    (dict(query=torch.zeros(2, 4, 3, 16, dtype=torch.float64)), NotImplementedError),
    (dict(key=torch.zeros(2, 2, 3, 16, dtype=torch.float16)), NotImplementedError),
    (dict(inv_freq=torch.ones(9)), ValueError),
    (dict(inv_freq=torch.ones(0)), ValueError),
    (dict(inv_freq=torch.ones(8, dtype=torch.float64)), ValueError),
    (dict(positions=torch.arange(4)), ValueError),
    (dict(positions=torch.zeros(3, 3, dtype=torch.long)), ValueError),
    (dict(positions=torch.zeros(3)), ValueError),
    (dict(out=(torch.zeros(2, 4, 3, 16), None)), ValueError),
    (dict(out=(torch.zeros(2, 4, 3, 8), torch.zeros(2, 2, 3, 16))), ValueError),
    (dict(out=(torch.zeros(1, 4, 3, 16).expand(2, 4, 3, 16), torch.zeros(2, 2, 3, 16))), ValueError),
    (dict(query=torch.zeros(2, 4, 3, 16, requires_grad=True)), NotImplementedError),
    (dict(), RuntimeError),  # no CPU path
])
def test_rotary_refusals(kw, error):
    with pytest.raises(error):
        _rotary(**kw)


def test_rotary_refuses_outputs_that_overlap():
    q, k = torch.zeros(2, 4, 3, 16), torch.zeros(2, 2, 3, 16)
    base = torch.zeros(2 * 4 * 3 * 16 + 8)
    q2, shifted = base[:-8].view(2, 4, 3, 16), base[8:].view(2, 4, 3, 16)
    with pytest.raises(ValueError, match="overlaps"):
        _rotary(query=q2, key=k, out=(shifted, torch.zeros_like(k)))
    with pytest.raises(ValueError, match="overlap"):  # the keys' place is not the queries' output
        _rotary(query=k, key=k.clone(), out=(k, k))
    with pytest.raises(RuntimeError, match="no CPU path"):  # in place is fine
        _rotary(query=q, key=k, out=(q, k))


def test_outputs_that_begin_where_another_tensor_does_are_refused():
    """Slices with gaps: an output over the other input, over its own input in
    another order, and both outputs in one place."""
    buf = torch.zeros(2, 3, 8, 16)
    q, k = buf[:, :, :2].transpose(1, 2), buf[:, :, 2:4].transpose(1, 2)
    for out in ((k, q), (q, q), (buf.view(2, 4, 6, 16)[:, :2, :3], k)):
        with pytest.raises(ValueError, match="overlap"):
            _rotary(query=q, key=k, out=out)
    with pytest.raises(ValueError, match="overlaps"):
        _window(query=buf[:1, :, :4].transpose(1, 2), key=torch.zeros(1, 2, 9, 16), value=torch.zeros(1, 2, 9, 16),
                out=buf.view(-1)[:3 * 4 * 16].view(1, 3, 4, 16))
    with pytest.raises(RuntimeError, match="no CPU path"):
        _rotary(query=q, key=k, out=(q, k))


def _window(**kw):
    a = dict(query=torch.zeros(2, 4, 3, 16), key=torch.zeros(2, 2, 9, 16), value=torch.zeros(2, 2, 9, 16), window=4)
    a.update(kw)
    return skv.sink_window_attention(a.pop("query"), a.pop("key"), a.pop("value"), **a)


@pytest.mark.parametrize("kw, error", [
    (dict(query=torch.zeros(4, 3, 16)), ValueError),
    (dict(value=torch.zeros(2, 2, 8, 16)), ValueError),
    (dict(query=torch.zeros(3, 4, 3, 16)), ValueError),
    (dict(query=torch.zeros(2, 5, 3, 16)), ValueError),
    (dict(query=torch.zeros(2, 4, 3, 16, dtype=torch.float16)), NotImplementedError),
    (dict(query=torch.zeros(2, 4, 3, 24), key=torch.zeros(2, 2, 9, 24), value=torch.zeros(2, 2, 9, 24)),
     NotImplementedError),
    (dict(window=0), ValueError),
    (dict(sinks=-1), ValueError),
    (dict(starts=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(ends=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(query_slots=torch.zeros(4, dtype=torch.int32)[::2]), ValueError),
    (dict(out=torch.zeros(2, 4, 3, 16)), ValueError),
    (dict(query=torch.zeros(2, 4, 3, 16, requires_grad=True)), NotImplementedError),
    (dict(), RuntimeError),
])
def test_window_refusals(kw, error):
    with pytest.raises(error):
        _window(**kw)


def test_window_refuses_an_output_over_an_input():
    q = torch.zeros(2, 4, 3, 16)
    with pytest.raises(ValueError, match="overlaps"):
        _window(query=q, out=q.view(2, 3, 4, 16))


def _sample(**kw):
    a = dict(logits=torch.zeros(2, 5), uniform=torch.zeros(2))
    a.update(kw)
    return skv.sample_tokens(a.pop("logits"), a.pop("uniform"), **a)


@pytest.mark.parametrize("kw, error", [
    (dict(logits=torch.zeros(5)), ValueError),
    (dict(logits=torch.zeros(2, 0)), ValueError),
    (dict(logits=torch.zeros(2, 5, dtype=torch.float64)), NotImplementedError),
    (dict(uniform=torch.zeros(3)), ValueError),
    (dict(uniform=torch.zeros(2, dtype=torch.float64)), ValueError),
    (dict(temperature=-0.5), ValueError),
    (dict(temperature=math.inf), ValueError),
    (dict(temperature=math.nan), ValueError),
    (dict(temperature=torch.ones(2, dtype=torch.float64)), ValueError),
    (dict(top_k=-1), ValueError),
    (dict(top_k=torch.ones(2, dtype=torch.int64)), ValueError),
    (dict(top_p=0.0), ValueError),
    (dict(top_p=1.5), ValueError),
    (dict(top_p=torch.ones(3)), ValueError),
    (dict(min_p=-0.1), ValueError),
    (dict(min_p=1.1), ValueError),
    (dict(out=torch.zeros(2)), ValueError),
    (dict(out=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(logits=torch.zeros(2, 5, requires_grad=True)), NotImplementedError),
    (dict(), RuntimeError),
])
def test_sample_refusals(kw, error):
    with pytest.raises(error):
        _sample(**kw)


@pytest.mark.parametrize("name", ["temperature", "top_p", "min_p"])
def test_sample_refuses_gradients_of_settings(name):
    with pytest.raises(NotImplementedError, match="no backward"):
        _sample(**{name: torch.full((2,), 0.5, requires_grad=True)})


@pytest.mark.parametrize("call, kw, error", [
    (_rotary, dict(inverse=torch.ones(2)), RuntimeError), (_window, dict(window=4.0), TypeError), (_window, dict(sinks=1.5), TypeError),
    (_window, dict(window=torch.tensor(4.0)), TypeError), (_window, dict(scaling="x"), ValueError),
    (_window, dict(scaling=torch.tensor(0.5, requires_grad=True)), NotImplementedError),
    (_sample, dict(top_k=2.0), TypeError), (_sample, dict(temperature="x"), ValueError),
    (_sample, dict(top_p=torch.tensor(0.5)), ValueError),
])
def test_settings_are_numbers(call, kw, error):
    with pytest.raises(error):
        call(**kw)


@pytest.mark.parametrize("call, name, x", [
    (_rotary, "query", torch.zeros(2, 4, 3, 16)), (_rotary, "key", torch.zeros(2, 2, 3, 16)), (_rotary, "inv_freq", torch.ones(8)),
    (_window, "query", torch.zeros(2, 4, 3, 16)), (_window, "value", torch.zeros(2, 2, 9, 16)), (_window, "scaling", torch.tensor(0.5)),
    (_sample, "logits", torch.zeros(2, 5)), (_sample, "temperature", torch.ones(2)), (_sample, "uniform", torch.zeros(2)),
])
def test_tangents_are_refused(call, name, x):
    """Forward-mode derivatives, which would be dropped."""
    from torch.autograd import forward_ad
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="no derivative"):
        call(**{name: forward_ad.make_dual(x, torch.ones_like(x))})
    with pytest.raises(NotImplementedError, match="no derivative"):
        torch.func.jvp(lambda y: call(**{name: y}), (x,), (torch.ones_like(x),))
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no CPU path"):
        call()


# -- C entries: every refusal comes before anything is launched ---------------------------

_P = 1 << 20  # an aligned address that nothing reads


def _rotary_args(**kw):
    a = RotaryArgs(2, 3, 4, 2, 16, 16, 0, 0, _lib.SKV_F16, 1.0, _P, _P, _P, _P)
    for name in ("q_stride", "k_stride", "q_out_stride", "k_out_stride"):
        setattr(a, name, (C.c_int64 * 3)(192, 48, 16))
    a.positions, a.inv_freq, a.position_stride = _P, _P, (C.c_int64 * 2)(0, 1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, status", [
    (dict(batch=0), 1), (dict(tokens=-1), 1), (dict(num_q_heads=0), 1), (dict(rotary_dim=15), 1),
    (dict(rotary_dim=0), 1), (dict(rotary_dim=18), 1), (dict(q=None), 1), (dict(q_out=None), 1),
    (dict(k_out=None), 1), (dict(num_kv_heads=0), 1), (dict(k=None), 1), (dict(positions=None), 1),
    (dict(inv_freq=None), 1), (dict(dtype=7), 2), (dict(q=_P + 1), 3), (dict(positions=_P + 4), 3),
])
def test_rotary_c_refusals(kw, status):
    assert _lib.lib().skv_rotary(C.byref(_rotary_args(**kw)), None) == status
    assert _lib.lib().skv_rotary(None, None) == 1


def _window_args(**kw):
    a = WindowArgs(2, 3, 9, 4, 2, 16, _lib.SKV_F16, 4, 1, 1.0, _P, _P, _P, _P)
    for name in ("q_stride", "k_stride", "v_stride"):
        setattr(a, name, (C.c_int64 * 3)(288, 144, 16))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, status", [
    (dict(batch=0), 1), (dict(q_tokens=0), 1), (dict(k_slots=0), 1), (dict(num_q_heads=5), 1), (dict(window=0), 1),
    (dict(sinks=-1), 1), (dict(q=None), 1), (dict(v=None), 1), (dict(out=None), 1), (dict(head_dim=24), 2),
    (dict(dtype=9), 2), (dict(batch=1 << 17), 2), (dict(k=_P + 8), 3), (dict(starts=_P + 2), 3),
    (dict(k_stride=(C.c_int64 * 3)(288, 144, 20)), 3), (dict(q_stride=(C.c_int64 * 3)(-16, 144, 16)), 1),
])
def test_window_c_refusals(kw, status):
    L = _lib.lib()
    assert L.skv_window_attention(C.byref(_window_args(**kw)), None) == status
    assert L.skv_window_attention(None, None) == 1


@pytest.mark.parametrize("kw", [
    dict(q_tokens=(1 << 29) + 1), dict(k_slots=(1 << 29) + 1), dict(q_tokens=1 << 29, num_q_heads=8),
])
def test_window_c_refuses_what_31_bits_do_not_hold(kw):
    assert _lib.lib().skv_window_attention(C.byref(_window_args(**kw)), None) == 2


@pytest.mark.parametrize("kw, status", [
    (dict(batch=0), 1), (dict(vocabulary=0), 1), (dict(logits=None), 1), (dict(uniform=None), 1),
    (dict(tokens=None), 1), (dict(row_stride=-1), 1), (dict(dtype=5), 2), (dict(vocabulary=(1 << 22) + 1), 2),
    (dict(logits=_P + 1), 3),
    (dict(tokens=_P + 4), 3), (dict(top_ps=_P + 2), 3),
])
def test_sample_c_refusals(kw, status):
    a = SampleArgs(2, 5, _lib.SKV_F16, 0, 1.0, 1.0, 0.0, 0, _P, 5, _P, None, None, None, None, _P)
    for k, v in kw.items():
        setattr(a, k, v)
    assert _lib.lib().skv_sample(C.byref(a), None) == status
    assert _lib.lib().skv_sample(None, None) == 1


def test_struct_sizes():
    L = _lib.lib()
    for i, st in ((3, RotaryArgs), (4, WindowArgs), (5, SampleArgs)):
        assert L.skv_struct_size(i) == C.sizeof(st)


# -- frequencies ---------------------------------------------------------------------------

SCALINGS = [
    None,
    {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 512},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 512},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 512},
    {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 4096, "beta_fast": 24.0, "beta_slow": 2.0,
     "attention_factor": 1.25},
]


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("dim, theta", [(64, 10000.0), (128, 500000.0)])
def test_frequencies_are_those_of_transformers(scaling, dim, theta):
    """transformers computes them in float32: every step is off by at most 2^-24
    relative, and pow's exponent error grows with ln(theta) * i (under 14 * 2^-24);
    32 such steps bound both."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    seq_len = 2000
    inv, scale = skv.rotary_frequencies(dim, theta, scaling, seq_len=seq_len)
    assert inv.dtype == torch.float32 and inv.shape == (dim // 2,)
    if scaling is None:
        want, want_scale = 1.0 / theta ** (torch.arange(0, dim, 2).double() / dim), 1.0
    else:
        params = dict(scaling, rope_theta=theta)
        original = scaling.get("original_max_position_embeddings", 512)
        cfg = LlamaConfig(hidden_size=dim * 2, num_attention_heads=2, head_dim=dim, max_position_embeddings=original,
                          rope_parameters=params)
        want, want_scale = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, torch.device("cpu"), seq_len=seq_len)
    assert torch.allclose(inv.double(), want.double(), rtol=32 * 2.0 ** -24, atol=0)
    assert scale == pytest.approx(want_scale, rel=1e-6)


@pytest.mark.parametrize("kw, error", [
    (dict(rotary_dim=7), ValueError), (dict(rotary_dim=0), ValueError), (dict(theta=0.0), ValueError),
    (dict(scaling={"rope_type": "linear"}), ValueError),
    (dict(scaling={"rope_type": "linear", "factor": -1.0}), ValueError),
    (dict(scaling={"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0,
                   "original_max_position_embeddings": 512}), ValueError),
    (dict(scaling={"rope_type": "longrope", "factor": 2.0}), NotImplementedError),
])
def test_frequency_refusals(kw, error):
    a = dict(rotary_dim=64, theta=10000.0, scaling=None)
    a.update(kw)
    with pytest.raises(error):
        skv.rotary_frequencies(**a)


_YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}


@pytest.mark.parametrize("scaling", [
    dict(_YARN, mscale=1.0, mscale_all_dim=1.0), dict(_YARN, mscale=0.707, mscale_all_dim=1.0),
    dict(_YARN, mscale=1.0, mscale_all_dim=0.707), dict(_YARN, mscale=0.707), dict(_YARN, mscale_all_dim=0.707),
    dict(_YARN, mscale=0.0, mscale_all_dim=1.0), dict(_YARN, mscale=1.0, mscale_all_dim=0.707, attention_factor=1.1),
    dict(_YARN, factor=1.0, mscale=0.5, mscale_all_dim=1.0), dict(_YARN, attention_factor=None, mscale=2.0, mscale_all_dim=0.5),
    dict(_YARN, beta_fast=16.0, truncate=False), dict(_YARN, truncate=None), dict(_YARN, beta_fast=None), {"rope_type": "default"},
    {"rope_type": "linear", "factor": 4.0, "original_max_position_embeddings": 512},
])
def test_frequencies_of_whole_dicts_are_those_of_transformers(scaling):
    """Dicts as a configuration holds them, theta among them; bounds as above."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    dim = 64
    original = scaling.get("original_max_position_embeddings", 512)
    params = dict(scaling, rope_theta=500000.0)
    cfg = LlamaConfig(hidden_size=2 * dim, num_attention_heads=2, head_dim=dim, max_position_embeddings=original,
                      rope_parameters=params)
    if scaling["rope_type"] == "default":
        want, want_scale = 1.0 / 500000.0 ** (torch.arange(0, dim, 2).double() / dim), 1.0
    else:
        want, want_scale = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, torch.device("cpu"))
    for inv, scale in (skv.rotary_frequencies(dim, scaling=params), skv.rotary_frequencies(dim, 500000.0, params),
                       skv.rotary_frequencies(dim, 500000.0, scaling), skv.rotary_frequencies(dim, scaling=cfg.rope_parameters)):
        assert torch.allclose(inv.double(), want.double(), rtol=32 * 2.0 ** -24, atol=0)
        assert scale == pytest.approx(want_scale, rel=1e-6)


def test_default_theta():
    for args in ((), (None,), (10000,), (None, {}), (None, {"rope_theta": None})):
        assert torch.equal(skv.rotary_frequencies(64, *args)[0], skv.rotary_frequencies(64, 10000.0)[0])


@pytest.mark.parametrize("theta, scaling, error", [
    (10000.0, {"rope_type": "default", "rope_theta": 500000.0}, ValueError),
    (None, {"rope_theta": -1.0}, ValueError),
    (None, {"rope_type": "default", "partial_rotary_factor": 0.5}, ValueError),
    (None, {"rope_type": "dynamic", "factor": 1.0, "original_max_position_embeddings": 512, "alpha": 1000.0}, NotImplementedError),
    (None, dict(_YARN, some_factor=2.0), NotImplementedError),
    (None, dict(_YARN, mscale=-1.0, mscale_all_dim=1.0), ValueError),
    (None, dict(_YARN, mscale=1.0, mscale_all_dim=math.nan), ValueError),
])
def test_frequency_dicts_that_are_refused(theta, scaling, error):
    with pytest.raises(error):
        skv.rotary_frequencies(64, theta, scaling)
