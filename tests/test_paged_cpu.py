"""CPU tests around the paged-cache operators: frequencies of the rotary
scalings, the mirrors of the C structures, and the argument checks that come
before any device work."""

import ctypes
import math
import shutil
import subprocess

import pytest
import torch

from tests.test_abi_cpu import ROOT


@pytest.fixture(scope="module")
def lib():
    from turbopress_b200 import _abi, build
    build.build()
    return _abi.lib()


# -- frequencies ---------------------------------------------------------------

def test_plain_and_linear_frequencies():
    from turbopress_b200.rotary import rope_frequencies
    from turbopress_b200.step import rope_inv_freq
    inv, scale = rope_frequencies(128, 1e6)
    assert torch.equal(inv, rope_inv_freq(128, 1e6)) and scale == 1.0  # as the decode step's
    lin, scale = rope_frequencies(128, 1e6, dict(rope_type="linear", factor=4.0))
    assert torch.equal(lin, inv / 4.0) and scale == 1.0


def test_llama3_frequencies():
    """Wavelengths below original / high stay, above original / low stretch by
    the factor, and a linear ramp in turns joins them (formula restated)."""
    from turbopress_b200.rotary import rope_frequencies
    base, _ = rope_frequencies(128, 500000.0)
    inv, scale = rope_frequencies(128, 500000.0, dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                                      original_max_position_embeddings=8192))
    assert scale == 1.0
    for f, g in zip(base.tolist(), inv.tolist()):
        wave = 2 * math.pi / f
        if wave < 8192 / 4.0:
            want = f
        elif wave > 8192 / 1.0:
            want = f / 8.0
        else:
            s = (8192 / wave - 1.0) / (4.0 - 1.0)
            want = (1 - s) * f / 8.0 + s * f
        assert abs(g - want) <= 2e-6 * want


def test_yarn_frequencies():
    from turbopress_b200.rotary import rope_frequencies
    base, _ = rope_frequencies(128, 10000.0)
    inv, scale = rope_frequencies(128, 10000.0, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768))
    assert abs(scale - (0.1 * math.log(4.0) + 1.0)) < 1e-12
    lo = math.floor(128 * math.log(32768 / (32 * 2 * math.pi)) / (2 * math.log(10000.0)))
    hi = math.ceil(128 * math.log(32768 / (1 * 2 * math.pi)) / (2 * math.log(10000.0)))
    for i, (f, g) in enumerate(zip(base.tolist(), inv.tolist())):
        ramp = min(1.0, max(0.0, (i - lo) / (hi - lo)))
        want = f * (1 - ramp) + f / 4.0 * ramp
        assert abs(g - want) <= 2e-6 * want
    assert rope_frequencies(64, 1e4, dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=4096,
                                          attention_factor=1.5))[1] == 1.5


def test_frequency_refusals():
    from turbopress_b200.rotary import Rotary, rope_frequencies
    for bad in (lambda: rope_frequencies(63), lambda: rope_frequencies(0), lambda: rope_frequencies(64, 1e4, dict(type="dynamic")),
                lambda: Rotary(128, torch.tensor([1.0, float("nan")]), device="cpu"), lambda: Rotary(258, device="cpu"),
                lambda: Rotary(64, torch.ones(40), device="cpu")):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(KeyError):
        rope_frequencies(64, 1e4, dict(rope_type="llama3", factor=8.0))


def test_rotary_from_config():
    from types import SimpleNamespace

    from turbopress_b200.rotary import Rotary, rope_frequencies
    r = Rotary.from_config(SimpleNamespace(head_dim=128, hidden_size=2560, num_attention_heads=32, rope_theta=1e6), device="cpu")
    assert r.rot_dim == 128 and torch.equal(r.inv_freq, rope_frequencies(128, 1e6)[0])
    p = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192,
             rope_theta=5e5)
    r = Rotary.from_config(SimpleNamespace(head_dim=None, hidden_size=4096, num_attention_heads=32, rope_parameters=p,
                                           partial_rotary_factor=0.5), device="cpu")
    assert (r.head_dim, r.rot_dim) == (128, 64) and torch.equal(r.inv_freq, rope_frequencies(64, 5e5, p)[0])


def test_frequency_words():
    """64-bit fractions of a turn: within 2^-64 of the exact quotient, whole turns dropped."""
    from fractions import Fraction

    from turbopress_b200.rotary import Rotary
    inv = torch.tensor([1.0, 0.37, 1e-7, 12.0, -0.25])
    r = Rotary(10, inv, device="cpu")
    two_pi = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494")
    for f, w in zip(inv.tolist(), r.freq.tolist()):
        turns = Fraction(f) / two_pi
        gap = (Fraction(w % 2 ** 64, 2 ** 64) - turns) % 1
        assert min(gap, 1 - gap) <= Fraction(1, 2 ** 65)


# -- the C boundary --------------------------------------------------------------

def _structures():
    from turbopress_b200 import paged, rotary, speculative
    return {"tp_paged_cache": paged._PagedCache, "tp_rotary_args": rotary._RotaryArgs, "tp_paged_attn_args": paged._AttnArgs,
            "tp_evict_args": paged._EvictArgs, "tp_verify_args": speculative._VerifyArgs}


def test_structures_mirror_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("needs gcc")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "turbopress_b200.h"', "int main(void) {"]
    for name, s in _structures().items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for field, _ in s._fields_:
            lines.append(f'printf("{name}.{field} %zu\\n", offsetof({name}, {field}));')
    src = tmp_path / "sizes.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = tmp_path / "sizes"
    subprocess.run([gcc, "-I", str(ROOT / "include"), "-o", str(exe), str(src)], check=True)
    got = dict(ln.split() for ln in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for name, s in _structures().items():
        assert int(got[name]) == ctypes.sizeof(s), name
        for field, _ in s._fields_:
            assert int(got[f"{name}.{field}"]) == getattr(s, field).offset, (name, field)


def _cache(**over):
    from turbopress_b200.paged import _PagedCache
    base = dict(k_pages=4096, v_pages=8192, block_table=256, lengths=256, scores=256, positions=256, num_pages=8, page_stride=4096,
                head_stride=1024, token_stride=64, table_stride=4, batch=2, kv_heads=4, head_dim=64, page_size=16, max_pages=4,
                dtype=0)
    return _PagedCache(**{**base, **over})


CACHE_REFUSALS = [(dict(k_pages=None), "ARG"), (dict(lengths=None), "ARG"), (dict(batch=0), "ARG"), (dict(table_stride=3), "ARG"),
                  (dict(page_size=12), "UNSUPPORTED"), (dict(page_size=0), "UNSUPPORTED"), (dict(head_dim=60), "UNSUPPORTED"),
                  (dict(head_dim=264), "UNSUPPORTED"), (dict(dtype=1), "UNSUPPORTED"), (dict(page_stride=-8), "ARG"),
                  (dict(k_pages=4104), "ALIGN"), (dict(token_stride=68), "ALIGN"),
                  (dict(max_pages=1 << 27, table_stride=1 << 27), "UNSUPPORTED")]


@pytest.mark.parametrize("over,code", CACHE_REFUSALS)
def test_cache_refusals(lib, over, code):
    from turbopress_b200 import _abi
    want = getattr(_abi, "TP_ERR_" + code)
    c = ctypes.byref(_cache(**over))
    addr = ctypes.addressof(c._obj)
    assert lib.tp_paged_attn_workspace_bytes(addr, 1, 8, 0) == -want
    assert lib.tp_cache_evict_workspace_bytes(addr, 8) == -want
    assert lib.tp_last_error()


def test_call_refusals(lib):
    from turbopress_b200 import _abi
    from turbopress_b200.paged import _AttnArgs, _EvictArgs
    from turbopress_b200.rotary import _RotaryArgs
    from turbopress_b200.speculative import _VerifyArgs
    cache = _cache()
    ca = ctypes.addressof(cache)
    assert lib.tp_paged_attn_workspace_bytes(ca, 1, 6, 0) == -_abi.TP_ERR_ARG  # heads not a multiple
    assert lib.tp_paged_attn_workspace_bytes(ca, 0, 8, 0) == -_abi.TP_ERR_ARG
    need = lib.tp_paged_attn_workspace_bytes(ca, 1, 8, 1)
    assert need > lib.tp_paged_attn_workspace_bytes(ca, 1, 8, 0) > 0

    def attn(cache=cache, ws=1 << 20, n=need, **over):
        a = _AttnArgs(**{**dict(q=256, out=512, tokens=1, q_heads=8, softmax_scale=1.0, accumulate=1), **over})
        return lib.tp_paged_attn(ctypes.addressof(a), ctypes.addressof(cache), ws, n, None)
    assert attn(q=None) == _abi.TP_ERR_ARG
    assert attn(cache=_cache(scores=None)) == _abi.TP_ERR_ARG
    assert attn(q=264) == _abi.TP_ERR_ALIGN
    assert attn(n=need - 1) == _abi.TP_ERR_WORKSPACE and attn(ws=None) == _abi.TP_ERR_WORKSPACE

    def rotary(cache=None, **over):
        a = _RotaryArgs(**{**dict(q=256, k=256, q_out=256, k_out=256, positions=256, freq=256, tokens=2, seq=1, q_heads=8, kv_heads=4,
                                  head_dim=64, rot_dim=64, dtype=0, scale=1.0), **over})
        return lib.tp_rotary(ctypes.addressof(a), None if cache is None else ctypes.addressof(cache), None)
    assert lib.tp_rotary(None, None, None) == _abi.TP_ERR_ARG
    for over, code in ((dict(tokens=3, seq=2), "ARG"), (dict(head_dim=63), "UNSUPPORTED"), (dict(rot_dim=66), "UNSUPPORTED"),
                       (dict(head_dim=258, rot_dim=2), "UNSUPPORTED"), (dict(dtype=3), "ARG"), (dict(freq=None), "ARG"),
                       (dict(positions=None), "ARG"), (dict(k_out=None), "ARG"), (dict(q_heads=0, kv_heads=0), "ARG")):
        assert rotary(**over) == getattr(_abi, "TP_ERR_" + code), over
    assert rotary(tokens=0) == _abi.TP_OK
    assert rotary(cache=cache) == _abi.TP_ERR_ARG  # no v
    assert rotary(cache=cache, v=256, dtype=2) == _abi.TP_ERR_ARG  # another dtype than the pages'
    assert rotary(cache=cache, v=256, tokens=3) == _abi.TP_ERR_ARG

    ev = lib.tp_cache_evict_workspace_bytes(ca, 8)

    def evict(cache=cache, n=ev, **over):
        a = _EvictArgs(**{**dict(next_pos=256, new_lengths=256, new_scores=512, new_positions=512, budget=8, recent=2, sinks=2), **over})
        return lib.tp_cache_evict(ctypes.addressof(a), ctypes.addressof(cache), 1 << 20, n, None)
    for over, code in ((dict(budget=0), "ARG"), (dict(recent=7), "ARG"), (dict(recent=-1), "ARG"), (dict(new_scores=256), "ARG"),
                       (dict(new_positions=256), "ARG"), (dict(next_pos=None), "ARG")):
        assert evict(**over) == getattr(_abi, "TP_ERR_" + code), over
    assert evict(cache=_cache(positions=None)) == _abi.TP_ERR_ARG
    assert evict(n=ev - 1) == _abi.TP_ERR_WORKSPACE
    assert lib.tp_cache_evict_workspace_bytes(ctypes.addressof(_cache(max_pages=1 << 16, table_stride=1 << 16)), 8) == \
        -_abi.TP_ERR_UNSUPPORTED

    vb = lib.tp_verify_workspace_bytes(2, 3, 100)
    assert vb > 0 and lib.tp_verify_workspace_bytes(0, 3, 100) == -_abi.TP_ERR_ARG
    assert lib.tp_verify_workspace_bytes(2, 64, 100) == -_abi.TP_ERR_UNSUPPORTED
    assert lib.tp_verify_workspace_bytes(40000, 3, 100) == -_abi.TP_ERR_UNSUPPORTED

    def verify(n=vb, **over):
        a = _VerifyArgs(**{**dict(logits=256, batch_stride=400, row_stride=100, draft_tokens=256, uniforms=256, noise=256,
                                  temperature=256, accepted=256, tokens=256, batch=2, drafts=3, vocab=100, dtype=0), **over})
        return lib.tp_verify_drafts(ctypes.addressof(a), 1 << 20, n, None)
    for over, code in ((dict(logits=None), "ARG"), (dict(draft_tokens=None), "ARG"), (dict(noise=None), "ARG"),
                       (dict(uniforms=None), "ARG"), (dict(dtype=7), "ARG"), (dict(logits=257), "ALIGN")):
        assert verify(**over) == getattr(_abi, "TP_ERR_" + code), over
    assert verify(n=vb - 1) == _abi.TP_ERR_WORKSPACE


def test_classes_need_cuda():
    from turbopress_b200.paged import PagedKVCache
    with pytest.raises(RuntimeError):
        PagedKVCache(1, 1, 64, 2, 16, 2, device="cpu")
