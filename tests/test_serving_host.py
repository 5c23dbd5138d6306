"""The serving ops without a GPU: argument structures against the header, refusals of the Python ops and of the C
entry points before any device is touched."""
import shutil
import struct
import subprocess
from pathlib import Path

import pytest
import torch

import kernelfuser_amd as kf
from kernelfuser_amd import _lib
from serving_ref import attention, logprobs, quantise

ROOT = Path(__file__).resolve().parent.parent
BF16, E4M3, E8M0 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
P = 1 << 20  # a fake aligned address that no check dereferences


# ---------------------------------------------------------------------------
# structures
# ---------------------------------------------------------------------------

FIELDS = {
    "kfmi_cache_write_args": ("CACHE_WRITE_ARGS", "q_stride B eps norm_style reserved"),
    "kfmi_decode_args": ("DECODE_ARGS", "work_bytes q_stride cache_stride pages_stride B window scale cache_type"),
    "kfmi_cache_read_args": ("CACHE_READ_ARGS", "cache_stride pages_stride B cache_type"),
    "kfmi_logprobs_args": ("LOGPROBS_ARGS", "work_bytes logits_stride ids_stride N0 V top reserved"),
}
# offsets of those fields as the packing formats of _lib lay them out
OFFSETS = {
    "kfmi_cache_write_args": [15 * 8, 33 * 8, 41 * 8, 42 * 8, 42 * 8 + 12],
    "kfmi_decode_args": [9 * 8, 10 * 8, 13 * 8, 18 * 8, 20 * 8, 28 * 8, 29 * 8, 31 * 8],
    "kfmi_cache_read_args": [8 * 8, 13 * 8, 15 * 8, 22 * 8],
    "kfmi_logprobs_args": [7 * 8, 8 * 8, 10 * 8, 12 * 8, 14 * 8, 15 * 8, 15 * 8 + 12],
}


def test_structures_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "kfmi.h"', "int main(void) {"]
    for name, (_, fields) in FIELDS.items():
        args = ", ".join([f"sizeof({name})"] + [f"offsetof({name}, {f})" for f in fields.split()])
        lines.append(f'  printf("{name}{" %zu" * (1 + len(fields.split()))}\\n", {args});')
    src = tmp_path / "s.c"
    src.write_text("\n".join(lines + ["  return 0;", "}", ""]))
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", "-I", str(ROOT / "include"), str(src), "-o",
                    str(tmp_path / "s")], check=True, timeout=120)
    out = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True, timeout=60).stdout
    for line in out.splitlines():
        name, size, *offs = line.split()
        fmt = getattr(_lib, FIELDS[name][0])
        assert fmt.size == int(size) and [int(o) for o in offs] == OFFSETS[name], name


def test_constants_match_the_header():
    import re

    from kernelfuser_amd import serving
    text = (ROOT / "include" / "kfmi.h").read_text()

    def value(name):
        return int(re.search(rf"#define {name} (\d+)", text).group(1))

    assert serving.COUNTER_BYTES == value("KFMI_DECODE_COUNTER_BYTES") == value("KFMI_LOGPROBS_COUNTER_BYTES")
    assert _lib.LOGPROBS_TOP_MAX == value("KFMI_LOGPROBS_TOP_MAX")
    assert (_lib.CACHE_BF16, _lib.CACHE_E4M3) == (value("KFMI_CACHE_BF16"), value("KFMI_CACHE_E4M3"))
    for n in ("POSITIONS", "SLOTS", "PAGES", "LENGTHS", "IDS"):
        assert getattr(_lib, "I64_" + n) == value("KFMI_I64_" + n)
    for t, n in ((torch.float32, "F32"), (BF16, "BF16"), (torch.float16, "F16")):
        assert _lib.LOGITS_TYPES[t] == value("KFMI_LOGITS_" + n)


# ---------------------------------------------------------------------------
# C entry points
# ---------------------------------------------------------------------------

def _write(**over):
    a = dict(q=P, k=P, v=P, gq=P, gk=P, cos=P, sin=P, positions=P, slots=P, qn=P, kn=0, kc=P, vc=P, ks=0, vs=0,
             qs=(4096, 128, 128), kst=(1024, 128, 128), vst=(1024, 128, 128), ps=(1, 1), ss=(1, 1),
             cs=(8192, 1024, 128), es=(0, 0), B=2, Hq=8, Hkv=2, S=1, D=128, rows=64, pages=4, page=16, eps=1e-6,
             style=0, kind=0, flags=0)
    a.update(over)
    return _lib.CACHE_WRITE_ARGS.pack(*(a[n] for n in "q k v gq gk cos sin positions slots qn kn kc vc ks vs".split()),
                                      *a["qs"], *a["kst"], *a["vst"], *a["ps"], *a["ss"], *a["cs"], *a["es"],
                                      *(a[n] for n in "B Hq Hkv S D rows pages page eps style kind flags".split()), 0)


def _dec(**over):
    a = dict(q=P, kc=P, vc=P, ks=0, vs=0, pages=P, lengths=P, out=P, work=0, wb=0, qs=(1024, 128, 128),
             cs=(8192, 1024, 128), es=(0, 0), pst=4, lst=1, B=2, Hq=8, Hkv=2, S=1, D=128, num=4, page=16, max=4,
             window=0, scale=0.1, cap=0.0, kind=0, flags=0)
    a.update(over)
    return _lib.DECODE_ARGS.pack(*(a[n] for n in "q kc vc ks vs pages lengths out work wb".split()), *a["qs"], *a["cs"],
                                 *a["es"], *(a[n] for n in "pst lst B Hq Hkv S D num page max window scale cap kind "
                                             "flags".split()))


def _read(**over):
    a = dict(kc=P, vc=P, ks=0, vs=0, pages=P, lengths=P, k=P, v=P, cs=(8192, 1024, 128), es=(0, 0), pst=4, lst=1, B=2,
             Hkv=2, L=16, D=128, num=4, page=16, max=4, kind=0, flags=0)
    a.update(over)
    return _lib.CACHE_READ_ARGS.pack(*(a[n] for n in "kc vc ks vs pages lengths k v".split()), *a["cs"], *a["es"],
                                     *(a[n] for n in "pst lst B Hkv L D num page max kind flags".split()))


def _lp(**over):
    a = dict(logits=P, ids=P, lp=P, h=P, tl=P, ti=P, work=0, wb=0, ls=(0, 100), ist=(0, 1), n0=1, n1=2, v=100, top=3,
             kind=0, flags=0)
    a.update(over)
    return _lib.LOGPROBS_ARGS.pack(*(a[n] for n in "logits ids lp h tl ti work wb".split()), *a["ls"], *a["ist"],
                                   *(a[n] for n in "n0 n1 v top kind flags".split()), 0)


WRITE, DECODE, READ, LOGPROBS = ("kfmi_norm_rope_to_cache_bf16", "kfmi_attention_decode_bf16",
                                 "kfmi_cache_to_dense_bf16", "kfmi_token_logprobs")
REFUSED = [
    (WRITE, _write, dict(B=0), ">= 1"), (WRITE, _write, dict(D=64), "D must be"),
    (WRITE, _write, dict(Hq=7), "multiple of Hkv"), (WRITE, _write, dict(style=5), "norm_style"),
    (WRITE, _write, dict(B=1, Hq=2 ** 16, Hkv=2 ** 16), "65535"), (READ, _read, dict(B=1, Hkv=2 ** 16), "65535"),
    (WRITE, _write, dict(B=2 ** 20, S=2 ** 12), "2^31"), (WRITE, _write, dict(B=2 ** 40, S=2 ** 40), "2^31"),
    (WRITE, _write, dict(flags=4), "index_flags"), (WRITE, _write, dict(k=0), "k must not"),
    (WRITE, _write, dict(qn=0), "qn must not"), (WRITE, _write, dict(v=P + 8), "v must be 16"),
    (WRITE, _write, dict(kst=(1024, 132, 128)), "k strides"), (WRITE, _write, dict(qs=(4, 8, 8)), "q strides"),
    (WRITE, _write, dict(sin=0), "both rotary"), (WRITE, _write, dict(positions=0), "positions must not"),
    (WRITE, _write, dict(positions=P + 4, flags=1), "positions must be 8"), (WRITE, _write, dict(slots=P + 2), "slots"),
    (WRITE, _write, dict(rows=0), "table_rows"), (WRITE, _write, dict(kc=0), "k_cache must not"),
    (WRITE, _write, dict(page=24), "page_size"), (WRITE, _write, dict(page=8), "page_size"),
    (WRITE, _write, dict(pages=0), "num_pages"), (WRITE, _write, dict(kind=2), "cache_type"),
    (WRITE, _write, dict(ks=P), "no scales"), (WRITE, _write, dict(kind=1), "k_scale must not"),
    (WRITE, _write, dict(kind=1, ks=P, vs=P + 2), "v_scale must be 4"),
    (WRITE, _write, dict(kind=1, ks=P, vs=P, cs=(8192, 1024, 136)), "cache strides"),
    (WRITE, _write, dict(kind=1, ks=P, vs=P, es=(34, 16)), "scale strides"),
    (WRITE, _write, dict(eps=-1.0), "eps"), (WRITE, _write, dict(eps=float("nan")), "eps"),
    (DECODE, _dec, dict(S=17), "at most 16"), (DECODE, _dec, dict(S=0), ">= 1"), (DECODE, _dec, dict(q=0), "q must not"),
    (DECODE, _dec, dict(Hq=9), "multiple of Hkv"), (DECODE, _dec, dict(max=0), "max_pages"),
    (DECODE, _dec, dict(B=65535, Hkv=64, Hq=64, max=2 ** 14), "too large"), (DECODE, _dec, dict(cs=(8192, 1024, 2 ** 24)), "tokens"),
    (DECODE, _dec, dict(cs=(-8192, 1024, 128)), "cache strides"),
    (DECODE, _dec, dict(max=2 ** 40), "2^30 keys"), (DECODE, _dec, dict(B=70000), "65535"),
    (DECODE, _dec, dict(flags=16), "index_flags"), (DECODE, _dec, dict(pages=0), "pages must not"),
    (DECODE, _dec, dict(lengths=P + 4, flags=8), "lengths must be 8"), (DECODE, _dec, dict(scale=0.0), "scale"),
    (DECODE, _dec, dict(cap=-1.0), "softcap"), (DECODE, _dec, dict(cap=float("nan")), "softcap"),
    (DECODE, _dec, dict(window=-1), "window"), (DECODE, _dec, dict(wb=-1), "work_bytes"),
    (DECODE, _dec, dict(work=P + 4, wb=100), "work must be"), (DECODE, _dec, dict(vc=P + 2), "v_cache must be"),
    (DECODE, _dec, dict(qs=(1, 8, 8)), "q strides"), (DECODE, _dec, dict(num=2 ** 31), "num_pages"),
    (READ, _read, dict(L=0), ">= 1"), (READ, _read, dict(L=2 ** 31), "2^31"), (READ, _read, dict(k=0), "k must not"),
    (READ, _read, dict(pages=P + 2), "pages must be 4"), (READ, _read, dict(B=65536), "65535"),
    (READ, _read, dict(max=2 ** 31), "2^30 keys"),
    (LOGPROBS, _lp, dict(v=0), ">= 1"), (LOGPROBS, _lp, dict(v=2 ** 30), "2^30"), (LOGPROBS, _lp, dict(n1=2 ** 26), "2^25"),
    (LOGPROBS, _lp, dict(top=33), "top must"), (LOGPROBS, _lp, dict(top=-1), "top must"),
    (LOGPROBS, _lp, dict(v=2), "top must"), (LOGPROBS, _lp, dict(kind=3), "logits_type"),
    (LOGPROBS, _lp, dict(flags=1), "index_flags"), (LOGPROBS, _lp, dict(logits=P + 2), "logits must be 4"),
    (LOGPROBS, _lp, dict(logits=P + 1, kind=1), "logits must be 2"), (LOGPROBS, _lp, dict(ti=0), "top_ids"),
    (LOGPROBS, _lp, dict(h=0), "entropy"), (LOGPROBS, _lp, dict(work=P, wb=-5), "work_bytes"),
]


@pytest.mark.parametrize("name,make,over,fragment", REFUSED, ids=[f"{r[0][5:]}-{i}" for i, r in enumerate(REFUSED)])
def test_c_refusals(name, make, over, fragment):
    lib = _lib.load()
    assert getattr(lib, name)(make(**over), None) == _lib.KFMI_EINVAL
    assert fragment in lib.kfmi_last_error().decode()
    assert lib.kfmi_last_launches(None, 0) == 0


def test_c_null_arguments():
    lib = _lib.load()
    for name in (WRITE, DECODE, READ, LOGPROBS):
        assert getattr(lib, name)(None, None) == _lib.KFMI_EINVAL
    for name, make in (("kfmi_attention_decode_workspace", _dec), ("kfmi_token_logprobs_workspace", _lp)):
        assert getattr(lib, name)(make(), None) == _lib.KFMI_EINVAL
        import ctypes
        got = ctypes.c_int64(-1)
        assert getattr(lib, name)(make(), ctypes.byref(got)) == _lib.KFMI_OK and got.value >= 0
        assert getattr(lib, name)(None, ctypes.byref(got)) == _lib.KFMI_EINVAL


# ---------------------------------------------------------------------------
# Python ops (CPU tensors: a call that is right stops at the device rule)
# ---------------------------------------------------------------------------

def _cpu_cache(dtype=BF16, pages=4, hk=2, page=16, d=128):
    return list(kf.make_cache(pages, hk, page, d, dtype, "cpu"))


def _append_args(**over):
    a = dict(q=torch.zeros(1, 4, 3, 128, dtype=BF16), k=torch.zeros(1, 2, 3, 128, dtype=BF16),
             v=torch.zeros(1, 2, 3, 128, dtype=BF16), gq=torch.ones(128, dtype=BF16), gk=torch.ones(128, dtype=BF16),
             cos=torch.ones(9, 128, dtype=BF16), sin=torch.ones(9, 128, dtype=BF16),
             positions=torch.arange(3).view(1, 3), slots=torch.arange(3).view(1, 3), cache=_cpu_cache(), kw={})
    a.update(over)
    return [a[n] for n in "q k v gq gk cos sin positions slots".split()] + a["cache"], a["kw"]


def _z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("over,match", [
    (dict(), "GPU device"), (dict(q=None, gq=None), "GPU device"), (dict(cache=_cpu_cache(E4M3)), "GPU device"),
    (dict(kw=dict(norm_style="x")), "norm_style"), (dict(sin=None), "both rotary"), (dict(gk=None), "Expected k, v and gk"),
    (dict(k=_z(1, 2, 3, 128).requires_grad_()), "forward-only"), (dict(v=_z(1, 2, 4, 128)), r"Expected q \[B"),
    (dict(q=_z(2, 4, 3, 128)), r"Expected q \[B"), (dict(q=_z(1, 3, 3, 128)), "multiple of Hkv"),
    (dict(k=_z(1, 2, 3, 64), v=_z(1, 2, 3, 64), q=_z(1, 4, 3, 64)), "D in"),
    (dict(q=_z(1, 4, 3, 128, dtype=torch.float16)), "BF16"), (dict(gq=torch.ones(64, dtype=BF16)), "gamma"),
    (dict(slots=torch.arange(3)), "slots"), (dict(slots=torch.zeros(1, 3)), "slots must be int32"),
    (dict(positions=None), "positions"), (dict(positions=torch.zeros(1, 3)), "positions must be int32"),
    (dict(cos=torch.ones(9, 64, dtype=BF16)), "rotary tables"), (dict(cos=torch.ones(128, 9, dtype=BF16).t(),
                                                                     sin=torch.ones(128, 9, dtype=BF16).t()), "contiguous"),
    (dict(cache=_cpu_cache(hk=4)), "Hkv and D"), (dict(cache=_cpu_cache(d=256)), "Hkv and D"),
    (dict(cache=_cpu_cache(E4M3)[:2] + [None, None]), "needs k_scale"),
    (dict(cache=_cpu_cache()[:2] + _cpu_cache(E4M3)[2:]), "no scales"),
    (dict(cache=[t.float() for t in _cpu_cache()[:2]] + [None, None]), "bfloat16 or float8"),
    (dict(cache=[_cpu_cache()[0], _cpu_cache(pages=3)[1], None, None]), "alike"),
    (dict(q=_z(1, 4, 3, 256)[..., ::2]), "contiguous rows"), (dict(q=_z(1, 4, 3, 132)[..., :128]), "multiples of 8"),
    (dict(kw=dict(qn=_z(1, 4, 3, 256)[..., :128])), "qn must be"), (dict(kw=dict(kn=_z(1, 4, 3, 128))), "kn must be"),
    (dict(kw=dict(eps=-1.0)), "GPU device"),
])
def test_append_refusals(over, match):
    args, kw = _append_args(**over)
    with pytest.raises(ValueError, match=match):
        kf.norm_rope_to_cache(*args, **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(), "GPU device"), (dict(q=_z(2, 4, 17, 128)), "at most 16"), (dict(q=_z(2, 3, 1, 128)), "multiple of"),
    (dict(q=_z(2, 4, 1, 256)), "cache's D"), (dict(q=_z(2, 4, 1, 128, dtype=torch.float32)), "BF16"),
    (dict(q=_z(2, 4, 1, 128).requires_grad_()), "forward-only"), (dict(pages=torch.zeros(3, 2, dtype=torch.int32)), "pages"),
    (dict(pages=torch.zeros(2, 2)), "pages must be int32"), (dict(pages=torch.zeros(2, 4, dtype=torch.int64)[:, ::2]), "pages"),
    (dict(pages=torch.zeros(2, 0, dtype=torch.int64)), "pages"), (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=torch.zeros(2, dtype=torch.int16)), "lengths must be int32"), (dict(window=0), "window"),
    (dict(softcap=0.0), "softcap"), (dict(softcap=float("nan")), "softcap"), (dict(scale=-1.0), "scale"),
    (dict(out=_z(2, 4, 2, 128)), "out must be"), (dict(out=_z(2, 4, 1, 256)[..., :128]), "out must be"),
])
def test_decode_refusals(kw, match):
    a = dict(q=_z(2, 4, 1, 128), pages=torch.zeros(2, 2, dtype=torch.int32), lengths=torch.ones(2, dtype=torch.int32))
    rest = {n: kw[n] for n in kw if n not in a}
    a.update({n: kw[n] for n in kw if n in a})
    c = _cpu_cache()
    with pytest.raises(ValueError, match=match):
        kf.attention_decode(a["q"], c[0], c[1], a["pages"], a["lengths"], **rest)


def test_read_and_make_cache_refusals():
    c, pages, lengths = _cpu_cache(), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for args, kw, match in (((pages, lengths, 0), {}, "max_length"), ((pages, lengths, 8), {}, "GPU device"),
                            ((pages, lengths[:1], 8), {}, "pages"), ((pages, lengths, 8), dict(k=_z(2, 2, 9, 128)), "k must be"),
                            ((pages, lengths, 2 ** 30), {}, "2\\*\\*31")):
        with pytest.raises(ValueError, match=match):
            kf.cache_to_dense(c[0], c[1], *args, **kw)
    for args, match in (((4, 2, 24, 128), "power of two"), ((4, 2, 16, 64), "D in"), ((0, 2, 16, 128), "pages"),
                        ((4, 2, 16, 128, torch.float16), "bfloat16 or float8")):
        with pytest.raises(ValueError, match=match):
            kf.make_cache(*args, device="cpu")
    q = _cpu_cache(E4M3)
    assert q[2].dtype is E8M0 and q[2].shape == (4, 2, 16) and q[0].dtype is E4M3


@pytest.mark.parametrize("logits,ids,top,match", [
    (torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64), 3, "GPU device"),
    (torch.zeros(2, 9, dtype=torch.float64), torch.zeros(2, dtype=torch.int64), 3, "float32"),
    (torch.zeros(2, 9), torch.zeros(3, dtype=torch.int64), 3, "ids"),
    (torch.zeros(2, 2, 2, 9), torch.zeros(2, 2, 2, dtype=torch.int64), 3, "two leading"),
    (torch.zeros(2, 9), torch.zeros(2), 3, "ids must be int32"),
    (torch.zeros(2, 18)[:, ::2], torch.zeros(2, dtype=torch.int64), 3, "contiguous rows"),
    (torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64), 10, "top must"),
    (torch.zeros(2, 90), torch.zeros(2, dtype=torch.int64), 33, "top must"),
    (torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64), -1, "top must"),
    (torch.zeros(2, 9).requires_grad_(), torch.zeros(2, dtype=torch.int64), 3, "forward-only"),
])
def test_logprobs_refusals(logits, ids, top, match):
    with pytest.raises(ValueError, match=match):
        kf.token_logprobs(logits, ids, top)


# ---------------------------------------------------------------------------
# the 64-bit computations themselves
# ---------------------------------------------------------------------------

def test_quantise_reference():
    v = torch.tensor([[448.0, -1.0], [449.0, 1.0], [0.0, 0.0], [1.0, 0.3]]).to(BF16)
    payload, scale, byte = quantise(v)
    assert scale.tolist() == [1.0, 1.0, 1.0, 2.0 ** -8]  # 449 is 448 in bf16
    assert byte.tolist() == [127, 127, 127, 119]
    assert payload[0].tolist() == [448.0, -1.0] and payload[3, 0] == 256.0


def test_attention_reference_against_a_loop():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((4, 2, 8), (2, 5, 8), (2, 5, 8)))
    out, bound = attention(q, k, v, window=2, softcap=3.0)
    for h in range(4):
        for i in range(2):
            t, w, acc = 5 - 2 + i, 0.0, torch.zeros(8, dtype=torch.float64)
            for j in (t - 1, t):
                z = float((q[h, i] * k[h // 2, j]).sum()) / 8 ** 0.5
                e = torch.exp(3.0 * torch.tanh(torch.tensor(z / 3.0, dtype=torch.float64)))
                w, acc = w + e, acc + e * v[h // 2, j]
            assert torch.allclose(out[h, i], acc / w, rtol=1e-12)
    assert float(bound.max()) < 1e-3 and float(bound.min()) > 0


def test_logprobs_reference():
    x = torch.tensor([[0.0, 1.0, 1.0, -float("inf")], [float("nan"), 0, 0, 0]], dtype=torch.float64)
    logp, h, tl, ti = logprobs(x, torch.tensor([3, 0]), 3)
    assert ti.tolist() == [[1, 2, 0], [-1, -1, -1]] and logp[0] == -float("inf") and torch.isnan(h[1])


def test_packed_structures_are_bytes_for_one_call():
    assert isinstance(_dec(), bytes) and struct.calcsize("P") == 8


def test_gradients_of_a_cache_are_refused():
    """A cache that is a leaf (a learned prefix) would get no gradient: every op says so."""
    args, kw = _append_args()
    for i in (0, 1):
        c = _cpu_cache()
        c[i].requires_grad_()
        with pytest.raises(ValueError, match="forward-only"):
            kf.norm_rope_to_cache(*args[:9], *c, **kw)
        pages, lengths = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
        with pytest.raises(ValueError, match="forward-only"):
            kf.attention_decode(_z(2, 4, 1, 128), c[0], c[1], pages, lengths)
        with pytest.raises(ValueError, match="forward-only"):
            kf.cache_to_dense(c[0], c[1], pages, lengths, 8)
        with torch.no_grad(), pytest.raises(ValueError, match="GPU device"):
            kf.cache_to_dense(c[0], c[1], pages, lengths, 8)
