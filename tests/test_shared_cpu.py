"""Refusals of the shared-prefix entry points (no GPU needed) and the float64
definitions they are tested against."""
import ctypes

import pytest
import torch

from oracle import shared as osh
from rotatek_b200 import _lib
from rotatek_b200.kernels import append_text, read_text, rotatek_shared_decode, verify_drafts
from tests.test_capi_cpu import _fake, lib  # noqa: F401

F32, BF16, U8, I32, I64 = 0, 1, 3, 4, 5


def test_shared_decode_refusals(lib):  # noqa: F811
    base = dict(q=_fake((6, 2, 8, 128)), R=_fake((2, 2, 128, 32)), dm=_fake((2, 2, 128)), kf=_fake((2, 2, 10, 128)),
                vf=_fake((2, 2, 10, 128)), mask=_fake((2, 10), U8), ks=_fake((2, 2, 50, 32)), vs=_fake((2, 2, 50, 128)),
                kt=_fake((6, 2, 20, 128)), vt=_fake((6, 2, 20, 128)), ksc=None, vsc=None, lens=_fake((6,), I32), g=4,
                out=_fake((6, 2, 8, 128)))

    def call(**kw):
        a = {**base, **kw}
        code = lib.rtk_shared_decode(a["q"], a["R"], a["dm"], a["kf"], a["vf"], a["mask"], a["ks"], a["vs"], a["kt"],
                                     a["vt"], a["ksc"], a["vsc"], a["lens"], a["g"], a["out"], None, 0, None, None)
        return code, lib.rtk_last_error().decode()

    assert call(q=_fake((6, 8, 128))) == (1, "q must be [B, T, H_q, D]")
    assert call(R=_fake((2, 128, 32))) == (1, "R_partial must be [P, H_kv, D, D_keep]")
    assert call(R=_fake((4, 2, 128, 32)))[1].startswith("B=6 questions are not the same number for each of P=4")
    assert call(g=3) == (1, "H_q=8 is not H_kv=2 * num_kv_groups=3")
    assert call(g=0)[0] == 1
    assert call(R=_fake((2, 2, 128, 0)))[0] == 1 and call(R=_fake((2, 2, 64, 32)))[0] == 1
    assert call(dm=_fake((2, 2, 64))) == (1, "delta_mu must be [P, H_kv, D]")
    assert call(vf=_fake((2, 2, 9, 128))) == (1, "v_full must be [P, H_kv, S_full, D]")
    assert call(mask=_fake((2, 9), U8))[1] == "mask_full must be a uint8 [P, S_full]"
    assert call(mask=_fake((2, 10), F32))[1] == "mask_full must be a uint8 [P, S_full]"
    assert call(ks=_fake((2, 2, 50, 16)))[1] == "k_sparse must be [P, H_kv, S_sparse, D_keep]"
    assert call(vs=_fake((2, 2, 51, 128)))[1] == "v_sparse must be [P, H_kv, S_sparse, D]"
    assert call(kt=_fake((5, 2, 20, 128)))[1] == "k_text must be [B, H_kv, C, D]"
    assert call(vt=_fake((6, 2, 21, 128)))[1] == "v_text must be [B, H_kv, C, D]"
    sc = _fake((6, 2, 20), F32)
    assert call(ksc=sc, vsc=sc)[1].startswith("k_text and v_text must be uint8")
    k8 = dict(kt=_fake((6, 2, 20, 128), U8), vt=_fake((6, 2, 20, 128), U8))
    assert call(**k8)[1].startswith("k_text and v_text must have q's dtype")
    assert call(**k8, ksc=sc)[1] == "k_scale and v_scale must both be float32 [B, H_kv, C]"
    assert call(**k8, ksc=sc, vsc=_fake((6, 2, 20), BF16))[0] == 1
    assert call(lens=_fake((6,), I64))[1] == "text_lens must be an int32 [B]"
    assert call(out=_fake((6, 2, 8, 64)))[1] == "out must be [B, T, H_q, D] in q's dtype"
    assert call(out=_fake((6, 2, 8, 128), F32))[0] == 1
    assert "must share a dtype" in call(vf=_fake((2, 2, 10, 128), F32))[1]
    assert "must share a dtype" in call(dm=_fake((2, 2, 128), F32))[1]
    assert call(ks=_fake((2, 2, 50, 32), data=0))[1] == "a tensor that is not empty has no address"
    assert call(q=_fake((0, 2, 8, 128)), kt=_fake((0, 2, 20, 128)), vt=_fake((0, 2, 20, 128)), lens=_fake((0,), I32),
                out=_fake((0, 2, 8, 128)))[0] == 0            # no questions: nothing to do


def test_text_cache_refusals(lib):  # noqa: F811
    new, cache, c8 = _fake((3, 2, 4, 128)), _fake((3, 2, 20, 128)), _fake((3, 2, 20, 128), U8)
    sc, lens = _fake((3, 2, 20), F32), _fake((3,), I32)

    def append(kn=new, vn=new, ln=lens, n=None, kt=cache, vt=cache, ks=None, vs=None):
        return lib.rtk_append_text(kn, vn, ln, n, kt, vt, ks, vs, None), lib.rtk_last_error().decode()

    assert append(kn=_fake((3, 4, 128))) == (1, "k_new must be [B, H_kv, T, D]")
    assert append(vn=_fake((3, 2, 5, 128))) == (1, "v_new must be [B, H_kv, T, D]")
    assert append(kt=_fake((3, 2, 20, 64))) == (1, "k_text must be [B, H_kv, C, D]")
    assert append(vt=_fake((3, 2, 19, 128))) == (1, "v_text must be [B, H_kv, C, D]")
    assert append(kt=c8, vt=c8)[1].startswith("k_text and v_text must have k_new's dtype")
    assert append(ks=sc, vs=sc)[1].startswith("k_text and v_text must be uint8")
    assert append(kt=c8, vt=c8, ks=sc)[1] == "k_scale and v_scale must both be float32 [B, H_kv, C]"
    assert append(ln=_fake((3,), I64))[1] == "text_lens must be an int32 [B]"
    assert append(n=_fake((2,), I32))[1] == "counts must be an int32 [B]"
    assert append(kn=_fake((3, 2, 4, 128), U8), vn=_fake((3, 2, 4, 128), U8))[0] == 1

    def read(kt=c8, vt=c8, ks=sc, vs=sc, ln=lens, ko=cache, vo=cache):
        return lib.rtk_read_text(kt, vt, ks, vs, ln, ko, vo, None), lib.rtk_last_error().decode()

    assert read(kt=cache)[1] == "k_text must be a uint8 (e4m3) [B, H_kv, C, D]"
    assert read(vt=_fake((3, 2, 19, 128), U8))[0] == 1
    assert read(ks=None)[1] == "k_scale and v_scale must both be float32 [B, H_kv, C]"
    assert read(vo=_fake((3, 2, 20, 128), F32))[0] == 1
    assert read(ln=_fake((2,), I32))[1] == "text_lens must be an int32 [B]"


def test_verify_refusals(lib):  # noqa: F811
    base = dict(tl=_fake((3, 5, 100)), dt=_fake((3, 4), I64), dl=_fake((3, 4, 100)), u=_fake((3, 4), F32),
                n=_fake((3, 100), F32), h=_fake((3,), F32), ln=_fake((3,), I32), to=_fake((3, 5), I64),
                ao=_fake((3,), I32), ws=None, size=0)

    def call(**kw):
        a = {**base, **kw}
        code = lib.rtk_verify_drafts(a["tl"], a["dt"], a["dl"], a["u"], a["n"], a["h"], a["ln"], a["to"], a["ao"],
                                     a["ws"], a["size"], None)
        return code, lib.rtk_last_error().decode()

    assert call(tl=_fake((5, 100))) == (1, "target_logits must be [B, T + 1, V]")
    assert call(dt=_fake((3, 5), I64)) == (1, "draft_tokens must be an int64 [B, T]")
    assert call(dt=_fake((3, 4), I32))[0] == 1
    assert call(dl=_fake((3, 4, 100), F32))[1] == "draft_logits must be [B, T, V] in target_logits' dtype"
    assert call(u=_fake((3, 4), BF16))[1] == "uniforms must be a float32 [B, T]"
    assert call(n=_fake((3, 99), F32))[1] == "noise must be a float32 [B, V]"
    assert call(h=_fake((2,), F32))[1] == "temperature must be a float32 [B]"
    assert call(ln=_fake((3,), I64))[1] == "draft_lens must be an int32 [B]"
    assert call(to=_fake((3, 4), I64))[1] == "tokens_out must be a contiguous int64 [B, T + 1]"
    assert call(tl=_fake((3, 66, 9)), dt=_fake((3, 65), I64), dl=None, u=_fake((3, 65), F32), n=_fake((3, 9), F32),
                to=_fake((3, 66), I64))[0] == _lib.RTK_ERR_UNSUPPORTED
    need = lib.rtk_verify_drafts_workspace_size(3, 4, 100)
    assert call()[0] == _lib.RTK_ERR_WORKSPACE
    assert call(ws=ctypes.c_void_p(0x1000), size=need - 1)[0] == _lib.RTK_ERR_WORKSPACE
    assert call(ws=ctypes.c_void_p(0x1008), size=need)[1] == "workspace must be 16-byte aligned"


def test_python_refuses_cpu_tensors_and_wrong_ranks():
    q, R = torch.zeros(2, 1, 8, 128), torch.zeros(1, 2, 128, 32)
    kf, ks, kt = torch.zeros(1, 2, 10, 128), torch.zeros(1, 2, 50, 32), torch.zeros(2, 2, 5, 128)
    lens = torch.ones(2, dtype=torch.int32)
    args = (R, None, kf, kf, None, ks, torch.zeros(1, 2, 50, 128), kt, kt, lens, 4)
    with pytest.raises(ValueError, match=r"q must be \[B, T, H_q, D\]"):
        rotatek_shared_decode(q[0], *args)
    with pytest.raises(ValueError, match=r"R_partial must be"):
        rotatek_shared_decode(q, R[0], *args[1:])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        rotatek_shared_decode(q, *args)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        append_text(kt, kt, lens, kt, kt)
    with pytest.raises(ValueError, match="k_new must be"):
        append_text(kt[0], kt[0], lens, kt, kt)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        read_text(kt.to(torch.uint8), kt.to(torch.uint8), lens, k_scale=torch.ones(2, 2, 5), v_scale=torch.ones(2, 2, 5))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        verify_drafts(torch.zeros(2, 3, 9), torch.zeros(2, 2, dtype=torch.int64), None, torch.zeros(2, 2),
                      torch.ones(2, 9), torch.ones(2))


def test_oracle_prefix_is_shared():
    """The definition with P prefixes equals the plain softmax of each question's own
    concatenated cache."""
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    q, R, dm = r(4, 2, 4, 16), torch.linalg.qr(r(2, 2, 16, 4))[0], r(2, 2, 16)
    kf, vf, ks, vs, kt, vt = r(2, 2, 5, 16), r(2, 2, 5, 16), r(2, 2, 7, 4), r(2, 2, 7, 16), r(4, 2, 6, 16), r(4, 2, 6, 16)
    lens = torch.tensor([6, 2, 1, 0], dtype=torch.int32)
    out, _ = osh.shared_decode(q, R, dm, kf, vf, None, ks, vs, kt, vt, lens, 2)
    for b in range(4):
        vis = ks[b // 2] @ R[b // 2].transpose(-1, -2) + dm[b // 2][:, None]
        for t in range(2):
            n = max(0, int(lens[b]) - 1 + t)
            k = torch.cat([kf[b // 2], vis, kt[b, :, :n]], 1).repeat_interleave(2, 0)
            v = torch.cat([vf[b // 2], vs[b // 2], vt[b, :, :n]], 1).repeat_interleave(2, 0)
            w = torch.softmax((k @ q[b, t, :, :, None])[..., 0] / 4.0, -1)
            torch.testing.assert_close(out[b, t], (w[:, None] @ v)[:, 0])


def test_oracle_rows_quantise_as_torch_does():
    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(1)) * 10
    val, scale = osh.quantize_rows(x)
    want = (x / scale[:, None]).to(torch.float8_e4m3fn).double()
    assert torch.equal(val, want)


def test_scratch_is_a_threads_own(monkeypatch):
    """A call is several launches over its scratch, and the launches of two threads on one
    stream may alternate: they share no scratch."""
    import threading

    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)
    here, barrier, got = torch.device("cpu"), threading.Barrier(2, timeout=60), {}

    def call(who):
        mine = _lib.scratch(here, 0, 5000)
        barrier.wait()                                   # both calls are under way
        got[who] = (mine, _lib.scratch(here, 0, 3000), _lib.scratch(here, 1, 3000))
        barrier.wait()

    threads = [threading.Thread(target=call, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for who in range(2):
        mine, again, elsewhere = got[who]
        assert again.data_ptr() == mine.data_ptr() != elsewhere.data_ptr()
    assert got[0][0].data_ptr() != got[1][0].data_ptr() and got[0][2].data_ptr() != got[1][2].data_ptr()


def test_long_scratch_is_not_kept(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)
    here = torch.device("cpu")
    long = _lib.scratch(here, 7, (64 << 20) + 1)
    assert long.numel() >= (64 << 20) + 1
    assert _lib.scratch(here, 7).numel() <= 64 << 20


def test_a_capture_leaves_no_workspace_behind(monkeypatch):
    """What a captured call fills with zeros reads zero when the graph runs, not before: calls
    outside the capture do not count on it."""
    zeros, capturing = torch.zeros, [True]
    monkeypatch.setattr(torch, "zeros", lambda n, dtype, device: zeros(n, dtype=dtype))
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: capturing[0])
    monkeypatch.setattr(_lib, "_workspaces", {})
    monkeypatch.setattr(_lib, "_zero_prefix", {})
    dev = torch.device("cuda", 0)
    assert _lib.workspace(dev, 5000, 700).numel() >= 5000 and not _lib._workspaces
    capturing[0] = False
    buf = _lib.workspace(dev, 5000, 700)
    assert _lib._workspaces[0] is buf and _lib._zero_prefix[0] == 700
    buf[700:] = 3                                        # scratch of that call
    capturing[0] = True
    assert _lib.workspace(dev, 5000, 4000) is buf and _lib._zero_prefix[0] == 700
    capturing[0] = False
    buf[700:] = 3                                        # as if the captured zeros had not been run
    assert (_lib.workspace(dev, 5000, 4000)[:4000] == 0).all()


OLD_DLPACK = """#define DLPACK_MAJOR_VERSION 1
#define DLPACK_MINOR_VERSION 0
typedef struct { int code; } DLSomethingOlder;
"""


@pytest.mark.parametrize("header", [OLD_DLPACK, None])
def test_direct_calls_build_without_the_exchange_api(header, tmp_path, lib):  # noqa: F811
    """A torch whose dlpack.h has no exchange API, or none at all: descriptors come from attributes."""
    import importlib.util
    import os
    import shutil
    import subprocess
    import sysconfig

    from rotatek_b200.csrc import build
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    if header is not None:
        (tmp_path / "ATen").mkdir()
        (tmp_path / "ATen" / "dlpack.h").write_text(header)
    out = str(tmp_path / "_calls.so")
    subprocess.run([cc, "-std=c11", "-Wall", "-Werror", "-shared", "-fPIC", "-I", sysconfig.get_paths()["include"], "-I",
                    str(tmp_path), os.path.join(build.CSRC, "calls.c"), "-o", out, "-ldl"], check=True)
    spec = importlib.util.spec_from_file_location("_calls", out)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.bind(_lib.LIB_PATH, _lib._DTYPES, torch.Tensor)
    x = torch.zeros(1, 1, 1, 128)
    assert mod.append_text(x, x, torch.zeros(1, dtype=torch.int32), None, x, x, None, None, 0) == -1     # not on a GPU
    assert mod.append_text(*[None] * 8, 0) == 1 and "k_new must be" in lib.rtk_last_error().decode()


def test_given_tensors_without_an_address_are_refused(lib):  # noqa: F811
    """Also the nullable ones: a NULL tensor is left out, a tensor with NULL data is not."""
    bad = lambda *a: _fake(*a, data=0)  # noqa: E731
    q, R, full = _fake((6, 2, 8, 128)), _fake((2, 2, 128, 32)), _fake((2, 2, 10, 128))
    ks, vs, kt, k8 = _fake((2, 2, 50, 32)), _fake((2, 2, 50, 128)), _fake((6, 2, 20, 128)), _fake((6, 2, 20, 128), U8)
    sc, lens = _fake((6, 2, 20), F32), _fake((6,), I32)
    why = (1, "a tensor that is not empty has no address")

    def attend(dm=None, mask=None, text=kt, ksc=None, vsc=None):
        return (lib.rtk_shared_decode(q, R, dm, full, full, mask, ks, vs, text, text, ksc, vsc, lens, 4, q, None, 0, None,
                                      None), lib.rtk_last_error().decode())

    assert attend(dm=bad((2, 2, 128))) == why
    assert attend(mask=bad((2, 10), U8)) == why
    assert attend(text=k8, ksc=bad((6, 2, 20), F32), vsc=sc) == why
    assert attend(text=k8, ksc=sc, vsc=bad((6, 2, 20), F32)) == why

    def append(counts=None, cache=kt, ksc=None, vsc=None):
        new = _fake((6, 2, 4, 128))
        return lib.rtk_append_text(new, new, lens, counts, cache, cache, ksc, vsc, None), lib.rtk_last_error().decode()

    assert append(counts=bad((6,), I32)) == why
    assert append(cache=k8, ksc=bad((6, 2, 20), F32), vsc=sc) == why
    assert append(cache=k8, ksc=sc, vsc=bad((6, 2, 20), F32)) == why

    def verify(dl=None, ln=None):
        return (lib.rtk_verify_drafts(_fake((3, 5, 100)), _fake((3, 4), I64), dl, _fake((3, 4), F32), _fake((3, 100), F32),
                                      _fake((3,), F32), ln, _fake((3, 5), I64), _fake((3,), I32), None, 0, None),
                lib.rtk_last_error().decode())

    assert verify(dl=bad((3, 4, 100))) == why
    assert verify(ln=bad((3,), I32)) == why
