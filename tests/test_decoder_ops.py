"""The decoder-block operators on the CPU: the oracle's gradients against differences, the refusals of the Python entry
points (shapes and types are checked before the device), and the argument checks and size queries of the C ABI, which
return before any device call -- those also under the host-sanitized build where it exists."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from oracle import decoder_oracle as orc
from visiontransformer_amd import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def rnd(*s, seed=0):
    return torch.randn(*s, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shared", [False, True])
def test_oracle_rope_against_differences(interleaved, shared):
    x = rnd(2, 3, 2, 11).requires_grad_()
    pos = torch.tensor([[0, 0], [3, -2], [1000003, 7]])
    f = lambda t: orc.rope_axes(t, pos, (2, 3), 100.0, interleaved, shared)
    assert torch.autograd.gradcheck(f, (x,))
    y = f(x)
    assert torch.equal(y[:, 0], x[:, 0])                                   # the origin turns by nothing
    assert torch.allclose(y.square().sum(-1), x.square().sum(-1))          # a rotation keeps lengths
    assert torch.equal(y[..., 10:], x[..., 10:])


def test_oracle_rope_scores_depend_on_distance_alone():
    q, k = rnd(1, 1, 1, 8), rnd(1, 1, 1, 8, seed=1)
    at = lambda t, p: orc.rope_axes(t, torch.tensor([[p, 2 * p]]), (2, 2))
    a = (at(q, 5) * at(k, 3)).sum()
    b = (at(q, 1005) * at(k, 1003)).sum()
    assert abs(a - b) < 1e-9


def test_oracle_cross_attention_against_differences():
    q, k, v = (rnd(2, 3, 4, 5).requires_grad_(), rnd(2, 6, 2, 5, seed=1).requires_grad_(), rnd(2, 6, 2, 5, seed=2).requires_grad_())
    keep = torch.ones(2, 6, dtype=torch.bool)
    keep[0, 2] = False
    keep[1] = False
    assert torch.autograd.gradcheck(lambda *t: orc.cross_attn(*t, keep), (q, k, v))
    full = torch.ones(2, 6, dtype=torch.bool)
    ref = torch.nn.functional.scaled_dot_product_attention(*(t.detach().transpose(1, 2) for t in (q, k.repeat_interleave(2, 2),
                                                                                                 v.repeat_interleave(2, 2))))
    assert torch.allclose(orc.cross_attn(q, k, v, full).detach(), ref.transpose(1, 2))


@pytest.mark.parametrize("post", [None, "layer", "rms"])
@pytest.mark.parametrize("pre", [None, "layer", "rms"])
@pytest.mark.parametrize("per_sample", [False, True])
def test_oracle_norm_gate_residual_against_differences(post, pre, per_sample):
    B, N, D = 3, 2, 5
    x, u = rnd(B, N, D).requires_grad_(), rnd(B, N, D, seed=1).requires_grad_()
    gate = (rnd(B, D, seed=2) if per_sample else rnd(D, seed=2)).requires_grad_()
    kw = {}
    for side, kind in (("post", post), ("pre", pre)):
        if kind:
            kw[side + "_weight"] = rnd(D, seed=3).requires_grad_()
            kw[side + "_bias"] = rnd(D, seed=4).requires_grad_()
    keys = list(kw)
    s = torch.tensor([1.0, 0.0, 1.25], dtype=torch.float64)

    def f(x, u, gate, *p):
        y, h = orc.norm_gate_residual(x, u, gate, s, 0.75, post, pre=pre, **dict(zip(keys, p)))
        return y if h is None else (y, h)
    assert torch.autograd.gradcheck(f, (x, u, gate, *kw.values()))


# ---------------------------------------------------------------------------------------------- refusals
def test_rope_refusals():
    q, k = torch.zeros(2, 3, 4, 16), torch.zeros(2, 3, 2, 16)
    pos = torch.zeros(3, 2, dtype=torch.int64)
    with pytest.raises(ValueError, match="batch, tokens, heads"):
        ops.rope_axes(q[0], k, pos, (4, 4))
    with pytest.raises(ValueError, match="agree"):
        ops.rope_axes(q, k[:, :2], pos, (4, 4))
    with pytest.raises(ValueError, match="agree"):
        ops.rope_axes(q, k.bfloat16(), pos, (4, 4))
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        ops.rope_axes(q.half(), None, pos, (4, 4))
    for sections in ((), (0, 4), (1, 1, 1, 1, 1)):
        with pytest.raises(ValueError, match="sections"):
            ops.rope_axes(q, k, pos, sections)
    with pytest.raises(ValueError, match="the head has 16"):
        ops.rope_axes(q, k, pos, (4, 5))
    with pytest.raises(TypeError, match="positions are"):
        ops.rope_axes(q, k, pos.double(), (4, 4))
    with pytest.raises(ValueError, match="must be"):
        ops.rope_axes(q, k, pos[:, :1], (4, 4))
    for base in (1.0, 0.5, (100.0,), float("inf"), float("nan")):
        with pytest.raises(ValueError, match="base"):
            ops.rope_axes(q, k, pos, (4, 4), base=base)
    with pytest.raises(ValueError, match="one base"):
        ops.rope_axes(q, k, pos, (4, 4), base=(10.0, 100.0), shared_ladder=True)
    with pytest.raises(RuntimeError, match="outside of autograd"):
        ops.rope_axes(q.clone().requires_grad_(), k, pos, (4, 4), inplace=True)
    with pytest.raises(ValueError, match="broadcast"):
        ops.rope_axes(q[:1].expand(2, 3, 4, 16), k, pos, (4, 4), inplace=True)
    with pytest.raises(ValueError, match="unit stride"):
        ops.rope_axes(q.transpose(2, 3), None, torch.zeros(3, 1, dtype=torch.int64), (2,), inplace=True)
    with pytest.raises(ValueError, match="apart"):
        ops.rope_axes(q, q, pos, (4, 4), inplace=True)
    for inplace in (False, True):
        with pytest.raises(RuntimeError, match="ROCm device tensors"):
            ops.rope_axes(q, k, pos, (4, 4), inplace=inplace)


def test_cross_attn_refusals():
    q, k = torch.zeros(2, 3, 4, 16), torch.zeros(2, 5, 2, 16)
    with pytest.raises(ValueError, match="batch, tokens, heads"):
        ops.cross_attn(q[0], k, k)
    with pytest.raises(TypeError, match="share a dtype"):
        ops.cross_attn(q, k, k.bfloat16())
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        ops.cross_attn(q.half(), k.half(), k.half())
    for kk, vv in ((k, k[:, :4]), (k[:1], k[:1]), (k[..., :8], k[..., :8])):
        with pytest.raises(ValueError, match="must be"):
            ops.cross_attn(q, kk, vv)
    with pytest.raises(ValueError, match="cannot share"):
        ops.cross_attn(q, torch.zeros(2, 5, 3, 16), torch.zeros(2, 5, 3, 16))
    big = torch.zeros(1, 1, 1, 129)
    with pytest.raises(ValueError, match="exceed"):
        ops.cross_attn(big, big, big)
    keep, lens = torch.ones(2, 5, dtype=torch.bool), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="not both"):
        ops.cross_attn(q, k, k, kv_len=lens, key_mask=keep)
    for bad in (lens.float(), lens[:1], lens[:, None]):
        with pytest.raises(ValueError, match="kv_len"):
            ops.cross_attn(q, k, k, kv_len=bad)
    for bad in (keep.int(), keep[:, :4], keep[0]):
        with pytest.raises(ValueError, match="key_mask"):
            ops.cross_attn(q, k, k, key_mask=bad)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            ops.cross_attn(q, k, k, scale=scale)
    with pytest.raises(RuntimeError, match="ROCm device tensors"):
        ops.cross_attn(q, k, k)


def test_norm_gate_residual_refusals():
    x = torch.zeros(2, 3, 8)
    w = torch.ones(8)
    with pytest.raises(ValueError, match="alike"):
        ops.norm_gate_residual(x, x[:, :2])
    with pytest.raises(ValueError, match="alike"):
        ops.norm_gate_residual(x[0], x[0])
    with pytest.raises(TypeError, match="bf16 residual"):
        ops.norm_gate_residual(x.bfloat16(), x)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        ops.norm_gate_residual(x.half(), x.half())
    wide = torch.zeros(1, 1, 8193)
    with pytest.raises(ValueError, match="outside"):
        ops.norm_gate_residual(wide, wide)
    with pytest.raises(ValueError, match="layer"):
        ops.norm_gate_residual(x, x, post="batch")
    with pytest.raises(ValueError, match="without post"):
        ops.norm_gate_residual(x, x, post_weight=w)
    with pytest.raises(ValueError, match="pre_bias must be"):
        ops.norm_gate_residual(x, x, pre="layer", pre_bias=w[:4])
    with pytest.raises(ValueError, match="pre_weight must be"):
        ops.norm_gate_residual(x, x, pre="layer", pre_weight=w.bfloat16())
    with pytest.raises(ValueError, match="gate"):
        ops.norm_gate_residual(x, x, gate=torch.zeros(3, 8))
    with pytest.raises(ValueError, match="branch_scale"):
        ops.norm_gate_residual(x, x, branch_scale=torch.ones(3))
    with pytest.raises(ValueError, match="not differentiated"):
        ops.norm_gate_residual(x, x, branch_scale=torch.ones(2).requires_grad_())
    with pytest.raises(RuntimeError, match="ROCm device tensors"):
        ops.norm_gate_residual(x, x)


# ---------------------------------------------------------------------------------------------- C ABI without a device
CHECKS = r"""
import ctypes, os, sys
sys.path.insert(0, sys.argv[2])
if sys.argv[1]:
    os.environ["VITMI_LIB"] = sys.argv[1]
from visiontransformer_amd import _lib, ops
lib, at = _lib.lib, ctypes.addressof
big = 2 ** 31 - 1
assert lib.vitmi_rope_axes(None, None) == -1
a = ops._RopeArgs()
def rope(**kw):
    for k, v in dict(dict(dt=1, axes=1, pos_type=1, B=1, N=1, DH=64), **kw).items():
        setattr(a, k, v)
    return lib.vitmi_rope_axes(at(a), None)
a.t[0].heads = 1
a.sections[0] = 16
a.log2_base[0] = 13.3
assert rope(N=0) == 0 and rope(B=0) == 0
for bad in (dict(dt=2), dict(axes=0), dict(axes=5), dict(pos_type=3), dict(B=-1), dict(DH=31), dict()):
    assert rope(**bad) == -1, bad               # dict(): null pointers
a.sections[0] = big
assert rope(DH=big) == -1
a.sections[0], a.log2_base[0] = 16, 0.0
assert rope() == -1
x = ops._XattnArgs()
def xattn(fn, **kw):
    base = dict(dt=1, B=1, Nq=1, Nk=1, Hq=2, Hk=1, D=64, scale=1.0)
    for k, v in dict(base, **kw).items():
        setattr(x, k, v)
    return fn(at(x), None, None)
f, b = lib.vitmi_cross_attn_fwd, lib.vitmi_cross_attn_bwd
assert f(None, None, None) == -1 and b(None, None, None) == -1
assert xattn(f, B=0) == 0 and xattn(f, Nq=0) == 0
for fn in (f, b):
    for bad in (dict(dt=2), dict(Nq=-1), dict(Hq=3, Hk=2), dict(Hk=0), dict(scale=0.0), dict(scale=float("inf")),
                dict(scale=float("nan")), dict(Nk=big), dict(Nq=big), dict(Hq=big - 1, Nq=4), dict()):
        assert xattn(fn, **bad) == -1, bad
    assert xattn(fn, D=129) == -3
assert xattn(b, Nk=0) == -1
for dt in (0, 1):
    for s in ((1, 1, 1, 1, 1, 1), (2, 4096, 4609, 16, 4, 128), (8, 1, 16411, 32, 8, 128), (1, 1, big - 300, 1, 1, 128),
              (4096, 197, 197, 12, 12, 64), (1, big - 300, 1, 1, 1, 1), (65535, 1, 1, 128, 1, 128)):
        assert lib.vitmi_cross_attn_fwd_workspace_bytes(dt, *s) >= 0
        assert lib.vitmi_cross_attn_bwd_workspace_bytes(dt, *s) > 0
    assert lib.vitmi_cross_attn_bwd_workspace_bytes(dt, 1, big, 1, 2, 1, 1) == 0
    assert lib.vitmi_cross_attn_fwd_workspace_bytes(dt, 1, 1, 1, 3, 2, 1) == 0
n = ops._NgrArgs()
def ngr(fn, **kw):
    for k, v in dict(dict(dt_x=1, dt_u=1, B=1, N=1, D=8, post=1, pre=1, eps=1e-6, res_scale=1.0), **kw).items():
        setattr(n, k, v)
    return fn(at(n), None) if fn is nf else fn(at(n), None, None)
nf, nb = lib.vitmi_norm_gate_residual_fwd, lib.vitmi_norm_gate_residual_bwd
assert nf(None, None) == -1 and nb(None, None, None) == -1
assert ngr(nf, B=0) == 0 and ngr(nf, N=0) == 0
for fn in (nf, nb):
    for bad in (dict(dt_x=2), dict(dt_x=1, dt_u=0), dict(D=0), dict(N=-1), dict(post=3), dict(pre=-1), dict()):
        assert ngr(fn, **bad) == -1, bad
    assert ngr(fn, D=8193) == -3
for s in ((1, 1, 1, 0), (256, 197, 768, 0), (65536, 1, 8192, 1), (big, 1, 8192, 0), (1, big, 8192, 1)):
    assert lib.vitmi_norm_gate_residual_bwd_workspace_bytes(*s) > 0
print("ok")
"""


@pytest.mark.parametrize("sanitized", [False, True])
def test_c_abi_checks_and_sizes(sanitized):
    path = os.path.join(ROOT, "visiontransformer_amd", "libvitmi_hip_hostsan.so") if sanitized else ""
    if sanitized and not os.path.exists(path):
        pytest.skip("host-sanitized library not built")
    r = subprocess.run([sys.executable, "-c", CHECKS, path, ROOT], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), (r.returncode, r.stdout, r.stderr[-2000:])


MORE_CHECKS = r"""
import ctypes, os, sys
sys.path.insert(0, sys.argv[2])
if sys.argv[1]:
    os.environ["VITMI_LIB"] = sys.argv[1]
from visiontransformer_amd import _lib, ops
lib, at = _lib.lib, ctypes.addressof
assert lib.vitmi_cross_attn_fwd.restype is ctypes.c_int
x = ops._XattnArgs(q=64, k=64, v=64, o=64, lse=64, dout=64, dt=1, B=1, Nq=100, Nk=8000, Hq=1, Hk=1, D=64, scale=1.0)
f, b = lib.vitmi_cross_attn_fwd, lib.vitmi_cross_attn_bwd
said = lambda: lib.vitmi_last_error().decode()
assert lib.vitmi_cross_attn_fwd_workspace_bytes(1, 1, 100, 8000, 1, 1, 64) > 0
for fn in (f, b):                       # nothing is launched: every call ends at a check
    assert fn(at(x), 0, None) == -1 and ("workspace" in said() or "null" in said())
    assert fn(at(x), 264, None) == -1 and "aligned" in said(), said()
    for name in ("qs", "ks", "vs", "dos"):
        s = getattr(x, name)
        s[1] = -64
        assert fn(at(x), 256, None) == -1 and "negative" in said(), said()
        s[1] = 0
    x.Nk = 2 ** 31 - 4096               # tiles looked at ahead would pass the largest int
    assert fn(at(x), 256, None) == -1 and "lengths" in said(), said()
    x.Nk = 8000
n = ops._NgrArgs(x=64, u=64, stats=64, dy=64, dpost_w=64, dt_x=1, dt_u=1, B=1, N=1, D=8, post=1, eps=1e-6, res_scale=1.0)
assert lib.vitmi_norm_gate_residual_bwd(at(n), 264, None) == -1 and "aligned" in said(), said()
n.eps = -1e-6
assert lib.vitmi_norm_gate_residual_bwd(at(n), 256, None) == -1 and "eps" in said(), said()
assert lib.vitmi_norm_gate_residual_fwd(at(n), None) == -1 and "eps" in said(), said()
print("ok")
"""


@pytest.mark.parametrize("sanitized", [False, True])
def test_c_abi_refuses_what_no_kernel_covers(sanitized):
    path = os.path.join(ROOT, "visiontransformer_amd", "libvitmi_hip_hostsan.so") if sanitized else ""
    if sanitized and not os.path.exists(path):
        pytest.skip("host-sanitized library not built")
    r = subprocess.run([sys.executable, "-c", MORE_CHECKS, path, ROOT], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), (r.returncode, r.stdout, r.stderr[-2000:])


def test_in_place_rotation_of_shared_memory_and_negative_eps_are_refused():
    buf, pos = torch.zeros(200), torch.zeros(3, 1)
    a, b = buf[:96].view(2, 3, 2, 8), buf[90:186].view(2, 3, 2, 8)
    with pytest.raises(ValueError, match="apart"):
        ops.rope_axes(a, b, pos, (2,), inplace=True)
    with pytest.raises(ValueError, match="apart"):
        ops.rope_axes(a, a, pos, (2,), inplace=True)
    with pytest.raises(RuntimeError, match="ROCm device tensors"):       # neighbours are apart: the next check speaks
        ops.rope_axes(a, buf[96:192].view(2, 3, 2, 8), pos, (2,), inplace=True)
    x = torch.zeros(2, 3, 8)
    for eps in (-1e-6, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            ops.norm_gate_residual(x, x, post="rms", eps=eps)


def test_argument_structs_match_the_header(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "%s/include/vitmi.h"\nint main(void) { printf("%%zu %%zu %%zu %%zu", '
                   'sizeof(vitmi_rope_tensor), sizeof(vitmi_rope_args), sizeof(vitmi_xattn_args), sizeof(vitmi_ngr_args)); '
                   'return 0; }\n' % ROOT)
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", str(src), "-o", exe], check=True)
    sizes = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [ctypes.sizeof(t) for t in (ops._RopeTensor, ops._RopeArgs, ops._XattnArgs, ops._NgrArgs)]


def test_entry_points_are_bound():
    for name in ("vitmi_rope_axes", "vitmi_cross_attn_fwd", "vitmi_cross_attn_bwd", "vitmi_norm_gate_residual_fwd",
                 "vitmi_norm_gate_residual_bwd"):
        assert name in _lib.SIGNATURES and hasattr(_lib.lib, name)


SHARES = r"""
#include <stdio.h>
#include <algorithm>
#include <map>
#include <random>
#include <utility>
#include "%s/visiontransformer_amd/csrc/shares.h"
// Every workgroup's walk over its share and every tile's join, as the kernels make them; a slot or a tile that is read holds
// what was written for it, the units of a tile in order and each once.
int check(long long tiles, int grid, int rt) {
    const Shares s = shares_of(tiles, grid, rt);
    if (s.nb < 0 || s.nb > grid || s.units != tiles * rt) return 1;
    std::map<long long, Share> slots;
    std::map<long long, int> whole;
    for (int i = 0; i < s.nb; ++i) {
        long long u = s.begin(i);
        const long long u1 = s.begin(i + 1);
        for (int part = 0; u < u1; ++part) {
            const Share p = s.piece(u, u1);
            if (p.t0 < 0 || p.t0 >= p.t1 || p.t1 > rt || p.tile < 0 || p.tile >= tiles) return 2;
            u += p.t1 - p.t0;
            if (p.t0 == 0 && p.t1 == rt) {
                if (whole[p.tile]++) return 3;
            } else if (!slots.insert(std::make_pair(Shares::slot(i, part), p)).second) {
                return 4;
            }
        }
    }
    for (long long tile = 0; tile < tiles; ++tile) {
        const long long x0 = tile * rt;
        const int i0 = s.owner(x0), i1 = s.owner(x0 + rt - 1);
        if (i0 < 0 || i1 >= s.nb || i0 > i1) return 5;
        if (i0 == i1) {
            if (whole[tile] != 1) return 6;
            continue;
        }
        if (whole[tile]) return 7;
        int next = 0;
        for (int i = i0; i <= i1; ++i) {
            const auto f = slots.find(Shares::slot(i, i == i0 ? s.part_of(i0, x0) : 0));
            if (f == slots.end()) return 8;               // read without having been written
            if (f->second.tile != tile || f->second.t0 != next) return 9;
            next = f->second.t1;
        }
        if (next != rt) return 10;
    }
    return 0;
}
int main() {
    std::mt19937 rng(1);
    auto pick = [&](int lo, int hi) { return (int)(lo + rng() %% (unsigned)(hi - lo + 1)); };
    for (int n = 0; n < 60000; ++n) {
        // the host sizes the launch for the padded tiles, four row tiles or more a workgroup; any number of them may be live
        const int rt = pick(8, n %% 3 ? 40 : 400), padded = pick(1, n %% 2 ? 30 : 1000);
        const int grid = (int)std::min<long long>(pick(0, 1) ? 256 : 512, (long long)padded * rt / 4);
        const int live = pick(0, pick(0, padded));
        if (const int rc = check(live, grid, rt)) {
            printf("%%d: %%d live tiles of %%d units, %%d workgroups\n", rc, live, rt, grid);
            return 1;
        }
    }
    printf("ok\n");
    return 0;
}
"""


def test_shares_of_live_tiles_are_all_written_before_they_are_joined(tmp_path):
    """The streamed dk / dv launch is sized for padded lengths and cut by live ones: with a few keys alive of many, a
    share must not be left empty while the join adds it."""
    src = tmp_path / "shares.cpp"
    src.write_text(SHARES % ROOT)
    exe = str(tmp_path / "shares")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", str(src), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout


def test_tracing_is_refused():
    """A traced program would hold the empty result tensors alone, or nodes for the sizes of the traced call, unchecked."""
    x, pos = torch.zeros(2, 3, 4, 16), torch.zeros(3, 2, dtype=torch.int64)
    for grad in (False, True):
        a, u = x.clone().requires_grad_(grad), torch.zeros(2, 3, 8).requires_grad_(grad)
        for f, t in ((lambda t: ops.rope_axes(t, None, pos, (4, 4)), a), (lambda t: ops.rope_axes(t, None, pos, (4, 4), inplace=True), a),
                     (lambda t: ops.cross_attn(t, t, t), a), (lambda t: ops.norm_gate_residual(t, t)[0], u)):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                torch.jit.trace(f, (t,), check_trace=False)


def test_arguments_without_a_gradient_do_not_drop_one():
    """Positions and plain numbers are not differentiated: such an argument that wants a gradient is refused while one would be
    recorded."""
    x, u = torch.zeros(2, 3, 4, 16), torch.zeros(2, 3, 8)
    pos, one = torch.zeros(3, 2, requires_grad=True), torch.ones((), requires_grad=True)
    calls = (lambda: ops.rope_axes(x, None, pos, (4, 4)), lambda: ops.rope_axes(x, x.clone(), pos, (4, 4), inplace=True),
             lambda: ops.rope_axes(x, None, pos.detach(), (4, 4), base=one * 100.0),
             lambda: ops.rope_axes(x, None, pos.detach(), (4, 4), base=(one * 100.0, 10.0)), lambda: ops.cross_attn(x, x, x, scale=one),
             lambda: ops.norm_gate_residual(u, u, res_scale=one), lambda: ops.norm_gate_residual(u, u, post="rms", eps=one))
    for f in calls:
        with pytest.raises(ValueError, match="not differentiated"):
            f()
        with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm device tensors"):      # nothing to lose: the next check speaks
            f()


def test_rotary_arguments_are_kept_by_value(monkeypatch):
    """A base or a section count that lies in a tensor and changes between two calls must not meet the first call's ladder."""
    seen = []
    monkeypatch.setattr(ops, "_one_device", lambda *t: 0)
    monkeypatch.setattr(ops, "_rope_launch", lambda device, xs, outs, pos, ladder, *rest: seen.append(ladder))
    x, pos = torch.zeros(2, 3, 4, 16), torch.zeros(3, 2)
    n, base = torch.tensor(4), torch.tensor(100.0)
    for _ in range(2):
        ops.rope_axes(x, None, pos, (n, 2), base)
        ops.rope_axes(x, None, pos, (n, 2), [base, 10.0])
        ops.rope_axes(x, None, pos, [int(n), 2], float(base))
        ops.rope_axes(x, None, pos, (int(n), 2), (float(base), 10.0))
        n += 1
        base *= 10
    assert seen[0] == seen[2] and seen[1] == seen[3] and seen[4] == seen[6] and seen[5] == seen[7] and seen[0] != seen[4]


def test_in_place_rotation_of_interleaved_views_that_share_elements_is_refused():
    """Slots of a packed projection are apart though their ranges meet; slots that share a head, a dim or a row are not, nor is a
    window view of its own memory."""
    pos = torch.zeros(5, 1)
    buf = torch.zeros(2, 5, 6, 16)
    for a, b in (((0, 3), (2, 6)), ((1, 5), (0, 2)), ((0, 6), (3, 4))):
        with pytest.raises(ValueError, match="apart"):
            ops.rope_axes(buf[:, :, slice(*a)], buf[:, :, slice(*b)], pos, (2,), inplace=True)
    with pytest.raises(ValueError, match="apart"):
        ops.rope_axes(buf[..., :9], buf[..., 7:], pos, (2,), inplace=True)
    rows = torch.zeros(2, 6, 3, 16)
    with pytest.raises(ValueError, match="apart"):
        ops.rope_axes(rows[:, :5], rows[:, 1:], pos, (2,), inplace=True)
    with pytest.raises(ValueError, match="overlap"):
        ops.rope_axes(torch.zeros(20).as_strided((1, 5, 1, 8), (20, 2, 8, 1)), None, pos, (2,), inplace=True)
    for a, b in ((buf[:, :, :4], buf[:, :, 4:]), (buf[..., :8], buf[..., 8:]), (buf[:1], buf[1:]), (buf.transpose(0, 1)[:2].transpose(0, 1), buf[:, 3:]),
                 (buf[:, :, ::2], buf[:, :, 1::2])):
        with pytest.raises(RuntimeError, match="ROCm device tensors"):           # apart: the next check speaks
            ops.rope_axes(a, b, torch.zeros(a.shape[1], 1), (2,), inplace=True)


def test_whether_strided_tensors_meet_against_counting():
    rng = torch.Generator().manual_seed(2)
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (), generator=rng))
    met = 0
    for _ in range(3000):
        size = (2, 4)[pick(0, 1)]
        shapes = [tuple(pick(1, 4) for _ in range(3)) for _ in range(2)]
        strides = [tuple(pick(0, 30) if pick(0, 2) else pick(1, 4) for _ in range(3)) for _ in range(2)]
        apart = pick(-80, 80)
        places = [[sum(i * s for i, s in zip(ix, st)) * size for ix in torch.cartesian_prod(*(torch.arange(n) for n in sh)).tolist()]
                  for sh, st in zip(shapes, strides)]
        want = any(abs(a - b - apart) < size for a in places[0] for b in places[1])
        assert ops._meet(apart, size, shapes[0], strides[0], shapes[1], strides[1]) == want
        met += want
        if 0 not in strides[0]:
            assert ops._meets_itself(size, shapes[0], strides[0]) == (len(set(places[0])) < len(places[0]))
    assert 300 < met < 2700
