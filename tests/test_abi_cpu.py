"""CPU-side checks of the boundary: the C-ABI library loads here (no GPU) and exports every symbol
that include/mmlearn_hip.h declares; the product refuses CPU tensors."""

import os
import re
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def built():
    from mmlearn_amd import _lib

    if not os.path.exists(_lib.LIB_PATH):
        _lib.build()
    return _lib


def _declared_symbols():
    text = open(os.path.join(ROOT, "include", "mmlearn_hip.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(mmk_[a-z0-9_]+)\s*\(", text)))


def test_header_symbols_are_exported(built):
    declared = _declared_symbols()
    assert len(declared) >= 20
    out = subprocess.run(["nm", "-D", "--defined-only", built.LIB_PATH], capture_output=True, text=True, check=True).stdout
    exported = set(re.findall(r" T (mmk_[a-z0-9_]+)", out))
    missing = [s for s in declared if s not in exported]
    assert not missing, missing
    # the ctypes stub binds exactly the declared set
    assert sorted(built.EXPORTED_SYMBOLS) == declared


def test_shipped_library_reads_no_experiment_switches(built):
    """ablation / A-B switches (some of which give wrong results by design) exist only in
    -DMMK_DEBUG_SWITCHES builds; the shipped library does not even contain their names."""
    blob = open(built.LIB_PATH, "rb").read()
    for name in (b"MMK_SIM_DBG", b"MMK_TILE", b"MMK_LOADER", b"MMK_STAGES", b"MMK_STATS_TILE", b"MMK_ATTN_BWD7", b"MMK_ATTN_STAGED", b"MMK_FUSED_DBG", b"MMK_WGRAD_MFMA", b"MMK_WGRAD_PAIR",
                 b"MMK_ATTN_STAMPS", b"MMK_ATTN_SPLIT", b"MMK_MLP_GEMM_DBG", b"MMK_MLP_GEMM_STAMPS", b"MMK_WGRAD_TILE", b"MMK_WGRAD_MAP",
                 b"MMK_WIN_MIN_WGS", b"MMK_GRAD_UNIT_MAP"):
        assert name not in blob, name


def test_library_loads_without_gpu(built):
    lib = built.lib()
    assert lib.mmk_abi_version() == 8
    assert lib.mmk_kernel_name(3) == b"sim_stats"
    for k, name in enumerate(built.KERNEL_NAMES):
        assert lib.mmk_kernel_name(k).decode() == name


def test_struct_layout_matches_header(built):
    # sizeof(mmk_clip_dir) as laid out by the C compiler vs the ctypes mirror
    src = '#include <stdio.h>\n#include "mmlearn_hip.h"\nint main(){printf("%zu %zu", sizeof(mmk_clip_dir), sizeof(mmk_ema_entry));return 0;}'
    exe = "/tmp/_mmk_sizeof"
    subprocess.run(["gcc", "-x", "c", "-", "-I", os.path.join(ROOT, "include"), "-o", exe], input=src, text=True, check=True)
    a, b = map(int, subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split())
    import ctypes

    assert ctypes.sizeof(built.ClipDir) == a
    assert ctypes.sizeof(built.EmaEntry) == b


def test_no_cpu_fallback():
    from mmlearn_amd import ContrastiveLoss, LossPairSpec, find_matching_indices

    a = torch.randn(4, 8)
    ids = torch.zeros(4, 2, dtype=torch.long)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ContrastiveLoss()({"rgb_embedding": a, "text_embedding": a}, {"rgb": ids, "text": ids}, torch.tensor(1.0), [LossPairSpec(("rgb", "text"))])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        find_matching_indices(ids, ids)
    with pytest.raises(TypeError):
        find_matching_indices([(0, 0)], ids)
    with pytest.raises(ValueError):
        find_matching_indices(torch.zeros(3), ids)


def test_product_does_not_import_oracle():
    import ast

    bad = []
    for dirpath, _, files in os.walk(os.path.join(ROOT, "mmlearn_amd")):
        for f in files:
            if f.endswith(".py"):
                tree = ast.parse(open(os.path.join(dirpath, f)).read())
                for node in ast.walk(tree):
                    names = []
                    if isinstance(node, ast.Import):
                        names = [a.name for a in node.names]
                    elif isinstance(node, ast.ImportFrom) and node.module:
                        names = [node.module]
                    bad += [(f, n) for n in names if n.split(".")[0] == "oracle"]
    assert not bad, bad


def test_the_driver_build_entry_point_passes(built):
    """``__graft_entry__.build()`` is what the driver runs every round: it must build (a no-op here, the fixture did), load the library
    and agree with the ABI version of the header and the ctypes stub -- a hard-coded version number there broke it once."""
    import __graft_entry__ as g

    g.build()
    src = open(g.__file__).read()
    assert "_lib.ABI_VERSION" in src and built.lib().mmk_abi_version() == built.ABI_VERSION


def _error(built, rc):
    return rc, built.lib().mmk_last_error().decode()


def test_missing_operands_of_the_tower_operators_are_refused_on_the_host(built):
    """A null pointer comes back as an error; nothing is launched with it (the addresses here belong to nobody)."""
    import ctypes as C

    lib, at, st = built.lib(), 1 << 20, (C.c_int64 * 3)(64, 64, 64)
    # mmk_qk_norm_rotary_fwd / _bwd
    q, k, qo, ko = at, at, at, at
    for hole in range(6):
        a = [x if i != hole else None for i, x in enumerate((q, k, qo, ko, st, st))]
        rc, why = _error(built, lib.mmk_qk_norm_rotary_fwd(a[0], a[1], None, None, None, 0, None, 0, 0, a[2], a[3], 1, 1, 1, 1, 64, 0, 0, a[4], a[5], 1e-6, 1, 1, None))
        assert rc == -1 and "missing operand" in why, (hole, why)
    for hole in range(10):
        a = [x if i != hole else None for i, x in enumerate((at, at, at, at, at, at, st, st, st, st))]
        rc, why = _error(built, lib.mmk_qk_norm_rotary_bwd(a[0], a[1], None, None, None, 0, None, 0, 0, a[2], a[3], a[4], a[5], None, None, None, None, 1, 1, 1, 1, 64, 0, 0,
                                                          a[6], a[7], a[8], a[9], 1e-6, 1, 1, None))
        assert rc == -1 and "missing operand" in why, (hole, why)
    # mmk_newton_schulz
    for hole in range(4):
        p = built.NewtonSchulz()
        arrays = [(C.c_void_p * 2)(at, None if hole == i else at) for i in range(3)]
        p.src, p.dst, p.momenta = (C.cast(x, C.c_void_p) for x in arrays)
        p.count, p.rows, p.cols, p.steps, p.eps, p.weights, p.row_stride, p.col_stride = 2, 300, 300, 5, 1e-7, 1, 300, 1
        rc, why = _error(built, lib.mmk_newton_schulz(C.byref(p), at + 8 if hole == 3 else at, None))
        assert rc == -1 and ("aligned" if hole == 3 else "missing operand") in why, (hole, why)
    # mmk_rel_attn_fwd / _bwd
    def described(Lq=200, **how):
        p = built.RelAttn()
        borders = (C.c_int32 * 1)(3)
        p.q, p.k, p.v, p.table, p.borders = at, at, at, at, C.cast(borders, C.c_void_p)
        p.B, p.H, p.Hk, p.Lq, p.Lk, p.D, p.dtype, p.table_dtype = 1, 1, 1, Lq, 200, 64, 1, 1
        p.buckets, p.near_buckets, p.n_borders, p.max_distance = 4, 2, 1, 8
        for n, x in how.items():
            setattr(p, n, x)
        return p

    for how in (dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(borders=None)):
        rc, why = _error(built, lib.mmk_rel_attn_fwd(C.byref(described(**how)), at, None, None, at, None))
        assert rc == -1 and "missing" in why, (how, why)
        rc, why = _error(built, lib.mmk_rel_attn_bwd(C.byref(described(**how)), *[at] * 9, None))
        assert rc == -1 and "missing" in why, (how, why)
    for hole in (0, 1, 2, 3, 4, 5, 6, 8):     # (7: the table's gradient may be unwanted)
        rc, why = _error(built, lib.mmk_rel_attn_bwd(C.byref(described()), *[at if i != hole else None for i in range(9)], None))
        assert rc == -1 and "missing" in why, (hole, why)
    for hole in (0, 1, 3, 4, 5, 6, 8):
        rc, why = _error(built, lib.mmk_rel_attn_bwd(C.byref(described()), *[at if i != hole else at + 8 for i in range(9)], None))
        assert rc == -1 and "aligned" in why, (hole, why)
    rc, why = _error(built, lib.mmk_rel_attn_fwd(C.byref(described(near_buckets=2**31 - 1, n_borders=0)), at, None, None, at, None))
    assert rc == -1
