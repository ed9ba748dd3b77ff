"""What the sequence operators refuse, on the CPU: nothing here launches a kernel."""
import ctypes as C

import pytest
import torch

from _dvae_pkg import dvae_amd

S, L = dvae_amd.sequence, dvae_amd._lib


def test_cpu_tensors_are_refused():
    with pytest.raises(L.DvaeHipError, match="no CPU fallback"):
        S.embed(torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(L.DvaeHipError, match="no CPU fallback"):
        S.gated_scan(torch.zeros(1, 3, 4), torch.zeros(1, 3, 4))
    with pytest.raises(L.DvaeHipError, match="no CPU fallback"):
        S.gated_step(torch.zeros(3, 4), torch.zeros(3, 4), torch.zeros(3, 4))


def test_wrong_types_and_ranks_are_refused():
    with pytest.raises(ValueError, match="2 dimensions"):
        S.embed(torch.zeros(4), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        S.embed(torch.zeros(3, 4, dtype=torch.float64), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="3 dimensions"):
        S.gated_scan(torch.zeros(3, 4), torch.zeros(3, 4))
    with pytest.raises(ValueError, match="2 dimensions"):
        S.gated_scan(torch.zeros(1, 3, 4), torch.zeros(1, 3, 4), torch.zeros(2, dtype=torch.int32))


def rc(name, *args):
    lib = L.load()
    code = getattr(lib, name)(*args)
    assert code < 0, "%s was not refused" % name
    return lib.dvae_last_error().decode()


def test_the_c_entries_refuse_bad_sizes_before_any_launch():
    p = C.c_void_p(4096)  # never read: every call below is refused on the host
    assert "element type" in rc("dvae_embed_fwd", p, 8, p, 0, p, 4, 4, 8, 1.0, 7, None)
    assert "row stride" in rc("dvae_embed_fwd", p, 7, p, 0, p, 4, 4, 8, 1.0, 0, None)
    assert "null" in rc("dvae_embed_fwd", None, 8, p, 0, p, 4, 4, 8, 1.0, 0, None)
    assert "tokens" in rc("dvae_embed_fwd", p, 8, p, 0, p, -1, 4, 8, 1.0, 0, None)
    assert "table" in rc("dvae_embed_fwd", p, 8, p, 0, p, 4, 0, 8, 1.0, 0, None)
    assert "row length" in rc("dvae_embed_fwd", p, 8, p, 0, p, 4, 4, 0, 1.0, 0, None)
    assert "null" in rc("dvae_embed_bwd", p, 8, p, 0, None, p, 4, 4, 8, 1.0, 0, None)
    assert "aligned" in rc("dvae_embed_bwd", p, 8, p, 0, p, C.c_void_p(4097), 4, 4, 8, 1.0, 0, None)
    assert "table" in rc("dvae_embed_bwd_ws_bytes", 4, 0, 8)
    assert "one length" in rc("dvae_scan_fwd", p, 8, p, 8, None, 0, None, p, p, None, p, 7, 2, 8, 0, None)
    assert "null" in rc("dvae_scan_fwd", p, 8, p, 8, None, 0, None, p, None, None, p, 8, 2, 8, 0, None)
    assert "row stride" in rc("dvae_scan_fwd", p, 8, p, 4, None, 0, None, p, p, None, p, 8, 2, 8, 0, None)
    assert "channels" in rc("dvae_scan_fwd", p, 8, p, 8, None, 0, None, p, p, None, p, 8, 2, 0, 0, None)
    assert "null" in rc("dvae_scan_bwd", p, 8, p, 8, None, 0, None, None, p, 8, p, p, p, p, p, 8, 2, 8, 0, None)
    assert "element type" in rc("dvae_scan_bwd", p, 8, p, 8, None, 0, None, p, p, 8, p, p, p, p, p, 8, 2, 8, 3, None)
    assert "rows" in rc("dvae_scan_ws_bytes", -1, 8)
    assert "pool" in rc("dvae_scan_step", p, 8, p, 8, p, 8, 3, None, 0, p, 4, 8, 0, None)
    assert "65536" in rc("dvae_scan_step", p, 8, p, 8, p, 8, 1 << 20, p, 0, p, 65537, 8, 0, None)
    assert "row stride" in rc("dvae_scan_fwd", p, (1 << 23) + 1, p, 8, None, 0, None, p, p, None, p, 8, 2, 8, 0, None)
    assert "row stride" in rc("dvae_scan_step", p, 8, p, 8, p, 7, 4, None, 0, p, 4, 8, 0, None)
    assert "null" in rc("dvae_scan_step", p, 8, p, 8, None, 8, 4, None, 0, p, 4, 8, 0, None)


def test_workspace_sizes_grow_with_the_work():
    lib = L.load()
    assert lib.dvae_scan_state_floats(0, 8) == 0 and lib.dvae_scan_state_floats(1, 8) == 8
    assert lib.dvae_scan_state_floats(1 << 39, 8) > 1 << 32  # 64 bits all the way
    assert lib.dvae_embed_bwd_ws_bytes(1 << 20, 1 << 20, 1 << 12) > 1 << 30


def test_matrix_descriptions_are_checked_before_any_launch():
    def desc(g=4096, out=4096, ld_g=8, ld_out=8, rows=8, cols=8):
        return (L.MatrixDesc * 1)(L.MatrixDesc(g, out, ld_g, ld_out, rows, cols))
    abc = (C.c_float * 15)(*[3.4445, -4.7750, 2.0315] * 5)
    p = C.c_void_p(4096)
    assert "null" in rc("dvae_orthogonalize", None, 1, 5, abc, p, 0, None)
    assert "element type" in rc("dvae_orthogonalize", desc(), 1, 5, abc, p, 5, None)
    assert "steps" in rc("dvae_orthogonalize", desc(), 1, 0, abc, p, 0, None)
    assert "sides" in rc("dvae_orthogonalize", desc(rows=0), 1, 5, abc, p, 0, None)
    assert "sides" in rc("dvae_orthogonalize_ws_bytes", desc(cols=40000), 1, 0)
    assert "row stride" in rc("dvae_orthogonalize", desc(ld_g=7), 1, 5, abc, p, 0, None)
    assert "null" in rc("dvae_orthogonalize", desc(out=None), 1, 5, abc, p, 0, None)
    assert "aligned" in rc("dvae_orthogonalize", desc(), 1, 5, abc, C.c_void_p(4097), 0, None)
    assert "singular" in rc("dvae_orthogonalize", desc(), 1, 5, (C.c_float * 15)(*[4.0, 0.0, 0.0] * 5), p, 0, None)
    assert "64" in rc("dvae_muon_begin_f32", p, p, p, p, p, p, 100, 0.9, 1, 1e-3, 0.9, 0.999, 1e-8, 1, 0, None)
    assert "step" in rc("dvae_muon_begin_f32", p, p, p, p, p, p, 128, 0.9, 1, 1e-3, 0.9, 0.999, 1e-8, 0, 0, None)
    assert "null" in rc("dvae_muon_apply_f32", p, None, p, 128, 0.1, 0.0, None)


def test_the_matrix_description_has_the_header_layout(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "layout.c"
    names = [f for f, _ in L.MatrixDesc._fields_]
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"dvae_hip.h\"\nint main(void) { printf(\"%zu\", sizeof(dvae_matrix_desc));\n"
                   + "".join('printf(" %%zu", offsetof(dvae_matrix_desc, %s));\n' % f for f in names) + "return 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out] == [C.sizeof(L.MatrixDesc)] + [getattr(L.MatrixDesc, f).offset for f in names]


def test_the_host_module_uses_declared_functions_and_has_no_fallback(monkeypatch, tmp_path):
    ops = L.load_sequence_ops()
    assert set(ops.functions) <= set(L.SIGNATURES)
    monkeypatch.setattr(L, "HERE", str(tmp_path))
    with pytest.raises(L.DvaeHipError, match="no fallback"):
        L.load_sequence_ops()


def test_half_products_are_refused_but_for_bf16():
    d = (L.MatrixDesc * 1)(L.MatrixDesc(4096, 4096, 600, 600, 600, 600))
    abc = (C.c_float * 15)(*[3.4445, -4.7750, 2.0315] * 5)
    assert "half products" in rc("dvae_orthogonalize", d, 1, 5, abc, C.c_void_p(4096), 16, None)
    assert "half products" in rc("dvae_orthogonalize_ws_bytes", d, 1, 18)
    lib = L.load()
    full, half = lib.dvae_orthogonalize_ws_bytes(d, 1, 1), lib.dvae_orthogonalize_ws_bytes(d, 1, 17)
    assert 0 < half < full  # one plane of A, B and the turned X
    small = (L.MatrixDesc * 1)(L.MatrixDesc(4096, 4096, 600, 600, 511, 600))
    assert lib.dvae_orthogonalize_ws_bytes(small, 1, 1) == lib.dvae_orthogonalize_ws_bytes(small, 1, 17)
    mixed = (L.MatrixDesc * 34)(*[L.MatrixDesc(4096, 4096, 600, 600, 511 + k % 2, 600) for k in range(34)])
    seventeen = (L.MatrixDesc * 17)(*[L.MatrixDesc(4096, 4096, 600, 600, 511, 600) for k in range(17)])
    assert lib.dvae_orthogonalize_ws_bytes(mixed, 34, 17) == lib.dvae_orthogonalize_ws_bytes(seventeen, 17, 17)


@pytest.mark.parametrize("extra", [0, 5])
def test_sizes_past_32_bits_are_refused_not_cut(extra):
    """the library takes rows of a step and row lengths in 32 bits; tensors without memory, nothing is launched"""
    ops, n = S._native(), 2 ** 32 + extra

    def meta(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="meta")

    ids, off = meta(2, dtype=torch.int64), meta(2, dtype=torch.int64)
    with pytest.raises(L.DvaeHipError, match="elements of a row: %d are not supported" % n):
        ops.embed(meta(1, n), ids, 1.0)
    with pytest.raises(L.DvaeHipError, match="channels: %d are not supported" % n):
        ops.scan(meta(1, n), meta(1, n), off, None, 1)
    with pytest.raises(L.DvaeHipError, match="rows: %d are not supported" % n):
        ops.step(meta(1, 1).expand(n, 1), meta(1, 1).expand(n, 1), meta(n, 1), None)
    with pytest.raises(L.DvaeHipError, match="channels: %d are not supported" % n):
        ops.step(meta(1, n), meta(1, n), meta(1, n), None)


def test_many_newton_schulz_steps_are_refused_before_they_are_listed():
    with pytest.raises(ValueError, match="steps"):
        dvae_amd.optim.orthogonalize(torch.zeros(3, 3), steps=2 ** 32 + 5)


def test_tensors_with_a_tangent_are_refused():
    """forward-mode derivatives would be dropped; also where nothing is recorded for the backward pass"""
    import torch.autograd.forward_ad as fwd
    ops, t = S._native(), torch.ones(3, 4)
    ids, off = torch.zeros(2, dtype=torch.int64), torch.tensor([0, 3])
    with fwd.dual_level():
        d = fwd.make_dual(t, t)
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in (lambda: ops.embed(d, ids, 1.0), lambda: ops.scan(d, t, off, None, 1), lambda: ops.scan(t, d, off, None, 1),
                             lambda: ops.scan(t, t, off, d[:1], 1), lambda: ops.step(d, t, t, None), lambda: ops.step(t, d, t, None),
                             lambda: ops.step(t, t, d, None), lambda: dvae_amd.optim.orthogonalize(d),
                             lambda: dvae_amd.optim.orthogonalize([t], out=[d])):
                    with pytest.raises(ValueError, match="forward-mode"):
                        call()


def test_inputs_are_copied_only_where_another_output_shares_their_memory():
    apart = dvae_amd.optim._kept_apart
    flat = torch.zeros(10, 4, 6)
    mats = list(flat)

    def copied(srcs, outs):
        return [a.data_ptr() != s.data_ptr() for a, s in zip(apart(srcs, outs), srcs)]

    assert copied(mats, mats) == [False] * 10 and copied(mats, list(torch.zeros(10, 4, 6))) == [False] * 10
    assert copied(mats, mats[1:] + mats[:1]) == [True] * 10
    assert copied(mats, mats[:8] + [mats[9], mats[8]]) == [False] * 8 + [True] * 2
    assert copied(mats, mats[:8] + [mats[8], torch.zeros(4, 6)]) == [False] * 10
    wide = torch.zeros(4, 100)
    assert copied([wide[:, :50], mats[0]], [mats[0], wide[:, 50:]]) == [True, True]
    assert copied([mats[3][:2], mats[3][2:], mats[4]], [wide[:2, :6], mats[5][:2], mats[3]]) == [True, True, False]


def accepts(triples):
    lib = L.load()
    flat = [v for t in triples for v in t]
    return lib.dvae_orthogonalize((L.MatrixDesc * 1)(), 0, len(triples), (C.c_float * len(flat))(*flat), None, 0, None) == 0


def walk(triples, samples):
    """largest singular value and largest |b s^2 + c s^4| over the steps, by following samples of [0, 1]"""
    import numpy as np
    s, most, big = samples, 0.0, 0.0
    for t, (a, b, c) in enumerate(np.float32(triples).astype(np.float64)):
        l = s * s
        big = max(big, float(np.abs(b * l + c * l * l).max()) * (2 if t == 0 else 1))
        s = np.abs(s * (a + b * l + c * l * l))
        most = max(most, float(s.max()))
    return most, big


def test_the_bound_on_coefficients_agrees_with_a_walk_over_samples():
    import numpy as np
    rng, samples = np.random.default_rng(0), np.linspace(0.0, 1.0, 20001)
    seen = [0, 0]
    for k in range(3000):
        n = int(rng.integers(1, 3))
        scale = rng.choice([1.0, 0.5, 0.25])
        triples = (rng.uniform(-1, 1, (n, 3)) * [4, 6, 3] * scale).round(3)
        triples[rng.random((n, 3)) < 0.1] = 0
        most, big = walk(triples, samples)
        # what the samples reach is reached; a point is at most 1 / 40000 from a sample and the slopes are at most 37 and 61,
        # so that the samples fall short by less than 0.06
        if most >= 1.95 or big >= 7.5:
            assert not accepts(triples), (triples, most, big)
            seen[0] += 1
        elif most < 1.2 and big < 7:
            assert accepts(triples), (triples, most, big)
            seen[1] += 1
    assert min(seen) > 200, seen


def test_coefficients_whose_peak_lies_between_samples_are_refused():
    quintic = (3.4445, -4.7750, 2.0315)
    assert accepts([quintic] * 5) and accepts([quintic] * 32) and accepts([(1.5, -0.5, 0.0)] * 20) and accepts([(2.0, -1.5, 0.5)] * 12)
    assert accepts([(0.0, 0.0, 0.0)] * 3) and accepts([(1.0, 0.0, 0.0)] * 32)
    # all but singular values next to 1 shrink, those grow to 1.94 and then to 5: 4097 samples of [0, 1] miss them
    narrow = [(0.6994, 1.0379, 0.2027), (0.1041, 0.0456, -0.0901), (-0.2401, 0.0324, 0.0787), (-0.1292, 0.4203, -0.1734),
              (0.1413, -0.0517, 0.0743), (0.9625, -3.9394, 0.9085)]
    import numpy as np
    assert walk(narrow, np.linspace(0.0, 1.0, 4097))[0] < 1.95 and walk(narrow, np.linspace(0.999, 1.0, 100001))[0] > 5
    assert accepts(narrow[:5]) and not accepts(narrow)
    for bad in ((float("nan"), 0.0, 0.0), (0.0, float("inf"), 0.0), (0.0, 0.0, float("-inf")), (1.96, 0.0, 0.0), (-1.96, 0.0, 0.0)):
        assert not accepts([bad])
    # p stays below 1.84, but the first step's B, which carries the rest of the norm (up to 2), reaches 8
    assert "b and c" in rc("dvae_orthogonalize", (L.MatrixDesc * 1)(), 0, 1, (C.c_float * 3)(4.5, -4.0, 0.0), None, 0, None)


def test_what_no_launch_can_hold_is_refused_before_the_first_one():
    """a grid has less than 2^32 threads"""
    p, lib = C.c_void_p(4096), L.load()
    most = (1 << 28) - 32
    assert lib.dvae_embed_bwd_ws_bytes(most, 8, 8) > 0 and "tokens" in rc("dvae_embed_bwd_ws_bytes", most + 1, 8, 8)
    assert lib.dvae_embed_bwd_ws_bytes(8, (1 << 30) - 64, 8) > 0 and "table" in rc("dvae_embed_bwd_ws_bytes", 8, (1 << 30) - 63, 8)
    assert "tokens" in rc("dvae_embed_bwd", p, 8, p, 0, p, p, most + 1, 4, 8, 1.0, 0, None)
    assert "too many" in rc("dvae_embed_bwd", p, 4096, p, 0, p, p, most, 4, 4096, 1.0, 0, None)
    for name, args in (("dvae_scan_fwd", (p, 65, p, 65, p, 0, None, p, p, None, p)), ("dvae_scan_bwd", (p, 65, p, 65, p, 0, None, p, p, 65, p, p, p, p, p))):
        assert "too many" in rc(name, *args, 1 << 30, 2, 64, 0, None)
        assert "too many" in rc(name, *args, 1 << 29, 2, 65, 0, None)  # two slabs of 64 channels
        assert "too many" in rc(name, *args, 300, 1 << 26, 64, 0, None)
        assert "too many" in rc(name, *args, 30, 1 << 26, 64, 0, None)  # one tile
        assert "too many" in rc(name, *args, 0, 1 << 26, 64, 0, None)
    assert "too many" in rc("dvae_scan_step", p, 1 << 13, p, 1 << 13, p, 1 << 13, 1 << 24, None, 0, p, 1 << 24, 1 << 13, 0, None)


def test_orthogonalize_refuses_an_output_that_needs_a_gradient():
    """it would keep the gradient of what it held before"""
    m, leaf = torch.ones(3, 4), torch.ones(3, 4, requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="no_grad"):
            dvae_amd.optim.orthogonalize(m, out=out)
        with pytest.raises(ValueError, match="no_grad"):
            dvae_amd.optim.orthogonalize([m, m], out=[m.clone(), out])
        with torch.no_grad(), pytest.raises(L.DvaeHipError, match="no CPU fallback"):
            dvae_amd.optim.orthogonalize(m, out=out)
