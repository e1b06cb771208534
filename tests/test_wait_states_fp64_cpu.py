"""The walk of tests/test_wait_states_cpu.py over the eigensolver: 18 wait states between v_mfma_f64_16x16x4_f64 and the first instruction
that touches its result."""

import pytest
import test_wait_states_cpu as walk

FP64 = {"v_mfma_f64_16x16x4_f64": 18}


def test_fp64_results_are_not_touched_too_early(tmp_path, monkeypatch):
    monkeypatch.setattr(walk, "NEEDED", {**walk.NEEDED, **FP64})
    kernels = 0
    for name, body in walk.disassemble("kf_eigh", tmp_path):
        kernels += any(op in FP64 for _, op, _, _ in body)
        assert not list(walk.violations(body)), name
    assert kernels > 0


@pytest.mark.parametrize("unit", ["kf_attention", "kf_norm", "kf_kernels", "kf_score_v2"])
def test_every_matrix_instruction_of_the_library_is_known_to_the_walk(unit, tmp_path):
    """An instruction without its number of wait states would be walked past."""
    found = {op for _, body in walk.disassemble(unit, tmp_path) for _, op, _, _ in body if op.startswith("v_mfma")}
    assert found <= {*walk.NEEDED, *FP64}, found
