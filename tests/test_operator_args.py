"""The operators on dense 16-bit arrays without a GPU: their entry points are
there for every type, and refuse a null handle before anything else."""
import pytest

TYPES = ["f16_i32", "f16_i64", "bf16_i32", "bf16_i64"]


@pytest.mark.parametrize("t", TYPES)
def test_null_handle(pf, t):
    lib = pf.lib
    assert getattr(lib, "pf_spmm_" + t)(None, 1, 1, 0, None, None, None, 1, 1.0, None, 1, 0.0, None,
                                        1, None) == 1
    assert getattr(lib, "pf_sddmm_" + t)(None, 1, 1, 0, None, None, 1, 1.0, None, 1, None, 1, 0.0,
                                         None, None) == 1
    assert getattr(lib, "pf_gmm_" + t)(None, 1, 1, 1, 1, None, None, 1, None, 1, 1, 1, 1.0, 0.0,
                                       None, 1, None) == 1
    assert getattr(lib, "pf_gmm_wgrad_" + t)(None, 1, 1, 1, 1, None, None, 1, None, 1, 1.0, 0.0,
                                             None, 2, 1, 1, None) == 1
    assert b"null handle" in lib.pf_last_error()


@pytest.mark.parametrize("t", TYPES + ["f32_i32", "f32_i64"])
def test_distill_null_handle(pf, t):
    f = getattr(pf.lib, "pf_distill_" + t)
    assert f(None, 1, 1, 0, None, None, None, 1.0, None, 1, None, None, None, 1, None) == 1
    assert b"null handle" in pf.lib.pf_last_error()


def test_wgrad_output_type(pf):
    assert pf.lib.pf_gmm_wgrad_f16_i32(None, 1, 1, 1, 1, None, None, 1, None, 1, 1.0, 0.0, None, 8,
                                       1, 1, None) == 1
    assert b"dw_bytes" in pf.lib.pf_last_error()
