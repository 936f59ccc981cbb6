"""tools/isa_barrier_audit.py on what the library is made of: every source whose kernels have a barrier, written out or through
lds_barrier() of operator_common.h, compiled with the flags it is shipped with."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "ur-mvo_amd", "csrc")


@pytest.fixture(scope="module")
def A():
    spec = importlib.util.spec_from_file_location("isa_barrier_audit", os.path.join(ROOT, "tools", "isa_barrier_audit.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("op", ["s_load_dword s0, s[2:3], 0x0", "s_buffer_load_dwordx2 s[0:1], s[4:7], 0x0", "s_memtime s[0:1]", "s_memrealtime s[0:1]"])
def test_scalar_memory_returns_out_of_order(A, op):
    """a counted wait says nothing about an LDS write once a scalar memory operation is in flight beside it"""
    def hits(body):
        return A.audit_text("kern:\n" + body + "\n\ts_endpgm\n.Lfunc_end0:\n")
    assert len(hits(f"\tds_write_b32 v0, v1\n\t{op}\n\ts_waitcnt lgkmcnt(1)\n\ts_barrier")) == 1
    assert hits(f"\tds_write_b32 v0, v1\n\t{op}\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier") == []
    for other in ("s_add_u32 s0, s1, s2", "s_setprio 1", "s_cmp_lg_u32 s0, 0", "s_and_saveexec_b64 s[0:1], vcc", "s_mov_b32 m0, s0"):
        assert hits(f"\tds_write_b32 v0, v1\n\tds_read_b32 v2, v0\n\t{other}\n\ts_waitcnt lgkmcnt(1)\n\ts_barrier") == [], other


def _make(name):
    """a variable of the Makefile"""
    for line in open(os.path.join(CSRC, "Makefile")):
        if line.startswith(name + " :="):
            return line.split(":=")[1].split()
    raise KeyError(name)


@pytest.mark.parametrize("source", [s for s in _make("OPERATORS") if s != "attention_api.hip"])
def test_no_barrier_of_the_operators_is_reached_with_an_lds_write_in_flight(A, source):
    """their barriers are all lds_barrier()'s, in headers: the sources' own text need not name one"""
    text = A.compile_to_asm(os.path.join(CSRC, source), _make("NO_PACKED_FP32"))
    assert "s_barrier" in text and A.audit_text(text) == []
    assert not any(op in text for op in ("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32"))


@pytest.mark.parametrize("source", ["sg_kernels.hip", "attn_h2.hip"])
def test_no_kernel_is_built_with_packed_fp32_instructions(A, source):
    """the sources whose code invites them (pairs of floats), with the flags every source is compiled with"""
    flags = _make("NO_PACKED_FP32")
    assert "$(NO_PACKED_FP32)" in _make("CXXFLAGS")
    text = A.compile_to_asm(os.path.join(CSRC, source), flags)
    assert not any(op in text for op in ("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32"))
