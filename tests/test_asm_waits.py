"""The build's check of scalar operands of vector-memory instructions in asm statements (tools/audit_asm_waits.py): on
small listings, and on the compiler's assembly of the kernels that issue such instructions, where it has been built."""
import os
import sys

import pytest

ROOT = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..")
sys.path.insert(0, os.path.join(ROOT, "tools"))
import audit_asm_waits as A  # noqa: E402

BUILD = os.path.join(ROOT, "symbolic-music-generation_amd", "csrc", "build")
LOAD = "\t;;#ASMSTART\n\ts_mov_b32 m0, s3\n\ts_nop {}\n\tbuffer_load_dwordx4 v1, s[8:11], {} offen lds\n\t;;#ASMEND\n"


def states(text):
    return [n for _, n in A.violations(("f:\n" + text + "\ts_endpgm\n").splitlines(True))]


@pytest.mark.parametrize("write,nop,soff,want", [
    ("v_readlane_b32 s21, v255, 19", 0, "s21", [2]), ("v_readlane_b32 s21, v255, 19", 3, "s21", []),
    ("v_readfirstlane_b32 s9, v4", 1, "0", [3]), ("v_readfirstlane_b32 s12, v4", 0, "0", []),
    ("s_mov_b32 s21, s4", 0, "s21", []), ("v_add_co_u32_e64 v2, s[20:21], v3, v4", 0, "s21", [2]),
    ("v_readlane_b32 s21, v255, 19\n\ts_add_i32 s4, s5, s6\n\tv_mov_b32_e32 v9, v8", 0, "s21", [4]),
    ("v_readlane_b32 s21, v255, 19\n\ts_add_i32 s4, s5, s6\n\tv_mov_b32_e32 v9, v8\n\ts_nop 0", 0, "s21", [])])
def test_distance(write, nop, soff, want):
    assert states("\t" + write + "\n" + LOAD.format(nop, soff)) == want


def test_over_branches():
    jump = "\tv_readlane_b32 s21, v255, 19\n\ts_cbranch_scc1 .LBB0_2\n" + "\ts_mov_b32 s1, 0\n" * 6
    assert states(jump + ".LBB0_2:\n" + LOAD.format(0, "s21")) == [3]
    away = "\tv_readlane_b32 s21, v255, 19\n\ts_branch .LBB0_3\n.LBB0_2:\n"
    assert states(away + LOAD.format(0, "s21") + ".LBB0_3:\n") == []
    loop = ".LBB0_1:\n" + LOAD.format(0, "s21") + "\tv_readlane_b32 s21, v255, 19\n\ts_cbranch_scc1 .LBB0_1\n"
    assert states(loop) == [3]


def test_instructions_that_the_compiler_sees_are_its_business():
    assert states("\tv_readlane_b32 s21, v255, 19\n\tbuffer_load_dwordx4 v[0:3], v1, s[8:11], s21 offen\n") == []


@pytest.mark.parametrize("name", ["attn", "attn_drop", "gemm_rs", "gemm_os", "gemm_skinny", "attn_decode_mx"])
def test_kernels(name):
    path = os.path.join(BUILD, name + ".s")
    if not os.path.exists(path):
        pytest.skip("the kernels' assembly has not been built here")
    with open(path) as f:
        assert A.violations(f) == []
