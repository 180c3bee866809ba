"""The build's check of the wait states behind matrix instructions, on short
pieces of assembly."""

import pytest

from ns_fps_amd.build import matrix_hazards

BF16 = "v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], 0"
F32 = "v_mfma_f32_16x16x4_f32 v[0:3], v4, v8, 0"
WIDE = "v_mfma_f32_32x32x8_bf16 v[0:15], v[16:17], v[18:19], 0"


def hazards(*lines):
    body = "".join(f"{ln}\n" if ln.endswith(":") else f"\t{ln}\n" for ln in lines)
    return matrix_hazards(f"\t.text\n_Zf:\n{body}\ts_endpgm\n.Lfunc_end0:\n")


@pytest.mark.parametrize("user", [
    "v_add_f32_e32 v20, v3, v21", "v_add_f32_e32 v3, v20, v21", "v_mov_b32_e32 v1, 0",
    "v_mfma_f32_16x16x32_bf16 v[12:15], v[0:3], v[8:11], 0",
    "v_mfma_f32_16x16x32_bf16 v[12:15], v[4:7], v[0:3], v[12:15]",
    "v_mfma_f32_16x16x4_f32 v[12:15], v2, v8, 0", "global_store_dwordx4 v20, v[0:3], s[0:1]",
    "global_load_dwordx4 v[0:3], v20, s[0:1]", "ds_read_b128 v[0:3], v20", "ds_write_b32 v20, v2",
    "ds_read_b64_tr_b16 v[2:3], v20", "ds_bpermute_b32 v20, v21, v0", "buffer_load_dword v2, v20, s[0:3], 0"])
@pytest.mark.parametrize("product,states", [(BF16, 8), (F32, 10)])
def test_users_of_sums_are_found_until_they_are_waited_for(product, states, user):
    assert len(hazards(product, user)) == 1
    assert len(hazards(product, f"s_nop {states - 2}", user)) == 1
    assert hazards(product, f"s_nop {states - 1}", user) == []
    assert hazards(product, *["s_mov_b32 s0, 0"] * states, user) == []


@pytest.mark.parametrize("other", [
    "v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]",   # adds to the sums
    "v_mfma_f32_16x16x32_bf16 v[12:15], v[4:7], v[8:11], v[0:3]",
    "v_add_f32_e32 v20, v4, v21", "s_add_u32 s0, s1, s2", "global_load_dwordx4 v[20:23], v24, s[0:1]"])
def test_others_are_not(other):
    assert hazards(BF16, other, "s_nop 7") == []


def test_a_second_product_is_waited_for_itself():
    add = "v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]"
    assert len(hazards(BF16, add, "s_nop 6", "v_add_f32_e32 v20, v0, v0")) == 1
    assert hazards(BF16, add, "s_nop 7", "v_add_f32_e32 v20, v0, v0") == []


def test_readers_behind_branches_are_found():
    read = "v_add_f32_e32 v20, v0, v21"
    assert len(hazards(BF16, "s_cbranch_scc1 .LBB0_1", "s_nop 7", ".LBB0_1:", read)) == 1
    assert hazards(BF16, "s_cbranch_scc1 .LBB0_1", "s_nop 7", ".LBB0_1:", "s_nop 7", read) == []
    # the product at a loop's end, its reader at the loop's start
    assert len(hazards(".LBB0_1:", read, "s_nop 7", BF16, "s_cbranch_scc1 .LBB0_1")) == 1


def test_a_path_with_fewer_sums_left_hides_no_other():
    """Both paths reach the reader with 12 states; the first has replaced the
    sums that it reads."""
    assert len(hazards(WIDE, "s_cbranch_scc1 .LBB0_1", BF16.replace("v[4:7], v[8:11]",
                                                                    "v[20:23], v[24:27]"),
                       "s_nop 9", "s_branch .LBB0_2", ".LBB0_1:", "s_nop 11", ".LBB0_2:",
                       "v_add_f32_e32 v30, v0, v0")) == 1
