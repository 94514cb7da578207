"""What the compiler made of the kernels of rows in 8 bits, of the layers on them and of the norm, from the code objects in the built library."""
from test_feature_registers import kernels


def test_no_vector_register_is_spilled(hip_library):
    names = ("linear8_", "rms_norm", "norm_join", "pack8_", "unpack8_")
    ours = {k[".name"]: k for k in kernels(hip_library) if any(n in k[".name"] for n in names)}
    assert len(ours) > 200
    assert not {n: k[".vgpr_spill_count"] for n, k in ours.items() if k[".vgpr_spill_count"]}


def test_two_workgroups_of_eight_waves_share_a_cu(hip_library):
    """Those whose LDS lets them: 128 registers a lane, four waves a SIMD."""
    ours = [k for k in kernels(hip_library) if "linear8_" in k[".name"] and k[".max_flat_workgroup_size"] == 512 and "few" not in k[".name"]]
    tight = [k for k in ours if 2 * k[".group_segment_fixed_size"] <= 160 << 10]
    assert len(tight) >= 6 and all(k[".vgpr_count"] <= 128 for k in tight), [(k[".name"], k[".vgpr_count"]) for k in tight]
