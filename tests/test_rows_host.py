"""Argument checks of the products whose weights are chosen row by row: they come before the device is looked for."""
import pytest

P = 1 << 20  # a well-aligned address nothing reads


def lora(lib, ptrs=None, **kw):
    d = dict(m=4, n=16, k=16, rank=8, adapters=2, ab_dtype=lib.BF16, c_dtype=lib.F32, ldx=0, ldy=0)
    tuning = kw.pop("tuning", (0, 0))
    d.update(kw)
    desc = lib.lora_desc(**d)
    desc.tuning[0], desc.tuning[1] = tuning
    lib.lora_tn(desc, *(ptrs or [P] * 8))


def backward(lib, ptrs=None, **kw):
    d = dict(m=4, n=16, k=16, rank=8, adapters=2, ab_dtype=lib.BF16, c_dtype=lib.F32, ldx=0, ldy=0)
    d.update(kw)
    lib.lora_tn_backward(lib.lora_desc(**d), *(ptrs or [P] * 12))


def moe(lib, ptrs=None, **kw):
    d = dict(tokens=2, experts=4, top=2, d=16, f=16, dtype=lib.BF16)
    d.update(kw)
    lib.moe_tn(lib.moe_desc(**d), *(ptrs or [P] * 7))


LORA_SIZES = [
    (dict(m=-1), "lora_tn: invalid size -1x16x16"),
    (dict(n=0), "lora_tn: invalid size 4x0x16"),
    (dict(k=0), "lora_tn: invalid size 4x16x0"),
    (dict(k=12), "lora_tn: k must be a multiple of 8, got 12"),
    (dict(rank=0), "lora_tn: rank must be a multiple of 8 in 8..128, got 0"),
    (dict(rank=12), "lora_tn: rank must be a multiple of 8 in 8..128, got 12"),
    (dict(rank=136), "lora_tn: rank must be a multiple of 8 in 8..128, got 136"),
    (dict(adapters=0), "lora_tn: at least one adapter is needed, got 0"),
    (dict(adapters=1 << 28, n=16), "lora_tn: 268435456 adapters of 16 rows are more than 2^31 rows"),
    (dict(ldx=20), "lora_tn: ldx must be 0 or a multiple of 8 of at least k = 16, got 20"),
    (dict(ldx=8), "lora_tn: ldx must be 0 or a multiple of 8 of at least k = 16, got 8"),
    (dict(ldy=15), "lora_tn: ldy must be 0 or at least n = 16, got 15"),
    (dict(m=(1 << 30) + 1), "lora_tn: m, n and k may be at most 2^30, got 1073741825x16x16"),
    (dict(tuning=(7, 0)), "lora_tn: tuning[0] must be 0, 1 (with m <= 128) or 2 to 6, got 7"),
    (dict(tuning=(1, 0), m=129), "lora_tn: tuning[0] must be 0, 1 (with m <= 128) or 2 to 6, got 1"),
]


@pytest.mark.parametrize("change,message", LORA_SIZES)
def test_lora_refuses_sizes(lib, change, message):
    with pytest.raises(lib.CuteB200Error) as e:
        lora(lib, **change)
    assert e.value.status == lib.ERR_INVALID_ARGUMENT and e.value.message == message


def test_lora_refuses_types_and_pointers(lib):
    with pytest.raises(lib.CuteB200Error) as e:
        lora(lib, ab_dtype=lib.F32)
    assert e.value.message == "lora_tn takes f16 or bf16 operands, not dtype 2"
    with pytest.raises(lib.CuteB200Error) as e:
        lora(lib, c_dtype=lib.I32)
    assert e.value.message == "lora_tn writes f32, f16 or bf16, not dtype 3"
    names = ["X", "W", "A", "B", "ids", "scale", "Y", "the workspace"]
    aligned = [16, 16, 16, 16, 4, 4, 4, 256]
    for i, (name, align) in enumerate(zip(names, aligned)):
        for value, status, message in ((0, lib.ERR_NULL_POINTER, f"lora_tn: {name} is null"),
                                       (P + align // 2, lib.ERR_MISALIGNED, f"lora_tn: {name} must be {align}-byte aligned")):
            ptrs = [P] * 8
            ptrs[i] = value
            with pytest.raises(lib.CuteB200Error) as e:
                lora(lib, ptrs)
            assert e.value.status == status and e.value.message == message


def test_backward_refusals(lib):
    for change, message in ((dict(n=20), "lora_tn_backward: n must be a multiple of 8, got 20"),
                            (dict(ldy=20), "lora_tn_backward: ldy must be a multiple of 8, got 20"),
                            (dict(rank=9), "lora_tn_backward: rank must be a multiple of 8 in 8..128, got 9")):
        with pytest.raises(lib.CuteB200Error) as e:
            backward(lib, **change)
        assert e.value.status == lib.ERR_INVALID_ARGUMENT and e.value.message == message
    # dA and dB come together
    for i, name in ((9, "dA"), (10, "dB")):
        ptrs = [P] * 12
        ptrs[i] = 0
        with pytest.raises(lib.CuteB200Error) as e:
            backward(lib, ptrs)
        assert e.value.status == lib.ERR_NULL_POINTER and e.value.message == f"lora_tn_backward: {name} is null"
    for i, name in ((0, "X"), (1, "W transposed"), (6, "dY"), (7, "the forward workspace"), (11, "the workspace")):
        ptrs = [P] * 12
        ptrs[i] = 0
        with pytest.raises(lib.CuteB200Error) as e:
            backward(lib, ptrs)
        assert e.value.status == lib.ERR_NULL_POINTER and e.value.message == f"lora_tn_backward: {name} is null"


def test_workspaces_grow_with_the_call(lib):
    small, large = lib.lora_desc(1, 16, 16, 8, 2, lib.BF16, lib.BF16), lib.lora_desc(1000, 16, 16, 128, 2, lib.BF16, lib.BF16)
    assert 0 < lib.lora_workspace(small) < lib.lora_workspace(large)
    assert 0 < lib.lora_backward_workspace(small) < lib.lora_backward_workspace(large)
    assert lib.lora_workspace(large) >= 1000 * 2 * 128 * 2
    with pytest.raises(lib.CuteB200Error):
        lib.lora_workspace(lib.lora_desc(1, 16, 15, 8, 2, lib.BF16, lib.BF16))
    assert 0 < lib.moe_workspace(lib.moe_desc(1, 4, 2, 16, 16, lib.F16)) <= lib.moe_workspace(lib.moe_desc(64, 4, 2, 16, 16, lib.F16))


MOE_SIZES = [
    (dict(tokens=-1), "moe_tn takes 0 to 64 tokens, got -1"),
    (dict(tokens=65), "moe_tn takes 0 to 64 tokens, got 65"),
    (dict(experts=0), "moe_tn takes 1 to 512 experts, got 0"),
    (dict(experts=513), "moe_tn takes 1 to 512 experts, got 513"),
    (dict(top=0), "moe_tn: top must be 1 to 16 and at most the 4 experts, got 0"),
    (dict(top=5), "moe_tn: top must be 1 to 16 and at most the 4 experts, got 5"),
    (dict(top=17, experts=32), "moe_tn: top must be 1 to 16 and at most the 32 experts, got 17"),
    (dict(d=12), "moe_tn: d and f must be positive multiples of 8, got 12 and 16"),
    (dict(f=0), "moe_tn: d and f must be positive multiples of 8, got 16 and 0"),
    (dict(experts=512, f=1 << 22), "moe_tn: 512 experts of 4194304 rows are more than 2^31 rows"),
    (dict(dtype=2), "moe_tn takes f16 or bf16, not dtype 2"),
]


@pytest.mark.parametrize("change,message", MOE_SIZES)
def test_moe_refuses_sizes(lib, change, message):
    with pytest.raises(lib.CuteB200Error) as e:
        moe(lib, **change)
    assert e.value.status == lib.ERR_INVALID_ARGUMENT and e.value.message == message


def test_moe_refuses_pointers(lib):
    names = ["X", "the router", "the gate weights", "the up weights", "the down weights", "Y", "the workspace"]
    for i, name in enumerate(names):
        align = 256 if i == 6 else 16
        for value, status, message in ((0, lib.ERR_NULL_POINTER, f"moe_tn: {name} is null"),
                                       (P + 8, lib.ERR_MISALIGNED, f"moe_tn: {name} must be {align}-byte aligned")):
            ptrs = [P] * 7
            ptrs[i] = value
            with pytest.raises(lib.CuteB200Error) as e:
                moe(lib, ptrs)
            assert e.value.status == status and e.value.message == message


def test_null_descriptors(lib):
    L = lib.load()
    assert L.cute_b200_lora_tn(None, *[P] * 8, None) == lib.ERR_NULL_POINTER
    assert L.cute_b200_lora_tn_backward(None, *[P] * 12, None) == lib.ERR_NULL_POINTER
    assert L.cute_b200_moe_tn(None, *[P] * 7, None) == lib.ERR_NULL_POINTER
    assert L.cute_b200_lora_workspace(None, None, None) == lib.ERR_NULL_POINTER
    assert L.cute_b200_moe_workspace(None, None) == lib.ERR_NULL_POINTER


def test_valid_arguments_reach_the_device(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("only without a GPU: the addresses are not real")
    for call in (lora, backward, moe):
        with pytest.raises(lib.CuteB200Error) as e:
            call(lib)
        assert e.value.status == lib.ERR_NO_DEVICE
