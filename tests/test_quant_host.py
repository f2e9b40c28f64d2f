"""The operators of the 8-bit and 4-bit formats without a GPU: what they refuse, and the packing of 4-bit weights."""
import pytest
import torch

from llm_steadyinfer_b200.csrc import ops

E4M3, BF16 = torch.float8_e4m3fn, torch.bfloat16


def test_cpu_tensors_are_refused():
    with pytest.raises(ops.KernelError, match="CUDA tensors only"):
        ops.quantize_q8(torch.zeros(2, 8), torch.zeros(2, 8).to(E4M3), torch.zeros(2))


@pytest.fixture
def checks_alone(monkeypatch):
    """The checks of arguments on CPU tensors: the device is not asked about, and a call that passes them would reach ``launched``."""
    launched = []

    def fn(lib, symbol, argtypes):
        def call(*args):
            assert len(args) == len(argtypes)
            launched.append(symbol)
            return 0
        return call

    monkeypatch.setattr(ops, "_here", lambda *a: 0)
    monkeypatch.setattr(ops, "_fn", fn)
    monkeypatch.setattr(ops, "gemm_tc05_available", lambda: True)
    return launched


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def norm_args(**kw):
    a = dict(resid=z(3, 16), delta=z(3, 16, dtype=BF16), weight=z(16), eps=1e-5, out=z(3, 16, dtype=E4M3), scale=z(3))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(resid=z(3, 16, dtype=BF16)), "fp32"),
    (dict(resid=z(16, 3).t()), "contiguous"),
    (dict(weight=z(15)), "weight"),
    (dict(delta=z(3, 15, dtype=BF16)), "delta"),
    (dict(delta=z(3, 16, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(delta2=z(3, 16)), "one dtype"),
    (dict(delta=None, delta2=z(3, 16)), "delta"),
    (dict(out=z(3, 16, dtype=BF16)), "float8"),
    (dict(out=z(2, 16, dtype=E4M3)), "float8"),
    (dict(scale=z(4)), "scale"),
    (dict(scale=z(6)[::2]), "scale"),
    (dict(dst=z(3, 17)), "dst"),
    (dict(rows=z(3, dtype=torch.int32), dst=z(3, 16)), "no stream"),
    (dict(rows=z(3, dtype=torch.int64)), "int32"),
])
def test_norm_refusals(checks_alone, kw, text):
    with pytest.raises(ops.KernelError, match=text):
        ops.add_rmsnorm_q8(**norm_args(**kw))
    assert not checks_alone


def test_norm_passes(checks_alone):
    ops.add_rmsnorm_q8(**norm_args())
    ops.add_rmsnorm_q8(**norm_args(rows=z(3, dtype=torch.int32)))
    assert checks_alone == ["si_add_rmsnorm_q8"] * 2


@pytest.mark.parametrize("gu,out,scale,group", [
    (z(2, 31), z(2, 16, dtype=E4M3), z(2), None), (z(2, 32), z(2, 16), z(2), None), (z(2, 32), z(2, 16, dtype=E4M3), z(2), 5),
    (z(2, 32), z(2, 16, dtype=E4M3), z(2), -8), (z(2, 32), z(2, 16, dtype=E4M3), z(1), None), (z(32, 2).t(), z(2, 16, dtype=E4M3), z(2), None),
    (z(2, 32, dtype=torch.float16), z(2, 16, dtype=E4M3), z(2), None), (z(2, 0), z(2, 0, dtype=E4M3), z(2), None)])
def test_swiglu_refusals(checks_alone, gu, out, scale, group):
    with pytest.raises(ops.KernelError):
        ops.swiglu_q8(gu, out, scale, group)
    assert not checks_alone


@pytest.mark.parametrize("x,out,scale", [
    (z(2, 8, dtype=torch.float16), z(2, 8, dtype=E4M3), z(2)), (z(8, 2).t(), z(2, 8, dtype=E4M3), z(2)), (z(2, 8), z(2, 9, dtype=E4M3), z(2)),
    (z(2, 8), z(2, 8, dtype=E4M3), z(3)), (z(2, 4, 8), z(2, 8, dtype=E4M3), z(2)), (z(2, 0), z(2, 0, dtype=E4M3), z(2))])
def test_quantize_refusals(checks_alone, x, out, scale):
    with pytest.raises(ops.KernelError):
        ops.quantize_q8(x, out, scale)
    assert not checks_alone


def q8_args(**kw):
    a = dict(a=z(3, 32, dtype=E4M3), a_scale=z(3), w=z(5, 32, dtype=E4M3), w_scale=z(5), out=z(3, 5, dtype=BF16))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(a=z(3, 32, dtype=BF16)), dict(w=z(5, 32, dtype=torch.float8_e5m2)), dict(w=z(5, 31, dtype=E4M3)), dict(out=z(3, 6, dtype=BF16)),
    dict(out=z(3, 5, dtype=torch.float16)), dict(out=z(5, 3, dtype=BF16).t()), dict(out=z(1, 5, dtype=BF16).expand(3, 5)), dict(a_scale=z(2)),
    dict(w_scale=z(5, dtype=BF16)), dict(a=z(32, 3, dtype=E4M3).t()), dict(status=z(1)), dict(a=z(3, 0, dtype=E4M3), w=z(5, 0, dtype=E4M3)),
    dict(a=z(32, dtype=E4M3))])
def test_gemm_q8_refusals(checks_alone, kw):
    with pytest.raises(ops.KernelError):
        ops.gemm_q8(**q8_args(**kw))
    assert not checks_alone


def w4_args(**kw):
    a = dict(x=z(3, 64, dtype=BF16), w=z(5, 8, dtype=torch.int32), scales=z(5, 2, dtype=BF16), zeros=z(5, 2, dtype=torch.uint8), group=32, out=z(3, 5, dtype=BF16))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(x=z(3, 64)), dict(w=z(5, 8)), dict(w=z(5, 7, dtype=torch.int32)), dict(group=48), dict(group=0), dict(group=-128), dict(group=96), dict(group=192),
    dict(group=64), dict(scales=z(5, 2)), dict(scales=z(2, 5, dtype=BF16).t()), dict(zeros=z(5, 2, dtype=torch.int8)), dict(zeros=z(5, 1, dtype=torch.uint8)),
    dict(out=z(3, 5, dtype=torch.float16)), dict(out=z(2, 5, dtype=BF16)), dict(out=z(1, 5, dtype=BF16).expand(3, 5)),
    dict(x=z(3, 60, dtype=BF16)), dict(x=z(64, 3, dtype=BF16).t()), dict(status=z(1))])
def test_gemm_w4_refusals(checks_alone, kw):
    with pytest.raises(ops.KernelError):
        ops.gemm_w4(**w4_args(**kw))
    assert not checks_alone


def test_products_pass_and_empty_ones_launch_nothing(checks_alone):
    ops.gemm_q8(**q8_args())
    ops.gemm_w4(**w4_args())
    n = len(checks_alone)
    assert n == 2
    ops.gemm_q8(**q8_args(a=z(0, 32, dtype=E4M3), a_scale=z(0), out=z(0, 5, dtype=BF16)))
    ops.gemm_w4(**w4_args(x=z(0, 64, dtype=BF16), out=z(0, 5, dtype=BF16)))
    ops.quantize_q8(z(0, 8), z(0, 8, dtype=E4M3), z(0))
    assert len(checks_alone) == n


def test_sizes_beyond_32_bits_are_refused(checks_alone):
    meta = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="meta")
    many = 2 ** 31
    for call in (lambda: ops.quantize_q8(meta(many, 8), meta(many, 8, dtype=E4M3), meta(many)),
                 lambda: ops.swiglu_q8(meta(many, 16), meta(many, 8, dtype=E4M3), meta(many)),
                 lambda: ops.add_rmsnorm_q8(meta(many, 8), None, meta(8), 1e-5, meta(many, 8, dtype=E4M3), meta(many)),
                 lambda: ops.gemm_q8(meta(many, 16, dtype=E4M3), meta(many), meta(8, 16, dtype=E4M3), meta(8), meta(many, 8)),
                 lambda: ops.gemm_w4(meta(1, 32, dtype=BF16), meta(many, 4, dtype=torch.int32), meta(many, 1, dtype=BF16), None, 128, meta(1, many))):
        with pytest.raises(ops.KernelError, match="32 bits"):
            call()
    assert checks_alone == []


@pytest.mark.parametrize("group", [384, 2 ** 32 + 128, 2 ** 40])
def test_a_group_beyond_the_row_is_one_group(monkeypatch, group):
    seen = []
    monkeypatch.setattr(ops, "_here", lambda *a: 0)
    monkeypatch.setattr(ops, "gemm_tc05_available", lambda: True)
    monkeypatch.setattr(ops, "_fn", lambda lib, symbol, argtypes: lambda packed: seen.append(ops._GEMM_W4_ARGS.unpack(packed)[6]) or 0)
    ops.gemm_w4(z(2, 160, dtype=BF16), z(3, 20, dtype=torch.int32), z(3, 1, dtype=BF16), None, group, z(2, 3))
    assert seen == [256]


def test_a_tensor_of_another_device_is_refused(monkeypatch):
    class Elsewhere:
        is_cuda = True

        def __init__(self, index):
            self.index = index

        def get_device(self):
            return self.index

    monkeypatch.setattr(ops, "_device_index", 1)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 1000 + index)
    assert ops._here("x", Elsewhere(1), None) == 1001              # the stream of the device that kernels are launched on
    for ts in ((Elsewhere(1), Elsewhere(0)), (Elsewhere(0), Elsewhere(0)), (Elsewhere(0), None)):
        with pytest.raises(ops.KernelError, match="device"):
            ops._here("x", *ts)


@pytest.mark.parametrize("N,K", [(1, 8), (5, 64), (3, 136)])
def test_pack_and_unpack(N, K):
    q = torch.randint(0, 16, (N, K), generator=torch.Generator().manual_seed(K))
    words = ops.pack_w4(q)
    assert words.shape == (N, K // 8) and words.dtype == torch.int32
    assert torch.equal(ops.unpack_w4(words), q.to(torch.int32))
    u = words.long() & 0xFFFFFFFF
    for i in range(8):                                           # entry i of the eight at bit 4 (i / 2) + 16 (i % 2)
        assert torch.equal((u >> (4 * (i // 2) + 16 * (i % 2))) & 15, q[:, i::8])
    with pytest.raises(ops.KernelError):
        ops.pack_w4(q[:, :7])


def test_weight_formats_of_models():
    """The layers' specs in a format, and what has none."""
    from llm_steadyinfer_b200.config import config_from_dict
    from llm_steadyinfer_b200.models import Model
    from nufasun_configs import CONFIGS as OTHERS
    from tiny_configs import TINY_A
    for fmt, arrangement, files in (("q8", "pre_norm_q8", {"quant_rows", "gemm_q8", "gemm_quant"}), ("w4", "pre_norm", {"gemm_w4", "gemm_quant", "swiglu"})):
        m = Model(config_from_dict(TINY_A), torch.bfloat16, "cpu", fmt)
        assert m.weight_format == fmt and m.capturable()
        assert {b.arrangement for b in m.blocks} == {arrangement}
        assert {ls.mixer.kind for ls in m.spec.layers} == {"quantized_attention"}
        assert files <= set(m.kernel_files(16))
        assert m.weight_shapes() == Model(config_from_dict(TINY_A), torch.bfloat16, "cpu").weight_shapes()
        with pytest.raises(ValueError, match="bfloat16"):
            Model(config_from_dict(TINY_A), torch.float32, "cpu", fmt)
    with pytest.raises(ValueError, match="weight_format"):
        Model(config_from_dict(TINY_A), torch.bfloat16, "cpu", "q4")
    other = next(iter(OTHERS.values()))
    with pytest.raises(ValueError, match="has no form for it|goes with the arrangement"):
        Model(config_from_dict(other[0] if isinstance(other, tuple) else other), torch.bfloat16, "cpu", "w4")


def test_quantize_w4_on_the_cpu():
    from llm_steadyinfer_b200.parts.quantized import quantize, quantize_w4
    g = torch.Generator().manual_seed(1)
    w = torch.randn(7, 200, generator=g).to(BF16) * 0.05
    for group in (32, 64, 128, 256):
        q = quantize_w4(w, group)
        G = -(-200 // group)
        assert q.scales.shape == q.zeros.shape == (7, G) and q.words.shape == (7, 25)
        step = q.scales.double().repeat_interleave(group, 1)[:, :200]
        assert ((q.dense().double() - w.double()).abs() <= step * (1 + 15 * 2.0 ** -8)).all()
    with pytest.raises(ValueError, match="multiple of 8"):
        quantize(w[:, :100].contiguous()[:, :99], "w4")


def test_aligned_cluster_barriers_are_met_by_whole_warps():
    """``barrier.cluster`` in its aligned form is undefined unless all lanes of a warp make it together; behind a loop or a branch that lanes leave at
    different times nothing but a warp barrier sees to that. So the one helper that issues it brings the warp together first, and no kernel issues it itself."""
    import glob
    import os
    folder = os.path.dirname(ops.__file__)
    found = {}
    for path in sorted(glob.glob(os.path.join(folder, "*.cu*"))):
        with open(path) as f:
            text = f.read()
        if "barrier.cluster" in text:
            found[os.path.basename(path)] = text
    assert list(found) == ["tma_common.cuh"]
    body = found["tma_common.cuh"].split("void cluster_sync_all() {")[1].split("}")[0]
    assert found["tma_common.cuh"].count("barrier.cluster.arrive") == 1 and found["tma_common.cuh"].count("barrier.cluster.wait") == 1
    assert body.index("__syncwarp();") < body.index("barrier.cluster.arrive") < body.index("barrier.cluster.wait")


@pytest.mark.parametrize("family", ["fevosun", "mivorax", "nufasun", "risizen", "samulorn", "vibunex"])
@pytest.mark.parametrize("fmt", ["q8", "w4"])
def test_models_without_a_form_for_the_formats_are_refused_by_name(family, fmt):
    """Every configuration of the other architectures, layers with one norm for both sublayers among them."""
    import importlib
    from llm_steadyinfer_b200.config import config_from_dict
    from llm_steadyinfer_b200.models import Model
    for config in importlib.import_module(family + "_configs").CONFIGS.values():
        with pytest.raises(ValueError, match="has no form for it|goes with the arrangement"):
            Model(config_from_dict(config[0] if isinstance(config, tuple) else config), torch.bfloat16, "cpu", fmt)


def test_rows_whose_last_step_ends_beyond_32_bits_are_refused():
    """4-bit weights on no 16-byte boundary: 2^30 - 8 entries of x are 2^31 - 16 bytes, and the last of a step's four loads of 16 bytes would begin there: its
    end passes 2^31 - 1 and compares as below the row's length. The entry returns before it launches anything (null pointers are not touched)."""
    import ctypes
    from llm_steadyinfer_b200.csrc import build
    fn = build.load("gemm_quant").si_gemm_quant_w4
    fn.argtypes, fn.restype = ops._GEMM_QUANT_W4_ARGS, ctypes.c_int
    for K in (2 ** 30 - 8, 2 ** 30 - 16, 2 ** 30 - 24):
        assert 2 * (32 * (-(-K // 32)) - 8) + 16 > 2 ** 31 - 1
        assert fn(None, K, None, K // 8, None, None, 128, None, 1, 0, 1, 1, K, None) == -2
    assert 2 * (2 ** 30 - 32 - 8) + 16 <= 2 ** 31 - 1          # the longest row that is taken
