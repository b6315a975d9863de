"""CPU: host-side logic of the boundary -- config surface, yaml, parameter table vs the reference's state-dict keys."""
import os

import numpy as np
import pytest
import yaml

from fithubert_amd.config import CustomStudentModelConfig, _eval_layer_spec, conv_out_length
from fithubert_amd.engine import param_table, unsupported
from oracle import student_ref as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CONF = os.path.join(ROOT, "conf")


def _fit():
    with open(os.path.join(CONF, "fithubert.yaml")) as f:
        return yaml.load(f, Loader=yaml.FullLoader)


def test_yaml_surface_parses_unchanged():
    y = _fit()
    assert set(y) == {"teacher", "train", "distiller", "optimizer", "data", "specaug"}
    cfg = CustomStudentModelConfig(**y["distiller"])
    assert cfg.encoder_layers == 12 and cfg.encoder_embed_dim == 480 and cfg.tr_layer_index == 0
    assert y["optimizer"]["lr"] == 5e-4
    # the reference yaml writes floats as '5.e-4'; FullLoader (train.py:462) parses that form as a float
    assert yaml.load("lr: 5.e-4", Loader=yaml.FullLoader)["lr"] == 5e-4
    with pytest.raises(TypeError):
        CustomStudentModelConfig(not_a_field=1)


def test_config_field_names_and_defaults_match_reference_dataclass():
    # the 44 fields of modules/model.py:24-251
    names = [f for f in CustomStudentModelConfig.__dataclass_fields__]
    assert len(names) == 44
    ref_defaults = S.DEFAULTS
    c = CustomStudentModelConfig()
    for k, v in ref_defaults.items():
        assert getattr(c, k) == v, k


def test_layer_spec_evaluator_matches_python_eval():
    for spec in ["[(128, 10, 5)] + [(256, 1, 1)] + [(256, 3, 2)] * 4 + [(512, 1, 1)] + [(512, 2, 2)] * 2",
                 "[(512, 10, 5)] + [(512, 3, 2)] * 4 + [(512,2,2)] * 2"]:
        assert _eval_layer_spec(spec) == [tuple(t) for t in eval(spec)]
    with pytest.raises(Exception):
        _eval_layer_spec("__import__('os').system('true')")


def test_frame_formula():
    layers = CustomStudentModelConfig(**_fit()["distiller"]).conv_layers()
    assert conv_out_length(160000, layers) == 499
    assert conv_out_length(32000, layers) == 99
    assert conv_out_length(25000, layers) == 77  # golden: valid frames of the padded pair


def test_native_param_table_equals_reference_state_dict():
    y = _fit()
    cfg = CustomStudentModelConfig(**y["distiller"])
    table, total = param_table(cfg, "bf16")
    ours = {n: s for n, _, s in table}
    ref = S.param_shapes(y["distiller"])
    assert set(ours) == set(ref)
    for k in ref:
        assert tuple(ours[k]) == tuple(ref[k]), k
    assert sum(int(np.prod(s)) for s in ours.values()) == 31629632
    # offsets are 8-float aligned and non-overlapping
    spans = sorted((o, o + int(np.prod(s))) for _, o, s in table)
    for (a0, a1), (b0, b1) in zip(spans, spans[1:]):
        assert a1 <= b0 and b0 % 8 == 0
    assert spans[-1][1] <= total


def test_unsupported_configs_fail_loudly():
    y = _fit()
    d = dict(y["distiller"])
    d["layer_type"] = "conformer"
    assert unsupported(CustomStudentModelConfig(**d))
    with pytest.raises(NotImplementedError):
        param_table(CustomStudentModelConfig(**d))


def test_ex_yaml_param_table_equals_reference_state_dict():
    """ex.yaml (DistilHuBERT-style head: proj_head.0 Linear, proj_head.2 SplitLinear [task][Din][Dout], no TR layer)."""
    import os
    y = yaml.safe_load(open(os.path.join(os.path.dirname(__file__), "..", "conf", "ex.yaml")))
    cfg = CustomStudentModelConfig(**y["distiller"])
    assert unsupported(cfg) is None
    table, total = param_table(cfg, "bf16")
    ours = {n: s for n, _, s in table}
    ref = S.param_shapes(y["distiller"])
    assert set(ours) == set(ref), (set(ours) ^ set(ref))
    for k in ref:
        assert tuple(ours[k]) == tuple(ref[k]), k
    assert ours["proj_head.2.weight"] == (3, 768, 768) and ours["proj_head.2.bias"] == (1, 1, 3, 768)
    d = dict(y["distiller"], pred_layer_id="[11]")      # single task: SplitLinear degenerates to nn.Linear (module.py:604-605)
    cfg1 = CustomStudentModelConfig(**d)
    assert unsupported(cfg1) is None
    ours1 = {n: s for n, _, s in param_table(cfg1, "bf16")[0]}
    assert ours1 == {k: tuple(v) for k, v in S.param_shapes(d).items()}


def test_gemm_table_roundtrip(tmp_path):
    """Per-shape main-loop table: import / export / file round trip (host-side map, no GPU needed)."""
    from fithubert_amd import _lib as L
    import ctypes as C
    lib = L.lib()
    lib.fh_gemm_tune(-1)
    keys = (C.c_ulonglong * 2)(0x1234567890ABCDEF, 42)
    paths = (C.c_int * 2)(7, 3)
    sks = (C.c_int * 2)(1, 43)
    assert lib.fh_gemm_tune_import(keys, paths, sks, 2) == 2
    f = str(tmp_path / "table.json")
    assert L.save_gemm_table(f) == 2
    lib.fh_gemm_tune(-1)
    assert lib.fh_gemm_tune(0) == 0
    assert L.load_gemm_table(f) == 2
    k2, p2, s2 = (C.c_ulonglong * 2)(), (C.c_int * 2)(), (C.c_int * 2)()
    assert lib.fh_gemm_tune_export(k2, p2, s2, 2) == 2
    assert sorted(zip(k2, p2, s2)) == sorted(zip(keys, paths, sks))
    lib.fh_gemm_tune(-1)
    assert L.load_gemm_table(str(tmp_path / "missing.json")) == 0


def test_units_are_compiled_without_packed_fp32_arithmetic():
    """v_pk_add / mul / fma_f32 give wrong results now and then (conv 0's fp32 forward beside another stream's work): all units but the 16-bit GEMM loops are built without them."""
    import glob
    from fithubert_amd import build
    units = {os.path.basename(f) for f in glob.glob(os.path.join(build.CSRC, "*.hip"))}
    packed = {u for u in units if "-packed-fp32-ops" not in build.file_flags(u)}
    assert packed == {"gemm_bf16.hip", "gemm_f16.hip"} and "conv0.hip" in units
