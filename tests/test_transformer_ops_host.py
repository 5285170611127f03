"""CPU: what the encoder-layer operators refuse before anything is launched, the bucket edges, and the encoder's options."""
import ctypes as C

import pytest
import torch

from tests._transformer_ref import bucket64


def test_no_cpu_path():
    from asr_amd.Models.transformer_ops import bucket_attention, gated_feed_forward, qk_norm_rope
    x = torch.zeros(1, 2, 2, 8)
    with pytest.raises(RuntimeError):
        qk_norm_rope(x, x, torch.ones(8), torch.ones(8))
    with pytest.raises(RuntimeError):
        bucket_attention(x, x, x, torch.zeros(32, 2))
    with pytest.raises(RuntimeError):
        gated_feed_forward(torch.zeros(2, 8), torch.zeros(4, 8), torch.zeros(4, 8), torch.zeros(8, 4))


def test_bucket_edges_are_the_definitions():
    from asr_amd.Models.transformer_ops import bucket_edges
    for nb, reach, causal in ((32, 128, False), (32, 128, True), (16, 64, False), (64, 448, True), (4, 2, False), (2, 3, True),
                              (256, 1024, True), (250, 800, False), (7, 1024, True)):
        n = nb if causal else nb // 2
        e = bucket_edges(nb, reach, causal)
        assert len(e) == n - n // 2 - 1 and list(e) == sorted(e) and all(x <= reach for x in e)
        r = torch.arange(-reach - 5, reach + 6)
        slot = bucket64(r, nb, reach, causal)
        for x, k in zip(r.tolist(), slot.tolist()):
            away = max(-x, 0) if causal else abs(x)
            want = away if away < n // 2 else n // 2 + sum(away >= y for y in e)
            assert k == want + (n if x > 0 and not causal else 0)


def _refused(fn, args, **change):
    from asr_amd import _lib
    lib = _lib.load()
    for k, v in change.items():
        setattr(args, k, v)
    assert getattr(lib, fn)(C.byref(args), None) == -1, change
    assert lib.asr_last_error()


def test_c_abi_refusals():
    """No case gets as far as a launch: the pointers are not memory."""
    from asr_amd import _lib

    def rope():
        a = _lib.RopeArgs()
        for n in ("q", "k", "gq", "gk", "wq", "wk", "q_out", "k_out", "dwq", "dwk", "ws"):
            setattr(a, n, 64)
        a.B = a.T = a.H = a.Hk = 1
        a.D, a.rot, a.base, a.eps = 8, 8, 1e4, 1e-6
        return a
    for change in (dict(q=None), dict(dtype=3), dict(D=7), dict(D=130), dict(rot=3), dict(rot=10), dict(rot=-2), dict(base=0.0), dict(eps=-1.0), dict(B=0)):
        _refused("asr_qk_norm_rope_fwd", rope(), **change)
    for change in (dict(gq=None), dict(ws=None), dict(dwq=None)):
        _refused("asr_qk_norm_rope_bwd", rope(), **change)

    def attn():
        a = _lib.BucketAttentionArgs()
        for n in ("q", "k", "v", "g", "table", "out", "out32", "lse", "dq", "dk", "dv", "dtable", "ws"):
            setattr(a, n, 64)
        a.B = a.Tq = a.Tk = a.H = a.Hk = 1
        a.D, a.nb, a.scale = 8, 32, 1.0
        attn.edges = (C.c_int32 * 7)(12, 16, 23, 32, 46, 64, 91)
        a.edges_host = C.addressof(attn.edges)
        return a
    for change in (dict(q=None), dict(out=None), dict(dtype=-1), dict(D=129), dict(D=0), dict(H=3, Hk=2), dict(nb=3), dict(nb=258), dict(nb=31),
                   dict(edges_host=None), dict(Tq=0), dict(Tk=1 << 25), dict(train=1, lse=None), dict(B=1 << 20, H=4, Hk=4)):
        _refused("asr_bucket_attention_fwd", attn(), **change)
    for change in (dict(g=None), dict(dtable=None), dict(ws=None), dict(lse=None)):
        _refused("asr_bucket_attention_bwd", attn(), **change)
    a = attn()
    for bad in ((12, 16, 23, 32, 46, 64, 2000), (12, 11, 23, 32, 46, 64, 91), (3, 16, 23, 32, 46, 64, 91)):
        attn.edges[:] = bad
        _refused("asr_bucket_attention_fwd", a)

    def ff():
        a = _lib.GatedFFArgs()
        for n in ("x", "wg", "wu", "wd", "dy", "y", "dx", "dwg", "dwu", "dwd", "ws"):
            setattr(a, n, 64)
        a.M = a.d = a.f = a.n = 1
        return a
    for change in (dict(x=None), dict(y=None), dict(ws=None), dict(dtype=5), dict(act=2), dict(M=0), dict(d=0), dict(f=1 << 21), dict(M=1 << 31)):
        _refused("asr_gated_ff_fwd", ff(), **change)
    for change in (dict(dy=None), dict(dwg=None)):
        _refused("asr_gated_ff_bwd", ff(), **change)


def test_native_module_loads_by_itself():
    import subprocess
    import sys
    code = "from asr_amd import _lib; m = _lib.native(); assert m.rope and m.attention and m.ff"
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)


def test_encoder_options():
    from asr_amd.Models.AttModel import AttModel
    from asr_amd.Models.Transformer_encoder import TransformerEncoder
    from oracle import ref_model as R
    plain = TransformerEncoder(20, 64, 2, 4, 0.1)
    assert not any("norm.q" in k or "linear_gate" in k or "distance_bias" in k for k in plain.state_dict())
    keys = TransformerEncoder(20, 64, 2, 4, 0.1, attention="bucket", feed_forward="gated").state_dict()
    assert keys["encoder.layers.0.attn.distance_bias"].shape == (32, 4) and keys["encoder.layers.1.ff_2.linear_gate.weight"].shape == (2048, 64)
    assert not any("distance_bias" in k for k in TransformerEncoder(20, 64, 1, 4, 0.1, attention="rotary").state_dict())
    for bad in (dict(attention="absolute"), dict(feed_forward="relu"), dict(attention="rotary", heads=3), dict(attention="bucket", d_model=60)):
        kw = dict(src_vocab=20, d_model=64, N_e=1, heads=4, dropout=0.1) | bad
        with pytest.raises(ValueError):
            TransformerEncoder(**kw)
    hp = R.make_hp(lmfb_dim=20, frame_stacking=1, num_hidden_nodes_encoder=256, num_hidden_nodes_decoder=24, num_classes=31,
                   encoder_type="Conformer", encoder_attention="bucket")
    assert any("distance_bias" in k for k in AttModel(hp).state_dict())
    with pytest.raises(RuntimeError):
        TransformerEncoder(20, 64, 1, 4, 0.1, attention="rotary")(torch.zeros(1, 30, 20), torch.ones(1, 30, dtype=torch.long))
