"""A model over MXFP4 weights: decode steps against the oracle model that holds the rounded weights' values, prompt chunks
against the operators called one after the other (each of which test_gpu_mxfp.py holds to 64 bits), and the loops and loaders around
them."""
import importlib

import numpy as np
import pytest

import ggufwriter as W
import mx_oracle as mx
from oraclelib import check_logits
from test_gpu_gguf import SMALL, WIDE_HEAD, _near_tie, oracle_from_weights, synth_weights

F16 = 1
LINEAR = ("attn_q", "attn_k", "attn_v", "attn_output", "ffn_gate", "ffn_up", "ffn_down")


def is_linear(name):
    return name == "output.weight" or (name.endswith(".weight") and name.split(".")[-2] in LINEAR)


def rounded(w):
    """The tensors with every linear weight at its MXFP4 value (two significant bits: f16 and bf16 hold it)."""
    out = {}
    for name, a in w.items():
        out[name] = a
        if is_linear(name):
            v = mx.values(*mx.quantize(a.astype(np.float32), True), True)
            out[name] = v.astype(np.float16)
            assert np.array_equal(out[name].astype(np.float64), v), name
    return out


def opened(tmp_path, d, w, **more):
    path = str(tmp_path / "model.gguf")
    W.qwen2_file(path, d, w, **more)
    return path


def qwen():
    return importlib.import_module("cpp-tensorlib_amd.qwen")


def tokens_of(d, n, seed):
    return np.random.default_rng(seed).integers(0, d["vocab"], n)


class Blobs:
    """The tensors as stored [K, N] bf16 blobs."""

    def __init__(self, orc, d, w):
        self.d = type("D", (), dict(d))()
        self.orc, self.w = orc, w

    def weight(self, li, name):
        names = dict(wq="attn_q.weight", wk="attn_k.weight", wv="attn_v.weight", wo="attn_output.weight", wg="ffn_gate.weight",
                     wu="ffn_up.weight", wd="ffn_down.weight", bq="attn_q.bias", bk="attn_k.bias", bv="attn_v.bias",
                     an="attn_norm.weight", fn="ffn_norm.weight")
        top = dict(embed="token_embd.weight", onorm="output_norm.weight", outw="output.weight")
        a = self.w[top[name] if li < 0 else "blk.%d.%s" % (li, names[name])]
        if a.dtype == np.float32:
            return a
        wide = a.astype(np.float32) if name == "embed" else np.ascontiguousarray(a.astype(np.float32).T)
        return self.orc.to_bf16(wide)


@pytest.mark.gpu
@pytest.mark.parametrize("dims,source", [(SMALL, "file"), (SMALL, "tied"), (WIDE_HEAD, "file"), (WIDE_HEAD, "blobs")])
@pytest.mark.parametrize("form", ["fused", "epilogue off", "one launch an op"])
def test_steps_are_those_of_the_rounded_weights(orc, tmp_path, dims, source, form):
    """Weights rounded on the device as they load; the steps' bar is that of the other formats' (1e-5 of 1 + |logit|)."""
    print("case", dims["hidden"], source, form, flush=True)
    tied = source == "tied"
    w = synth_weights(dims, seed=7, tied=tied)
    if source == "blobs":
        # (cut to bf16's bits, which f16 holds)
        w = {k: (v if v.dtype == np.float32 else (v.astype(np.float32).view(np.uint32) & 0xffff0000).view(np.float32).astype(np.float16))
             for k, v in w.items()}
        g = qwen().QwenGPU.from_blobs(Blobs(orc, dims, w), fmt="mxfp4")
    else:
        g = qwen().QwenGPU.from_gguf(opened(tmp_path, dims, w, tied=tied), fmt="mxfp4", max_ctx=dims["max_ctx"])
    if form == "epilogue off":
        g.set_gateup_epilogue(False)
    if form == "one launch an op":
        g.set_fused(False)
    om = oracle_from_weights(orc, dims, rounded(w), q4=False)
    tok = 3
    for pos in range(12):
        want_tok, want = om.step(tok, pos)
        got_tok, got = g.step(tok, pos, want_logits=True)
        check_logits(got, want, 1e-5, "pos %d" % pos, 1.0)
        if got_tok != want_tok:
            assert _near_tie(want)
        tok = want_tok
    c = g.census()
    assert c["quantize_mx"] > 0 and c["gemv_mxfp4"] > 0
    g.close()
    om.close()


def operators_prompt(lib, d, w, chunks):
    """Final-norm rows of the last chunk, from the library's calls."""
    E, H, Hk, D, FF, L, ctx = d["hidden"], d["n_q_heads"], d["n_kv_heads"], d["head_dim"], d["ff"], d["n_layers"], d["max_ctx"]
    QD, QKV = H * D, (H + 2 * Hk) * D
    keep = []

    def dev(a):
        keep.append(lib.to_device(np.ascontiguousarray(a)))
        return keep[-1]

    def four(*names):
        a = np.concatenate([w[n] for n in names]).astype(np.float16)
        src, codes, scales = dev(a.view(np.uint16)), dev(np.zeros(a.size // 2, np.uint8)), dev(np.zeros(a.size // 32, np.uint8))
        lib.quantize_mxfp4(src, F16, codes, scales, *a.shape)
        return codes, scales

    rows = max(len(c) for c in chunks)
    b = {k: dev(np.zeros(rows * n, np.float32)) for k, n in dict(x=E, qh=QD, at=QD, out=E).items()}
    b["table"] = dev(np.zeros(rows * D, np.float32))
    h8, a8, m8 = [(dev(np.zeros(rows * n, np.uint8)), dev(np.zeros(rows * n // 32, np.uint8))) for n in (E, QD, FF)]
    parts = dev(np.zeros(16 * rows * max(E, QKV), np.float32))
    table = dev(w["token_embd.weight"].view(np.uint16))
    caches = [(dev(np.zeros(Hk * ctx * D, np.float32)), dev(np.zeros(Hk * ctx * D, np.float32))) for _ in range(L)]
    W4 = []
    for l in range(L):
        p = "blk.%d." % l
        W4.append(dict(qkv=four(p + "attn_q.weight", p + "attn_k.weight", p + "attn_v.weight"), o=four(p + "attn_output.weight"),
                       gu=four(p + "ffn_gate.weight", p + "ffn_up.weight"), d=four(p + "ffn_down.weight"),
                       an=dev(w[p + "attn_norm.weight"]), fn=dev(w[p + "ffn_norm.weight"]),
                       bias=[dev(w[p + "attn_%s.bias" % c]) for c in "qkv"]))
    onorm = dev(w["output_norm.weight"])
    pos = 0

    for c in chunks:
        T = len(c)
        lib.embed_rows(table, F16, c, b["x"], E, d["vocab"])
        lib.rope_table_range(b["table"], D, pos, T, d["rope_base"])
        lib.rmsnorm_res_mxfp8(b["x"], None, 0, W4[0]["an"], None, *h8, E, d["eps"], T)
        for l, m in enumerate(W4):
            n = lib.gemm_mxfp4_nt_parts(*h8, *m["qkv"], parts, T, QKV, E)
            lib.qkv_rope_fill(parts, *m["bias"], b["table"], b["qh"], *caches[l], T, H, Hk, D, pos, ctx, n_parts=n)
            lib.attn_prefill_tok(b["qh"], *caches[l], b["at"], H, Hk, T, ctx, D, 1.0 / np.sqrt(np.float32(D)), pos0=pos)
            lib.quantize_mxfp8(b["at"], *a8, T, QD)
            n = lib.gemm_mxfp4_nt_parts(*a8, *m["o"], parts, T, E, QD)
            lib.rmsnorm_res_mxfp8(b["x"], parts, n, m["fn"], b["x"], *h8, E, d["eps"], T)
            lib.gemm_mxfp4_nt_swiglu(*h8, *m["gu"], *m8, T, FF, E)
            n = lib.gemm_mxfp4_nt_parts(*m8, *m["d"], parts, T, E, FF)
            if l + 1 < L:
                lib.rmsnorm_res_mxfp8(b["x"], parts, n, W4[l + 1]["an"], b["x"], *h8, E, d["eps"], T)
            else:
                lib.rmsnorm_res_parts(b["x"], parts, n, onorm, b["x"], b["out"], E, d["eps"], T)
        pos += T
    out = b["out"].numpy()[:T * E].reshape(T, E).copy()
    for k in keep:
        k.free()
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dims,lengths", [(SMALL, (1,)), (SMALL, (5,)), (SMALL, (16, 16, 3)), (SMALL, (70,)), (WIDE_HEAD, (33, 33, 7)), (WIDE_HEAD, (64, 9))])
def test_prompt_is_the_operators_in_order(lib, tmp_path, dims, lengths):
    print("case", dims["hidden"], lengths, flush=True)
    w = synth_weights(dims, seed=11)
    g = qwen().QwenGPU.from_gguf(opened(tmp_path, dims, w), fmt="mxfp4", max_ctx=dims["max_ctx"])
    ids, chunks, at = tokens_of(dims, sum(lengths), 13), [], 0
    for n in lengths:
        chunks.append(ids[at:at + n])
        at += n
    logits = g.prefill(ids, chunk=lengths[0])
    got = g.prefill_hidden(lengths[-1])
    want = operators_prompt(lib, dims, w, chunks)
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))
    # the last row's logits: the f32 row over the rounded head
    head = mx.values(*mx.quantize(w["output.weight"].astype(np.float32), True), True)
    row, E = want[-1].astype(np.float64), dims["hidden"]
    bound = (128 + E / 128 + 64) * 2.0 ** -24 * (np.abs(head) @ np.abs(row)) + 1e-30
    assert np.all(np.abs(logits - head @ row) <= bound)
    assert g.census()["gemm_mxfp4"] > 0
    g.close()


@pytest.mark.gpu
def test_loops_over_a_prompt_agree(tmp_path):
    """Eager steps, the recorded decoder and the token loop on the device behind the same prompt."""
    w = synth_weights(SMALL, seed=17)
    path, ids, got = opened(tmp_path, SMALL, w), tokens_of(SMALL, 21, 19), {}
    for how in ("eager", "recorded", "device"):
        g = qwen().QwenGPU.from_gguf(path, fmt="mxfp4", max_ctx=SMALL["max_ctx"])
        first = int(np.argmax(g.prefill(ids, chunk=16)))
        if how == "device":
            g.greedy_init(first, 21)
            g.greedy_run(20)
            got[how] = list(g.greedy_tokens(21, 20))
        else:
            if how == "recorded":
                g.decoder_init(first, 21)
            tok, out = first, []
            for pos in range(21, 41):
                tok = g.decoder_step(tok) if how == "recorded" else g.step(tok, pos)
                tok = tok[0] if isinstance(tok, tuple) else tok
                out.append(tok)
            got[how] = out
        g.close()
    assert got["eager"] == got["recorded"] == got["device"]


@pytest.mark.gpu
def test_rows_of_logits_do_not_depend_on_how_many_are_asked_for(tmp_path):
    model = importlib.import_module("cpp-tensorlib_amd.model")
    w = synth_weights(WIDE_HEAD, seed=23)
    path, ids = opened(tmp_path, WIDE_HEAD, w), tokens_of(WIDE_HEAD, 30, 29)
    m = model.Model.open(path, max_ctx=WIDE_HEAD["max_ctx"], mxfp4=True)
    many = m.feed(ids, want=[0, 7, 29])
    for i, t in enumerate((0, 7, 29)):
        m.reset()
        assert np.array_equal(m.feed(ids, want=[t])[0], many[i])
    m.close()


@pytest.mark.gpu
def test_seeded_weights_run():
    """Weights tiled from seeded blocks (of throughput runs) give finite logits in a step and in a prompt."""
    g = qwen().QwenGPU(SMALL)
    g.set_random(3, fmt="mxfp4")
    assert np.all(np.isfinite(g.step(5, 0, want_logits=True)[1]))
    g.set_cache_pos(0)
    assert np.all(np.isfinite(g.prefill(tokens_of(SMALL, 40, 1))))
    g.close()


@pytest.mark.parametrize("also", [dict(q4=True), dict(exact=True)])
def test_formats_exclude_each_other(tmp_path, also):
    model = importlib.import_module("cpp-tensorlib_amd.model")
    with pytest.raises(RuntimeError, match="exclude"):
        model.Model.open(str(tmp_path / "none.gguf"), mxfp4=True, **also)


def test_folders_have_no_mxfp4_form(tmp_path):
    model = importlib.import_module("cpp-tensorlib_amd.model")
    with pytest.raises(RuntimeError, match="GGUF"):
        model.Model.open(str(tmp_path), mxfp4=True)
