"""The 8-bit key/value pairs, the attention that reads them and the channels-last group norm as the framework runs them:
in the attention module, the host network, the captured evaluation, the loader and the command line."""
import copy
import json
import os

import numpy as np
import pytest
import torch

from helpers import GOLDEN, load_masks, rel_err
from style_transfer_amd import feature_store as fs
from style_transfer_amd import ops, synth
from style_transfer_amd import unet as U
from style_transfer_amd.attention import CrossAttention
from style_transfer_amd.graphed import GraphedUNet
from style_transfer_amd.loader import FeatureLoader

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# 160 channels: head_dim 20 on the outermost level (which the 8-bit cache leaves as tensors), 40 and 80 below
CASE = json.load(open(os.path.join(GOLDEN, "unet_case.json")))
CFG = dict(CASE["cfg"], model_channels=160)

_model = {}


def build(channels_last):
    if channels_last not in _model:
        m = U.UNetModel(**CFG).eval()
        with torch.no_grad():
            for name, p in m.named_parameters():
                p.copy_(torch.from_numpy(synth.param_init(name, p.shape)))
        m = m.to(DEV)
        _model[channels_last] = m.use_channels_last() if channels_last else m
    for a in _model[channels_last].attention_modules():
        a.compute = None
    _model[channels_last].set_content_name("/nowhere/img.jpg")
    return _model[channels_last]


def feature_list(seed, steps=50):
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(steps):
        e = {"config": {"T": 1.5}, "z_enc": torch.randn(1, 4, 16, 16, generator=g)}
        for b in range(6, 12):
            n, d = (64, 40) if b < 9 else (256, 20)
            for t in "qkv":
                e["output_block_%d_self_attn_%s" % (b, t)] = torch.randn(8, n, d, generator=g)
        out.append(e)
    return out


def on_device(feats):
    return [{k: v.to(DEV) if torch.is_tensor(v) else v for k, v in e.items()} for e in feats]


def read_back(feats):
    """The list with every 8-bit pair as the float32 numbers that it stands for."""
    out = []
    for e in feats:
        e = dict(e)
        for k in [k for k in e if isinstance(e[k], ops.QuantKV) and k.endswith("_k")]:
            kv = e[k]
            e[k], e[k[:-1] + "v"] = (t[0] for t in ops.kv_cache_read(kv, 0, kv.S, torch.float32))
        out.append(e)
    return out


# 'fp32' is the split arithmetic (1e-3), 'f16' and 'bf16' round queries, probabilities and values once: 2^-11 and 2^-8
# relative each, below 2 % of the largest output with the projection behind them
@pytest.mark.parametrize("compute,tol", [("fp32", 1e-3), ("f16", 5e-3), ("bf16", 2e-2)])
@pytest.mark.parametrize("b,injected_q,dtype,fmt", [(1, True, torch.float32, "int8"), (3, True, torch.float32, "e4m3"),
                                                     (3, False, torch.float32, "int8"), (2, True, torch.bfloat16, "int8")])
def test_attention_module_on_a_quantised_pair(compute, tol, b, injected_q, dtype, fmt):
    if dtype == torch.bfloat16:
        tol = 2e-2                   # the projections' own roundings
    torch.manual_seed(5)
    heads, n, S, d, T, gamma = 8, 70, 133, 40, 1.5, 0.75
    attn = CrossAttention(heads * d, heads=heads, dim_head=d).to(DEV)
    attn.cnt_name, attn.compute = "/nowhere/img.jpg", compute
    x = torch.randn(b, n, heads * d, device=DEV)
    qi, k, v = (torch.randn(heads, m, d, device=DEV) for m in (n, S, S))
    kv = ops.kv_cache(1, heads, S, d, fmt, DEV)
    ops.kv_cache_write(kv, k[None], v[None])
    kd, vd = (t[0].double().cpu() for t in ops.kv_cache_read(kv, 0, S, torch.float32))
    ref = copy.deepcopy(attn).to(dtype).double().cpu()
    xd = x.to(dtype).double().cpu()
    with torch.no_grad():
        q = ref.to_q(xd).reshape(b, n, heads, d).transpose(1, 2)
        if injected_q:
            q = qi.to(dtype).double().cpu()[None] * gamma + q * 0.5
        p = ((q @ kd.transpose(-1, -2)[None]) * (T * d ** -0.5)).softmax(-1)
        want = ref.to_out((p @ vd[None]).transpose(1, 2).reshape(b, n, heads * d))
        attn = attn.to(dtype)
        got = attn(x.to(dtype), q_injected=qi.to(dtype) if injected_q else None, k_injected=kv, v_injected=kv,
                   injection_config={"T": T, "gamma": gamma})
    assert got.dtype == dtype and got.shape == want.shape
    assert rel_err(got.float().cpu().numpy(), want.numpy()) < tol


def test_negative_temperature_takes_the_numbers():
    torch.manual_seed(6)
    attn = CrossAttention(80, heads=2, dim_head=40).to(DEV)
    attn.cnt_name = "/nowhere/img.jpg"
    x, (k, v) = torch.randn(2, 9, 80, device=DEV), torch.randn(2, 2, 33, 40, device=DEV)
    kv = ops.kv_cache(1, 2, 33, 40, "int8", DEV)
    ops.kv_cache_write(kv, k[None], v[None])
    kn, vn = (t[0] for t in ops.kv_cache_read(kv, 0, 33, torch.float32))
    with torch.no_grad():
        got = attn(x, k_injected=kv, v_injected=kv, injection_config={"T": -1.0, "gamma": 0.5})
        want = attn(x, k_injected=kn, v_injected=vn, injection_config={"T": -1.0, "gamma": 0.5})
    assert torch.equal(got, want)


def test_channels_last_network_equals_the_stock_one():
    """float32 sums in another order, through some sixty layers: 1e-3 of the largest value."""
    x = torch.from_numpy(synth.normal(8400, (2, 4, 16, 16))).to(DEV)
    ctx = torch.from_numpy(synth.normal(8500, (1, 77, 768), sigma=0.5)).to(DEV).expand(2, -1, -1).contiguous()
    t = torch.tensor([481, 21], device=DEV)
    out = []
    for cl in (False, True):
        model = build(cl)
        for a in model.attention_modules():
            a.compute = "fp32"
        with torch.no_grad():
            out.append(model(x, t, ctx))
    assert out[1].is_contiguous()
    assert rel_err(out[1].cpu().numpy(), out[0].cpu().numpy()) < 1e-3


def test_high_frequency_patch_channels_last():
    """The patched decoder blocks add HF(h_cnt) to what a channels-last block leaves, as to what the stock one leaves."""
    from style_transfer_amd.high_frequency import patch_decoder_resblocks_h_and_cnt_hf, unpatch_decoder_resblocks
    from style_transfer_amd.sampler import capture_residuals, last_resblocks
    x = torch.from_numpy(synth.normal(8400, (1, 4, 16, 16))).to(DEV)
    ctx = torch.from_numpy(synth.normal(8500, (1, 77, 768), sigma=0.5)).to(DEV)
    t = torch.tensor([481], device=DEV)
    out, bare = [], None
    for cl in (False, True):
        model = build(cl)
        for a in model.attention_modules():
            a.compute = "fp32"
        with torch.no_grad():
            bare = model(x, t, ctx)
            residuals = {481: capture_residuals(model)}
            patch_decoder_resblocks_h_and_cnt_hf(model, {481}, residuals, ratio=0.3)
            for _, m in last_resblocks(model):
                m.ri_timestep = 481
            try:
                out.append(model(x, t, ctx))
            finally:
                unpatch_decoder_resblocks(model)
    assert rel_err(out[1].cpu().numpy(), out[0].cpu().numpy()) < 1e-3
    assert rel_err(out[1].cpu().numpy(), bare.cpu().numpy()) > 1e-2          # the patch does something


def test_resblock_gradients_channels_last():
    """Forward and every gradient of a ResBlock against 64 bits; the convolutions sum up to 9 * 96 products in float32:
    sqrt(864) * 2^-24 relative a layer, far below 1e-4."""
    torch.manual_seed(7)
    block = U.ResBlock(96, 32, 64)
    ref = copy.deepcopy(block).double()
    for m in ref.modules():
        if isinstance(m, U.GroupNorm32):
            m.__class__ = torch.nn.GroupNorm                # without the cast to float32
    block = block.to(DEV).to(memory_format=torch.channels_last)
    block.fused_norm = True
    x, emb, g = torch.randn(2, 96, 12, 10), torch.randn(2, 32), torch.randn(2, 64, 12, 10)
    xr, er = x.double().requires_grad_(), emb.double().requires_grad_()
    (ref(xr, er) * g.double()).sum().backward()
    xd, ed = x.to(DEV).requires_grad_(), emb.to(DEV).requires_grad_()
    y = block(xd, ed)
    (y * g.to(DEV)).sum().backward()
    pairs = [(y, ref(xr, er)), (xd.grad, xr.grad), (ed.grad, er.grad)]
    pairs += [(p.grad, q.grad) for p, q in zip(block.parameters(), ref.parameters())]
    for got, want in pairs:
        assert rel_err(got.detach().float().cpu().numpy(), want.detach().numpy()) < 1e-4


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_batch_behind_one_style_eager_and_captured(fmt):
    """The three operators together, as a run uses them: two images behind one 8-bit style entry through the channels-last
    network, eagerly and as a captured graph whose slots take another step's entry each time, against the stock network on
    the same numbers as tensors (2e-2: the bar of the default arithmetic through the whole network)."""
    store = fs.FeatureStore(on_device(feature_list(1, 3)), on_device(feature_list(2, 3)))
    before = store.nbytes()
    store.quantize(heads=8, fmt=fmt)
    assert store.nbytes() < before
    assert isinstance(store.char[0]["output_block_6_self_attn_k"], ops.QuantKV)
    assert torch.is_tensor(store.char[0]["output_block_9_self_attn_k"])          # head_dim 20
    numbers = read_back(store.char)

    def step(i, sty):
        e = {"config": {"gamma": 0.75, "T": 1.5}}
        for k in sty[i]:
            if "_self_attn_" in k:
                e[k] = store.cnt[i][k] if k.endswith("q") else sty[i][k]
        return e

    x = torch.from_numpy(synth.normal(8400, (2, 4, 16, 16))).to(DEV)
    ctx = torch.from_numpy(synth.normal(8500, (1, 77, 768), sigma=0.5)).to(DEV).expand(2, -1, -1).contiguous()
    stock, model = build(False), build(True)
    graph = GraphedUNet(model)
    seen = []
    with torch.no_grad():
        for i in (0, 1, 2, 0, 1):
            t = torch.tensor([981 - 20 * i] * 2, device=DEV)
            want = stock(x, t, ctx, injected_features=step(i, numbers)).cpu().numpy()
            eager = model(x, t, ctx, injected_features=step(i, store.char)).cpu().numpy()
            torch.cuda.synchronize()
            replay = graph(x, t, ctx, injected_features=step(i, store.char)).cpu().numpy()
            assert rel_err(eager, want) < 2e-2
            assert rel_err(replay, eager) < 2e-3          # the library's convolutions differ by this much between runs
            seen.append(replay)
    assert rel_err(seen[1], seen[0]) > 1e-2               # every step reads its own entry
    assert rel_err(seen[3], seen[0]) < 2e-3
    # a format change under the same keys is captured anew, not replayed over the old slots
    other = fs.FeatureStore(store.cnt, on_device(feature_list(2, 3))).quantize(8, "e4m3" if fmt == "int8" else "int8")
    with torch.no_grad():
        t = torch.tensor([981, 981], device=DEV)
        assert rel_err(graph(x, t, ctx, injected_features=step(0, other.char)).cpu().numpy(),
                       model(x, t, ctx, injected_features=step(0, other.char)).cpu().numpy()) < 2e-3


def make_root(tmp_path, lines, masks=()):
    root, pre = tmp_path / "data", tmp_path / "pre"
    for sub in ("cnt", "sty/char", "sty/back"):
        os.makedirs(root / sub, exist_ok=True)
    os.makedirs(pre, exist_ok=True)
    done = set()
    for ln in lines:
        for sub, name, suffix in zip(("cnt", "sty/char", "sty/back"), ln.split(), ("_cnt.pkl", "_sty.pkl", "_sty.pkl")):
            (root / sub / name).write_bytes(b"x")
            f = os.path.splitext(name)[0] + suffix
            if f not in done:
                done.add(f)
                fs.save_feature_file(str(pre / f), feature_list(20 + len(done)))
    (root / "dataset.txt").write_text("\n".join(lines) + "\n")
    for n in masks:
        np.save(str(root / "cnt" / (n + "_mask.npy")), load_masks()[CASE["mask"]])
    (tmp_path / "unet.json").write_text(json.dumps(CFG))
    return root, pre


@pytest.mark.parametrize("extra", [[], ["--graph_unet"], ["--lanes", "2"]], ids=["eager", "graph", "lanes"])
def test_command_line_with_both_flags(tmp_path, extra):
    """Two single-style lines and one two-style line that shares a style with them: the 8-bit and the packed entry of that
    style live side by side.  Against the stock run: int8 rows are off by at most 1/254 of their largest value and the
    default arithmetic by 2e-2 through the network; both together stay within 5e-2 after the steps of this run."""
    from style_transfer_amd import run as cli
    root, pre = make_root(tmp_path, ["c1.jpg a.png", "c2.jpg a.png", "c3.jpg a.png b.png"], masks=("c3",))
    args = ["--data_root", str(root), "--precomputed", str(pre), "--random_unet", "--unet_config", str(tmp_path / "unet.json"),
            "--H", "128", "--W", "128", "--start_step", "4", "--gamma", "0.75", "--T", "1.5"] + extra
    cli.main(args + ["--output_path", str(tmp_path / "stock")])
    cli.main(args + ["--output_path", str(tmp_path / "fused"), "--quantize_store", "int8", "--channels_last"])
    want = torch.load(str(tmp_path / "stock" / "latents_all.pt"), weights_only=True)
    got = torch.load(str(tmp_path / "fused" / "latents_all.pt"), weights_only=True)
    assert tuple(got.shape) == (3, 4, 16, 16) and torch.isfinite(got).all()
    for a, b in zip(got, want):
        assert rel_err(a.numpy(), b.numpy()) < 5e-2


def test_loader_quantises_and_keeps_its_allocations(tmp_path):
    root, pre = make_root(tmp_path, ["c1.jpg a.png"])
    loader = FeatureLoader(str(pre), DEV, heads=8, quantize="e4m3")
    loader.request(("c1", "a", None))
    store = loader.get(("c1", "a", None))
    kv = store.char[3]["output_block_7_self_attn_k"]
    assert isinstance(kv, ops.QuantKV) and kv is store.char[3]["output_block_7_self_attn_v"]
    host = fs.load_feature_file(str(pre / "a_sty.pkl"), DEV)
    want = fs.FeatureStore(host, host).quantize(8, "e4m3").char[3]["output_block_7_self_attn_k"]
    torch.cuda.synchronize()
    for a, b in zip(kv.tensors(), want.tensors()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    blocks = {t.untyped_storage().data_ptr() for t in loader._cache[("sty1", "a")].blocks}
    assert all(t.untyped_storage().data_ptr() in blocks for t in kv.tensors())
    loader.close()


def test_scratch_is_the_calls_own():
    """Two graphs captured on one stream, replayed on two streams at once with eager calls between: each keeps its results
    (long lists of keys for few queries, so every call passes partial results through scratch memory)."""
    torch.manual_seed(8)
    q = [torch.randn(2, 8, 1, 64, device=DEV, dtype=torch.float16) for _ in range(2)]
    pre = [tuple(torch.randn(8, 4096, 64, device=DEV, dtype=torch.float16) for _ in range(2)) for _ in range(2)]
    x = [torch.randn(2, 40, 40, 64, device=DEV).permute(0, 3, 1, 2) for _ in range(2)]
    call = lambda i: (ops.shared_prefix_attention(q[i], pre[i]), ops.group_norm_act(x[i], 1))
    want = [call(i) for i in range(2)]
    stream, graphs, outs = torch.cuda.Stream(), [], []
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):          # no call warmed this stream up
            outs.append(call(i))
        graphs.append(g)
    lanes = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for i in range(2):
            for t in outs[i]:
                t.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(lanes[i]):
                graphs[i].replay()
        eager = [call(i) for i in range(2)]
        torch.cuda.synchronize()
        for i in range(2):
            for a, b, c in zip(outs[i], want[i], eager[i]):
                assert torch.equal(a, b) and torch.equal(c, b)


def test_threads_on_one_stream():
    """Calls of two threads on one stream interleave their launches; every call's partial results are its own."""
    import threading
    torch.manual_seed(9)
    q = [torch.randn(2, 8, 1, 64, device=DEV, dtype=torch.float16) for _ in range(2)]
    pre = [tuple(torch.randn(8, 4096, 64, device=DEV, dtype=torch.float16) for _ in range(2)) for _ in range(2)]
    x = [torch.randn(2, 70, 64, 64, device=DEV).permute(0, 3, 1, 2) for _ in range(2)]
    call = lambda i: (ops.shared_prefix_attention(q[i], pre[i]), ops.group_norm_act(x[i], 1))
    want, bad = [call(i) for i in range(2)], []

    def work(i):
        for _ in range(100):
            if not all(torch.equal(a, b) for a, b in zip(call(i), want[i])):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_training_step_captured():
    """Forward and backward of the group norm in one graph, replayed on new values."""
    torch.manual_seed(10)
    x = torch.randn(2, 30, 30, 64, device=DEV).permute(0, 3, 1, 2).requires_grad_()
    w, b = (torch.randn(64, device=DEV).requires_grad_() for _ in range(2))
    dy = torch.randn(2, 30, 30, 64, device=DEV).permute(0, 3, 1, 2)

    def step():
        y = ops.group_norm_act(x, 4, w, b)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    for _ in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(2, 30, 30, 64, device=DEV).permute(0, 3, 1, 2))
        graph.replay()
        got = [t.clone() for t in out]
        for a, c in zip(got, step()):
            assert torch.equal(a, c)
        torch.cuda.synchronize()
