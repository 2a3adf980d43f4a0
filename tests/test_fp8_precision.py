"""
Precision "fp8" of the embedding path: block outputs, catconv's and the first convs' weights in 8 bits with block scales,
everything else as in "bf16".

Bars.  Rounding to e4m3 is off by at most 2^-4 of a value, evenly spread at worst: 2^-4 / sqrt(3) = 0.036 in the mean
square.  A product has two rounded factors, so sums of products are off by at most 0.036 sqrt(2) = 0.051 of their norm (the
errors of the terms are independent, and the terms add like them).  One such layer is followed by others that see a relative
error of their input: an embedding off by 0.051 of its norm has a cosine of 1 - 0.051^2 / 2 = 0.9987 with the exact one;
the bar for whole embeddings is 0.998.
"""
import ctypes as C

import pytest
import torch
import torch.nn.functional as F

import sugar_amd
from oracle import ref_cpu
from sugar_amd import _lib, layout, synth
from sugar_amd.graphs import GraphedEmbedder

gpu = pytest.mark.gpu
DEV = "cuda:0"
CONFIGS = {
    "base": layout.BASE,                                              # first convs in 8 bits (512 channels = 4 blocks)
    "largest": layout.LARGEST,
    "smallest": layout.SMALLEST,                                      # 128 channels: one block a slice, 16-bit first convs
    "three_blocks": (3, [384, 256, 384, 176], [3, 1, 3, 5], 768),     # a slice of three blocks: exponents off the dword
    "odd": (4, [176, 136, 256, 176, 200], [5, 3, 1, 5, 3], 536),      # a slice that ends inside its second block
}


def model_of(supernet, cfg, precision):
    sub = supernet.clone(cfg).set_precision(precision)
    supernet.config = None
    return sugar_amd.WrappedModel(sugar_amd.SpeakerModel(sub, transform=sugar_amd.LogMelFbanks())).to(DEV).eval()


def test_precision_names(supernet):
    sub = supernet.clone(layout.SMALLEST)
    supernet.config = None
    g = sub.generation
    assert sub.set_precision("fp8") is sub and sub.dtype_id == _lib.SUGAR_FP8 and sub.feature_dtype == torch.bfloat16
    assert sub.generation == g + 1
    assert sub.set_precision("fp32").feature_dtype == torch.float32 and sub.set_precision("bf16").feature_dtype == torch.bfloat16
    with pytest.raises(ValueError):
        sub.set_precision("fp16")
    with pytest.raises(ValueError):
        sugar_amd.TDNNSubnet(layout.SMALLEST, precision="fp16")
    assert _lib.lib().sugar_subnet_create(C.byref(_lib.SugarSubnetDesc()), 3, 0, C.byref(C.c_void_p())) == -1


@gpu
@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_embeddings_match_the_oracle(name, supernet, sup_state):
    cfg = CONFIGS[name]
    wav = synth.waveforms(6, 20000, seed=3)
    want = ref_cpu.embed(ref_cpu.clone_state(sup_state, cfg), cfg[0], wav)
    model = model_of(supernet, cfg, "fp8")
    emb = model(wav.to(DEV)).cpu()
    cos = F.cosine_similarity(emb.double(), want.double(), dim=1)
    print(name, "cosine to the f32 oracle: min %.6f" % cos.min().item())
    assert cos.min() >= 0.998
    assert torch.equal(model(wav.to(DEV)).cpu(), emb)                   # repeats bit for bit


@gpu
def test_full_batch_and_ragged_lists(supernet, sup_state):
    """256 x 3 s (the persistent product, the 128 x 128 tiles) and utterances of unlike lengths in one call, against the
    same model's bf16 embeddings (cosine >= 0.999 to the oracle themselves)."""
    fp8, b16 = model_of(supernet, layout.BASE, "fp8"), model_of(supernet, layout.BASE, "bf16")
    g = torch.Generator(device=DEV).manual_seed(5)
    wav = torch.randn(256, 48000, device=DEV, generator=g)
    cos = F.cosine_similarity(fp8(wav).double(), b16(wav).double(), dim=1)
    print("256 x 3 s: cosine to bf16 min %.6f" % cos.min().item())
    assert cos.min() >= 0.998
    lens = [10000, 48000, 16000, 100000, 32001, 9999]
    wavs = [w.to(DEV) for w in synth.ragged_waveforms(lens, seed=2)]
    cos = F.cosine_similarity(fp8(wavs).double(), b16(wavs).double(), dim=1)
    assert cos.min() >= 0.998
    want = ref_cpu.embed_ragged(ref_cpu.clone_state(sup_state, layout.BASE), 3, [w.cpu() for w in wavs])
    assert F.cosine_similarity(fp8(wavs).cpu().double(), want.double(), dim=1).min() >= 0.998


@gpu
@pytest.mark.parametrize("name", ["base", "odd", "three_blocks"])
def test_stage_taps(name, supernet):
    """Every stage against the bf16 path: identical up to the first 8-bit rounding (block 0's end), relative errors within
    the bars above behind it (0.051 a layer of products in 8 bits)."""
    cfg = CONFIGS[name]
    T = 120
    feats = torch.randn(2 * T, 80, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    row_off = torch.tensor([0, T, 2 * T], dtype=torch.int32, device=DEV)
    subs = [supernet.clone(cfg).set_precision(p) for p in ("bf16", "fp8")]
    supernet.config = None
    rel = lambda a, b: ((a.double() - b.double()).norm() / b.double().norm()).item()
    taps = [0] + [1 + k for k in range(4 * cfg[0])] + [100, 102]
    for what in taps:
        want, got = [s.tap(feats, row_off, 2, 2 * T, T, what)[0] for s in subs]
        err = rel(got, want)
        if what <= 3:
            assert torch.equal(got, want), what
        elif what == 4:
            assert 0 < err <= 0.036                                     # one rounding
        else:
            assert err <= 0.051 * (1 + (what - 4) // 4 if what < 100 else cfg[0] + 1), (what, err)
    for s in subs:
        s.release()


@gpu
def test_graph_recalibration_and_precision_changes(supernet, sup_state):
    """A captured forward replays bit for bit; recalibration of an fp8 subnet moves the statistics as a bf16 one's and its
    eval path (first convs' affine included) uses them; precisions can be switched to and fro."""
    model = model_of(supernet, layout.BASE, "fp8")
    g = GraphedEmbedder(model, synth.waveforms(3, 32000, seed=1).to(DEV), normalize=True)
    for seed in (2, 3, 4):
        wav = synth.waveforms(3, 32000, seed=seed).to(DEV)
        got = g(wav).clone()
        ref = model(wav, normalize=True)
        torch.cuda.synchronize()
        assert torch.equal(got, ref)
    wav = synth.waveforms(8, 24000, seed=9).to(DEV)
    before = model(wav)
    sub = model.module.__S__
    sub.set_precision("bf16")
    other = model(wav)
    sub.set_precision("fp8")
    assert torch.equal(model(wav), before) and not torch.equal(other, before)
    pair = [model_of(supernet, layout.BASE, p) for p in ("fp8", "bf16")]
    for m in pair:
        m.train()
        for seed in (11, 12):
            m(synth.waveforms(8, 24000, seed=seed).to(DEV))
        m.eval()
    states = [m.module.__S__.state_dict() for m in pair]
    assert all(torch.equal(states[0][k], states[1][k]) for k in states[0])
    embs = [m(wav) for m in pair]
    assert F.cosine_similarity(embs[0].double(), embs[1].double(), dim=1).min() >= 0.998
    assert not torch.equal(embs[0], before)


@gpu
def test_host_packed_weights_are_the_quantisers(supernet):
    """catconv from its own tap: the block outputs in 8 bits times the weights as sugar_fp8_quant would give them."""
    cfg = CONFIGS["smallest"]
    sub = supernet.clone(cfg).set_precision("fp8")
    supernet.config = None
    T = 90
    feats = torch.randn(T, 80, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    row_off = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    outs = torch.cat([sub.tap(feats, row_off, 1, T, T, 4 + 4 * i)[0] for i in range(cfg[0])], 1)
    w = dict(sub.named_parameters())["catconv.weight"].detach()[:, :, 0].to(DEV)
    want = torch.relu(outs.double() @ sugar_amd.quantize_block_fp8(w.contiguous()).dequantize().double().t())
    got = sub.tap(feats, row_off, 1, T, T, 100)[0].double()
    # outs are the 8-bit values themselves; what differs is the product's float32 rounding (2^-13 cuts) and bf16's
    mag = outs.double().abs() @ w.double().abs().t()
    assert ((got - want).abs() <= 2.0 ** -8 * want + 2.0 ** -10 * mag).all()
    sub.release()


class _Utts:
    """Stand-in for sugar.database.Utterance: items are {"file", "input": [1, L]}."""

    def __init__(self, wavs):
        self.wavs = wavs

    def __len__(self):
        return len(self.wavs)

    def __getitem__(self, i):
        return {"file": "utt%04d.wav" % i, "input": self.wavs[i].unsqueeze(0)}


class _Trials(list):
    utterances = None


class _Loader:
    def __init__(self, dataset, batch_size):
        self.dataset, self.batch_size, self.num_workers = dataset, batch_size, 0


@gpu
def test_lists_and_sweeps(supernet, meta):
    """extract_vectors over a staged list, its features kept or not, against the model's own forward; a sweep over subnets in
    this precision, with and without recalibration, against one model at a time."""
    n = 12
    wavs = synth.ragged_waveforms(synth.ragged_lengths(n, lo=20000, hi=40000, seed=13).tolist(), seed=13)
    utts = _Utts(wavs)
    model = model_of(supernet, layout.BASE, "fp8")
    want = model([w.to(DEV) for w in wavs], normalize=True)
    tables = []
    for keep in (False, True, True):
        packed = sugar_amd.PackedUtterances(utts, DEV, batch_size=5, cache_features=keep)
        tables += [sugar_amd.extract_vectors(model, packed).matrix.clone() for _ in range(2)]
    assert all(torch.equal(t, tables[0]) for t in tables[1:])
    # other batches: another kernel may serve the same row (float32 sums in another order, then the same bf16 roundings)
    assert F.cosine_similarity(tables[0].double(), want.double(), dim=1).min() >= 0.9999
    lab, a, b = synth.trial_pairs(n, 120, seed=13)
    trials = _Trials({"label": int(lab[i]), "enroll": "utt%04d.wav" % a[i], "test": "utt%04d.wav" % b[i]} for i in range(len(lab)))
    trials.utterances = utts
    loader = _Loader(trials, 4)
    configs = [layout.SMALLEST, layout.BASE, CONFIGS["three_blocks"]]
    recal = [(synth.waveforms(6, 32000, seed=40),)]
    for recal_loader in (None, recal):
        got = sugar_amd.evaluate_subnets(supernet, configs, loader, recal_loader=recal_loader, device=DEV, precision="fp8")
        assert len(got) == len(configs)
        for cfg in configs:
            one = model_of(supernet, cfg, "fp8")
            if recal_loader is not None:
                sugar_amd.batch_forward(recal_loader, one, device=DEV)
            eer, dcf = sugar_amd.veri_validate(loader, one, device=DEV)
            r = got[(cfg[0], tuple(cfg[1]), tuple(cfg[2]), cfg[3])]
            assert r["eer"] == eer[0] and r["mindcf"] == dcf[0], (recal_loader is not None, cfg)


def test_stage_roofline_counts_8_bit_tensors_and_products():
    """bench.py's bytes and operations a stage, against counts written out here."""
    import bench
    B, T = 4, 301
    R, ones = B * T, {k: 1.0 for k in ("first_conv", "se_apply", "catconv", "last_conv")}
    e8 = 1 + 1 / 128
    got = {}
    for name in ("base", "three_blocks"):
        depth, ch, ks, ccat = CONFIGS[name]
        for p in ("bf16", "fp8"):
            got[name, p] = bench.stage_roofline(ones, CONFIGS[name], B, 48000, R, p)
            assert got[name, p]["catconv"]["gflop"] == round(2.0 * R * depth * ch[0] * ccat / 1e9, 2)
    mb = lambda per_row: round(per_row * R / 1e6, 1)
    c = 512                                             # base: 3 blocks of 512, all first convs but the first in 8 bits, 1536 out
    assert got["base", "bf16"]["se_apply"]["mbytes"] == mb(11 * c * 2) and got["base", "bf16"]["catconv"]["mbytes"] == mb((3 * c + 1536) * 2)
    assert got["base", "bf16"]["first_conv"]["mbytes"] == mb(3 * 2 * c * 2)
    assert got["base", "fp8"]["se_apply"]["mbytes"] == mb(2 * (6 + e8) * c + (4 + e8) * c)
    assert got["base", "fp8"]["catconv"]["mbytes"] == mb(3 * c * e8 + 1536 * 2)
    assert got["base", "fp8"]["first_conv"]["mbytes"] == mb(3 * c * 2 + c * 2 + 2 * c * e8)
    c = 384                                             # three scale blocks a slice: 16-bit first convs, block outputs in both types
    mid = [8 * (x // 8) for x in CONFIGS["three_blocks"][1][1:]]
    assert got["three_blocks", "fp8"]["first_conv"] == got["three_blocks", "bf16"]["first_conv"]
    assert got["three_blocks", "fp8"]["se_apply"]["mbytes"] == mb(2 * (8 + e8) * c + (4 + e8) * c)
    assert got["three_blocks", "fp8"]["last_conv"]["mbytes"] == mb(sum(m + c for m in mid) * 2)
    # a product that is bound by the matrix pipes: two of three first convs at twice the rate
    wide = (3, [4096, 4096, 4096, 4096], [5, 3, 3, 3], 1536)
    t = {p: bench.stage_roofline(ones, wide, B, 48000, R, p)["first_conv"] for p in ("bf16", "fp8")}
    assert t["bf16"]["bound"] == t["fp8"]["bound"] == "mfma" and abs(t["fp8"]["frac"] / t["bf16"]["frac"] - 2 / 3) < 0.02
