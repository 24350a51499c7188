"""Benchmark configuration 3's input generator (bench_reads.py) against outputs of the reference's
own code (tests/golden/reads_golden.npz, written by tests/golden/make_reads_golden.py from the
reference's PoreModel, tile_read, SignalEncoder, SignalEvalModel and AveragePooler): the
synthetic pore-model signal and the window offsets must be identical, the seeded encoder must
start from the same weights, and the fp32 window embeddings must agree to 1e-5."""
import os

import numpy as np
import pytest
import torch

import bench_reads as BR

GOLD = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden", "reads_golden.npz")


@pytest.fixture(scope="module")
def gold():
    return np.load(GOLD)


def test_pore_model_signal_is_identical(gold):
    sig = BR.sequence_to_signal(gold["codes"].astype(np.int64), BR.kmer_levels())
    assert sig.dtype == np.float32 and np.array_equal(sig, gold["signal"])


def test_window_offsets_follow_tile_read(gold):
    offs = np.split(gold["offsets"], np.cumsum(gold["offsets_count"])[:-1])
    for n, want in zip(gold["lengths"].tolist(), offs):
        got = np.array(BR.window_offsets(n), np.int64).reshape(-1, 2)
        assert np.array_equal(got, want), n
    # the batched tiling of bench_reads gives the same windows
    lens = torch.tensor([n for n in gold["lengths"].tolist() if n > 0])
    sig = torch.arange(int(lens.max()), dtype=torch.float32)[None, :].repeat(len(lens), 1)
    w, val, rid = BR.read_windows(sig, lens)
    k = 0
    for r, n in enumerate(lens.tolist()):
        for off, v in BR.window_offsets(n):
            assert rid[k].item() == r and val[k].item() == v
            assert torch.equal(w[k, :v], sig[r, off:off + v]) and not w[k, v:].any()
            k += 1
    assert k == w.shape[0]


def test_encoder_weights_windows_and_embeddings(gold):
    enc = BR.make_encoder(int(gold["enc_seed"]), "cpu")
    chk = np.array([float(p.detach().double().sum()) for p in enc.parameters()])
    assert np.array_equal(chk, gold["weights_checksum"])  # same initial weights as the reference
    lens = gold["window_lengths"]
    parts = np.split(gold["windows"], np.cumsum(lens)[:-1])
    sig = torch.zeros((len(parts), BR.WIN))
    for i, p in enumerate(parts):
        sig[i, :len(p)] = torch.from_numpy(p)
    val = torch.from_numpy(lens.astype(np.int64))
    x, mask_t = BR.prep_windows(sig, val)
    assert np.allclose(x.numpy(), gold["prepped"], rtol=0, atol=1e-5)
    assert np.array_equal(mask_t.numpy(), gold["mask_t"])
    emb = BR.encode_windows(enc, sig, val, amp=False).numpy()
    assert np.allclose(emb, gold["embeddings"], rtol=0, atol=1e-5)


def test_simulated_reads_have_the_configured_shape():
    gen = torch.Generator().manual_seed(5)
    genome = torch.randint(0, 4, (200_000,), generator=gen, dtype=torch.uint8)
    codes, lens, starts, rc = BR.simulate_reads(genome, 64, 5000, gen)
    assert codes.shape[0] == 64 and ((lens > 4800) & (lens < 5200)).all()
    assert abs(lens.float().mean().item() - 5000) < 25  # 2 % insertions balance 2 % deletions
    assert 0.3 < rc.float().mean().item() < 0.7
    for r in range(64):  # every base code is valid up to the read's length, -1 after it
        row = codes[r]
        assert (row[:lens[r]] >= 0).all() and (row[:lens[r]] < 4).all() and (row[lens[r]:] == -1).all()
    # forward reads start with the genome (matching the first 20 template bases, errors aside)
    fwd = [r for r in range(64) if not rc[r]]
    agree = np.mean([(codes[r, :20] == genome[starts[r]:starts[r] + 20].long()).float().mean().item() for r in fwd])
    assert agree > 0.7


@pytest.mark.gpu
def test_encoder_on_the_library_operators():
    """encode_windows(kernels=True) against the fp32 encoder: per block eight results on the path are
    rounded to 16 bits (two norms, five projections or sums, the attention product) and four around
    the blocks; each moves the norm of what passes by at most u, one half of fp16's eps."""
    enc = BR.make_encoder(4242, "cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    sig = 90 + 20 * torch.randn((37, BR.WIN), generator=gen, device="cuda")
    val = torch.full((37,), BR.WIN, device="cuda", dtype=torch.long)
    val[5], val[20], val[36] = 1500, 1000, 1733
    sig *= torch.arange(BR.WIN, device="cuda")[None, :] < val[:, None]
    want = BR.encode_windows(enc, sig, val, amp=False)
    got = BR.encode_windows(enc, sig, val, kernels=True)
    u = torch.finfo(torch.float16).eps / 2
    rel = ((got - want).norm(dim=1) / want.norm(dim=1)).max()
    assert float(rel) <= (8 * 6 + 4) * u
    again = BR.encode_windows(enc, sig, val, kernels=True)
    assert torch.equal(got, again)


@pytest.mark.gpu
def test_encoder_on_the_library_operators_trains():
    """A contrastive step through the encoder: every weight gets a gradient near the fp32 encoder's (twice
    the roundings of the forward pass: each layer's backward pass rounds as often)."""
    import torch.nn.functional as F
    enc = BR.make_encoder(7, "cuda", d=64, heads=2)
    gen = torch.Generator(device="cuda").manual_seed(2)
    sig = 90 + 20 * torch.randn((12, BR.WIN), generator=gen, device="cuda")
    x, mask_t = BR.prep_windows(sig, torch.full((12,), BR.WIN, device="cuda"))
    bank = F.normalize(torch.randn((100, 64), generator=gen, device="cuda"), dim=1)
    target = torch.arange(12, device="cuda") * 8
    names = [n for n, _ in enc.named_parameters() if not n.startswith("conv")]
    params = [p for n, p in enc.named_parameters() if not n.startswith("conv")]

    def embed(h):
        return F.normalize(h.float().mean(1), dim=-1)

    e = embed(enc.forward_kernels(x, mask_t)).half()
    loss = torch.ops.rbq.softmax_loss(e, bank.half(), target, 5.0)[0]
    got = torch.autograd.grad(1024.0 * loss.mean(), params)
    logits = 5.0 * embed(enc(x, mask_t)) @ bank.half().float().t()
    want = torch.autograd.grad(1024.0 * F.cross_entropy(logits, target), params)
    u = torch.finfo(torch.float16).eps / 2
    for n, a, b in zip(names, got, want):
        assert float((a - b).norm()) <= 2 * (8 * 6 + 6) * u * float(b.norm()) + 1e-6, n
