"""vqb_rotary_append against the rotation in 64 bits.

Tolerance, before any run: the output takes one rounding (half a unit: 2^-8 of
the value in bf16, 2^-11 in fp16, 2^-25 absolute among fp16 subnormals).  The
fraction of a turn is exact to 2^-32, its fp32 rounding adds at most 2^-25 turns
(2 pi 2^-25 < 2^-22 radians), sine and cosine 2 ulp (2^-23 * 2) and three fp32
operations 2^-24 each of |a| + |b|: under 2^-20 (|a| + |b|) amplitude in all.
"""
import math

import numpy as np
import pytest
import torch

from vqlab_b200 import rotary, rotary_append, rotary_frequencies

pytestmark = pytest.mark.gpu
HALF_UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}  # 2^-8, 2^-11


def reference(x, positions, freq, interleaved, amplitude):
    """(rotated x, |a| + |b| of each element's pair) in float64 on the host."""
    x = x.detach().cpu().double().numpy()
    rot = 2 * freq.numel()
    turns = np.array([[((int(p) * int(f)) % (1 << 64)) / 2.0 ** 64 for f in freq.tolist()] for p in positions.tolist()])
    turns = turns.reshape(len(positions), 1, rot // 2)
    c, s = np.cos(2 * np.pi * turns) * amplitude, np.sin(2 * np.pi * turns) * amplitude
    i0, i1 = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(rot // 2),
                                                                               np.arange(rot // 2, rot))
    a, b = x[..., i0], x[..., i1]
    out, size = x.copy(), np.zeros_like(x)
    out[..., i0], out[..., i1] = a * c - b * s, b * c + a * s
    size[..., i0] = size[..., i1] = (np.abs(a) + np.abs(b)) * amplitude
    return out, size


def close(got, want, size, dtype):
    got = got.detach().cpu().double().numpy()
    lim = HALF_UNIT[dtype] * np.abs(want) + 2.0 ** -20 * size + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
    bad = np.abs(got - want) > lim
    assert not bad.any(), (int(bad.sum()), float(np.max(np.abs(got - want) / lim)))


def tensors(N, H, KH, D, dtype, page, pages, seed, fused=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((N, H + 2 * KH, D), device="cuda", generator=g).to(dtype)
    q, k, v = x[:, :H], x[:, H:H + KH], x[:, H + KH:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    kc = torch.randn((pages, KH, page, D), device="cuda", generator=g).to(dtype)
    vc = torch.randn((pages, KH, page, D), device="cuda", generator=g).to(dtype)
    return q, k, v, kc, vc


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("N,H,KH,D,rot,page,far", [
    (1, 40, 8, 128, 128, 16, 5000), (3, 5, 1, 64, 64, 16, 1 << 20), (37, 8, 2, 128, 64, 32, 100000),
    (37, 3, 3, 128, 124, 64, 1000), (9, 6, 2, 80, 20, 1, 4096), (700, 4, 1, 64, 16, 128, 2 ** 31 - 1),
    (5, 4, 2, 64, 2, 16, 77), (601, 2, 1, 34, 34, 16, 50), (4, 2, 2, 128, 0, 16, 9)])
def test_against_64_bits(dtype, interleaved, N, H, KH, D, rot, page, far):
    rng = np.random.default_rng(N * D + rot)
    pages = -(-N // page) + 2
    q, k, v, kc, vc = tensors(N, H, KH, D, dtype, page, pages, N + rot)
    freq = rotary_frequencies(rot, 10000.0)[0] if rot else torch.empty(0, dtype=torch.int64, device="cuda")
    pos = rng.integers(0, far + 1, N)
    pos[-1] = far
    slots = rng.permutation(pages * page)[:N]
    slots[rng.random(N) < 0.2] = -1
    if N > 3:
        slots[2] = pages * page  # outside the pool
    amp = 1.25
    kc0, vc0 = kc.clone(), vc.clone()
    dpos, dslots = (torch.from_numpy(a).to("cuda", torch.int32) for a in (pos, slots))
    got = rotary_append(q, k, v, dpos, freq, kc, vc, dslots, interleaved=interleaved, amplitude=amp)
    want, size = reference(q, pos, freq, interleaved, amp)
    close(got, want, size, dtype)
    want, size = reference(k, pos, freq, interleaved, amp)
    flat = lambda t: t.transpose(1, 2).reshape(-1, KH, D)  # noqa: E731
    keep = [i for i in range(N) if 0 <= slots[i] < pages * page]
    close(flat(kc)[slots[keep]], want[keep], size[keep], dtype)
    assert torch.equal(flat(vc)[slots[keep]], v[keep])
    rest = np.setdiff1d(np.arange(pages * page), slots[keep])
    assert torch.equal(flat(kc)[rest], flat(kc0)[rest]) and torch.equal(flat(vc)[rest], flat(vc0)[rest])


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_alone(interleaved):
    x = torch.randn((19, 6, 128), device="cuda").to(torch.bfloat16)
    freq, amp = rotary_frequencies(96, 1e6, "linear", 4.0)
    pos = torch.arange(100, 119, dtype=torch.int32, device="cuda")
    want, size = reference(x, pos, freq, interleaved, amp)
    close(rotary(x, pos, freq, interleaved=interleaved, amplitude=amp), want, size, torch.bfloat16)
    y = x.clone()
    assert rotary(y, pos, freq, interleaved=interleaved, amplitude=amp, out=y) is y
    close(y, want, size, torch.bfloat16)


@pytest.mark.parametrize("shift", [1, 2, 4])
def test_unaligned_and_strided(shift):
    """Heads that start off a 16-byte boundary, tokens far apart, a token-major cache."""
    N, H, KH, D, page, pages = 11, 4, 2, 64, 16, 3
    buf = torch.randn(N * 1000 + 8, device="cuda").to(torch.float16)
    x = buf[shift:shift + N * 1000].view(N, 1000)
    q, k, v = (x[:, a:a + n * D].view(N, n, D) if False else x[:, a:a + n * D].unflatten(1, (n, D))
               for a, n in ((0, H), (H * D + 6, KH), ((H + KH) * D + 12, KH)))
    kc = torch.zeros((pages, page, KH, D), dtype=torch.float16, device="cuda").transpose(1, 2)
    vc = torch.zeros((pages, page, KH, D), dtype=torch.float16, device="cuda").transpose(1, 2)
    freq, _ = rotary_frequencies(64)
    pos = torch.arange(N, dtype=torch.int32, device="cuda")
    slots = torch.arange(20, 20 + N, dtype=torch.int32, device="cuda")
    got = rotary_append(q, k, v, pos, freq, kc, vc, slots)
    want, size = reference(q, pos, freq, False, 1.0)
    close(got, want, size, torch.float16)
    want, size = reference(k, pos, freq, False, 1.0)
    close(kc.transpose(1, 2).reshape(-1, KH, D)[20:20 + N], want, size, torch.float16)
    assert torch.equal(vc.transpose(1, 2).reshape(-1, KH, D)[20:20 + N], v)


def test_slots_past_32_bits():
    """A pool of over 2^31 elements, the slots at its end."""
    q, k, v, _, _ = tensors(5, 4, 2, 128, torch.float16, 64, 1, 3)
    pages = 140000
    kc, vc = (torch.empty((pages, 2, 64, 128), dtype=torch.float16, device="cuda") for _ in range(2))
    assert kc.numel() > 2 ** 31
    freq, _ = rotary_frequencies(128)
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    slots = (pages * 64 - 1 - 13 * torch.arange(5, device="cuda")).to(torch.int32)
    rotary_append(q, k, v, pos, freq, kc, vc, slots)
    want, size = reference(k, pos, freq, False, 1.0)
    page, off = (slots // 64).long(), (slots % 64).long()
    close(kc[page, :, off], want, size, torch.float16)
    assert torch.equal(vc[page, :, off], v)


def test_rotation_keeps_relative_scores():
    """q.k after rotation depends on the positions' difference alone, also at far positions."""
    freq, _ = rotary_frequencies(128, 1e6)
    q, k = (torch.randn((1, 1, 128), device="cuda").to(torch.float16) for _ in range(2))
    scores = []
    for start in (0, 1 << 20, (1 << 31) - 100):
        at = lambda p: torch.tensor([p], dtype=torch.int32, device="cuda")  # noqa: E731
        a, b = rotary(q, at(start + 37), freq), rotary(k, at(start), freq)
        scores.append(float((a.double() * b.double()).sum()))
    # each of the 128 products has two roundings of 2^-11 of its size
    bound = 2 * 2.0 ** -11 * float((q.double().abs().sum() * k.double().abs().max()))
    assert max(scores) - min(scores) <= bound


def test_frequencies():
    """Each scaling against its formula (turns per position, 2^-64 resolution)."""
    base, d = 10000.0, 64
    plain = np.array([base ** (-2 * i / d) for i in range(d // 2)]) / (2 * math.pi)
    as_turns = lambda f: np.array([(int(v) % (1 << 64)) / 2.0 ** 64 for v in f.tolist()])  # noqa: E731
    assert np.allclose(as_turns(rotary_frequencies(d, base)[0]), plain, rtol=1e-14)
    assert np.allclose(as_turns(rotary_frequencies(d, base, "linear", 8.0)[0]), plain / 8, rtol=1e-14)
    f = as_turns(rotary_frequencies(d, base, "base", 8.0)[0])
    assert np.allclose(f[0], plain[0], rtol=1e-14) and np.allclose(f[-1], plain[-1] / 8, rtol=1e-12)
    f, amp = rotary_frequencies(d, base, "ramp", 8.0, original_length=4096, low=1.0, high=32.0)
    f, turns = as_turns(f), plain * 4096
    assert np.allclose(f[turns > 40], plain[turns > 40], rtol=1e-14) and (turns > 40).any()
    assert np.allclose(f[turns < 0.7], plain[turns < 0.7] / 8, rtol=1e-12) and (turns < 0.7).any()
    assert abs(amp - (0.1 * math.log(8) + 1)) < 1e-15
    for bad in (dict(rotary_dim=3), dict(rotary_dim=8, scaling="x"), dict(rotary_dim=8, scaling="ramp")):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_refusals():
    q, k, v, kc, vc = tensors(4, 4, 2, 64, torch.float16, 16, 2, 0)
    freq, _ = rotary_frequencies(64)
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    args = dict(positions=pos, freq=freq, k_cache=kc, v_cache=vc, slots=pos)
    rotary_append(q, k, v, **args)
    assert rotary_append(q[:0], k[:0], v[:0], **args).shape == (0, 4, 64)
    for change in (dict(positions=pos[:3]), dict(positions=pos.long()), dict(slots=pos[:2]),
                   dict(freq=torch.zeros(33, dtype=torch.int64, device="cuda")), dict(k_cache=kc.bfloat16()),
                   dict(v_cache=vc[:1]), dict(k_cache=kc[:, :1])):
        with pytest.raises(ValueError):
            rotary_append(q, k, v, **{**args, **change})
    with pytest.raises(ValueError):
        rotary_append(q.float(), k, v, **args)
    with pytest.raises(ValueError):
        rotary_append(q, k[:, :1], v, **args)
    with pytest.raises(ValueError):
        rotary(q.cpu(), pos, freq)
