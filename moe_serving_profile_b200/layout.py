"""Device layout of the expert weights (built once, at load time).

Logically every format is ``[E_loc][planes][feat_pad][k_pad]`` (K
contiguous): gate/up (planes = 2) holds the gate rows in plane 0 and the up
rows in plane 1, both padded to ``I_p = ceil(I / 128) * 128`` features and
``H_k = ceil(H / 64) * 64`` reduction columns; down (planes = 1) is
``[E_loc][H_f][I_p]`` with ``H_f = ceil(H / 128) * 128``. GPT-OSS stores
gate/up interleaved (even / odd columns, moe_serving/gpt_oss_parallel.py:198);
it is de-interleaved here, once. Padding is zero (MXFP4 padding groups get
scale 127 = 2^0).

* BF16 weights stay in that layout (the GEMM streams 128-byte-swizzled tiles
  of it with TMA).
* Quantised weights (FP8 block-scaled E4M3, moe_serving/qwen3_parallel.py:48-70;
  MXFP4 E2M1 with ue8m0 group scales, gpt_oss_parallel.py:183-193) are packed
  into one contiguous blob per (expert, feature tile, 64-column k-block), the
  unit the GEMM converts, so each k-block arrives with a single bulk copy:
  ``[E_loc][feat_tiles][k_pad / 64][blob_bytes]``. A feature tile is 64
  features of a gated pair (rows 0-63 gate, 64-127 up) or 128 features of a
  single projection. A blob is 128 rows of 64 bytes (e4m3) or 32 bytes
  (e2m1 pairs), each row's 16-byte chunks permuted (chunk c of row r stored at
  c ^ ((r >> 1) & 3), resp. c ^ ((r >> 2) & 1)) so that one lane per row reads
  shared memory without bank conflicts, followed by the k-block's scales:
  FP8 with block scales covering whole 64 x 64 halves, the two fp32 scales of
  rows 0-63 and 64-127 plus 8 zero bytes; other FP8 blocks, 128 x 4 fp32
  (row, 16-column chunk); MXFP4, 128 x 2 ue8m0 bytes (row, 32-column group).
* Int8 weights (one fp32 scale per output channel) are stored as the 16 KB
  images the int8 GEMM multiplies from: ``[E_loc][feat_tiles][H_p / 128][128
  rows][128 columns]`` with ``H_p = ceil(H / 128) * 128``, chunk c of row r at
  c ^ (r & 7). Rows 32 j + 0..15 of a gated tile are the gate rows and 32 j +
  16..31 the up rows of features 16 j .. 16 j + 15. Scales and biases are fp32
  ``[E_loc][feat_tiles][128]`` in the same row order.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from moe_serving_profile_b200 import _lib
from moe_serving_profile_b200.ops import Int8Matrix


def _ceil(v: int, m: int) -> int:
    return (v + m - 1) // m * m


@dataclass
class ExpertWeights:
    """One layer's local experts in device layout: w1 (gate/up) and w2 (down)
    are bf16 [E, planes, F_p, K_p] for BF16 weights, packed blobs [E, feature
    tiles, K_p / 64, blob bytes] for FP8 / MXFP4 (scales inside) and tiles for
    int8 (m1 / m2 describe them, s1 / s2 and b1 / b2 are their scales and biases)."""

    fmt: int
    n_experts: int
    hidden: int
    inter: int
    w1: torch.Tensor
    w2: torch.Tensor
    s1: torch.Tensor | None = None
    s2: torch.Tensor | None = None
    b1: torch.Tensor | None = None
    b2: torch.Tensor | None = None
    block: tuple[int, int] = (128, 128)
    gated_epilogue: int = _lib.EPI_SWIGLU
    alpha: float = 1.702
    limit: float = 7.0
    m1: Int8Matrix | None = None
    m2: Int8Matrix | None = None

    @property
    def i_pad(self) -> int:
        return _ceil(self.inter, 128)

    @property
    def h_k(self) -> int:
        return _ceil(self.hidden, 128 if self.fmt == _lib.W_INT8 else 64)

    @property
    def h_f(self) -> int:
        return _ceil(self.hidden, 128)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in
                   (self.w1, self.w2, self.s1, self.s2, self.b1, self.b2) if t is not None)


def _tile_rows(w: torch.Tensor, planes: int) -> torch.Tensor:
    """[E, planes, F_p, C] -> [E, feat_tiles, 128, C]: a gated tile stacks 64
    gate rows over the 64 up rows of the same features; a single-plane tile
    takes 128 rows."""
    E, P, Fp, C = w.shape
    if planes == 2:
        return w.reshape(E, 2, Fp // 64, 64, C).permute(0, 2, 1, 3, 4).reshape(E, Fp // 64, 128, C)
    return w.reshape(E, Fp // 128, 128, C)


def _swizzle_sel(row_bytes: int) -> torch.Tensor:
    r = torch.arange(128)
    return ((r >> 1) & 3) if row_bytes == 64 else ((r >> 2) & 1)


def _kblock_rows(t: torch.Tensor, row_bytes: int) -> torch.Tensor:
    """[E, FT, 128, nkb * row_bytes] bytes -> [E, FT, nkb, 128 * row_bytes]
    with each row's 16-byte chunk c stored at position c ^ sel(row)."""
    E, FT, R, C = t.shape
    nkb, nch = C // row_bytes, row_bytes // 16
    t = t.reshape(E, FT, R, nkb, nch, 16).permute(0, 1, 3, 2, 4, 5)      # [E, FT, nkb, 128, nch, 16]
    src = torch.arange(nch)[None, :] ^ _swizzle_sel(row_bytes)[:, None]  # position p holds chunk p ^ sel
    idx = src.reshape(1, 1, 1, R, nch, 1).expand(E, FT, nkb, R, nch, 16).to(t.device)
    return torch.gather(t, 4, idx).reshape(E, FT, nkb, R * row_bytes)


def _fp8_blob_scales(s: torch.Tensor, planes: int, n_feat: int, feat_pad: int, k_pad: int,
                     block: tuple[int, int]) -> torch.Tensor:
    """Scale section of each FP8 blob: [E, FT, nkb, 16 or 2048] bytes."""
    E, P, nbr, nbc = s.shape
    br, bc = block
    feat_tile = 64 if planes == 2 else 128
    FT = feat_pad // feat_tile
    nkb = k_pad // 64
    dev = s.device
    s = s.float()
    if br % 64 == 0 and bc % 64 == 0:
        ft = torch.arange(FT, device=dev)
        sci = torch.clamp(torch.arange(nkb, device=dev) // (bc // 64), max=nbc - 1)
        out = torch.zeros(E, FT, nkb, 4, device=dev)
        for h in range(2):
            pl = h if planes == 2 else 0
            f = ft * feat_tile + (0 if planes == 2 else 64 * h)
            sri = torch.clamp(torch.clamp(f, max=n_feat - 1) // br, max=nbr - 1)
            out[..., h] = s[:, pl][:, sri][:, :, sci]
        return out.view(torch.uint8).reshape(E, FT, nkb, 16)
    r = torch.arange(128, device=dev)
    pl = (r // 64) if planes == 2 else torch.zeros_like(r)
    f = torch.arange(FT, device=dev)[:, None] * feat_tile + ((r % 64) if planes == 2 else r)[None, :]
    sri = torch.clamp(torch.clamp(f, max=n_feat - 1) // br, max=nbr - 1)          # [FT, 128]
    k0 = torch.arange(nkb, device=dev)[:, None] * 64 + torch.arange(4, device=dev)[None, :] * 16
    sci = torch.clamp(k0 // bc, max=nbc - 1)                                        # [nkb, 4]
    vals = s[:, pl[None, :].expand(FT, 128), sri]                                   # [E, FT, 128, nbc]
    out = vals[:, :, None, :, :].expand(E, FT, nkb, 128, nbc)
    idx = sci[None, None, :, None, :].expand(E, FT, nkb, 128, 4)
    return torch.gather(out, 4, idx).contiguous().view(torch.uint8).reshape(E, FT, nkb, 2048)


def pack_fp8_blobs(w: torch.Tensor, s: torch.Tensor, planes: int, n_feat: int,
                   block: tuple[int, int]) -> torch.Tensor:
    """e4m3 bytes [E, planes, F_p, k_pad] + fp32 block scales [E, planes, nbr, nbc]
    -> blobs [E, FT, k_pad / 64, 8192 + scale section]."""
    data = _kblock_rows(_tile_rows(w.view(torch.uint8), planes), 64)
    scales = _fp8_blob_scales(s, planes, n_feat, w.shape[2], w.shape[3], block)
    return torch.cat([data, scales], dim=-1).contiguous()


def pack_mxfp4_blobs(w: torch.Tensor, s: torch.Tensor, planes: int) -> torch.Tensor:
    """e2m1 pairs [E, planes, F_p, k_pad / 2] + ue8m0 scales [E, planes, F_p, k_pad / 32]
    -> blobs [E, FT, k_pad / 64, 4096 + 256]."""
    data = _kblock_rows(_tile_rows(w, planes), 32)
    st = _tile_rows(s, planes)                                    # [E, FT, 128, G]
    E, FT, R, G = st.shape
    sc = st.reshape(E, FT, R, G // 2, 2).permute(0, 1, 3, 2, 4).reshape(E, FT, G // 2, R * 2)
    return torch.cat([data, sc], dim=-1).contiguous()


def unpack_blob_rows(blobs: torch.Tensor, row_bytes: int, planes: int) -> torch.Tensor:
    """Inverse of the data part of the packing: blobs -> [E, planes, F_p, nkb * row_bytes]."""
    E, FT, nkb, _ = blobs.shape
    R, nch = 128, row_bytes // 16
    d = blobs[..., : R * row_bytes].reshape(E, FT, nkb, R, nch, 16)
    src = torch.arange(nch)[None, :] ^ _swizzle_sel(row_bytes)[:, None]   # involution
    idx = src.reshape(1, 1, 1, R, nch, 1).expand(E, FT, nkb, R, nch, 16).to(blobs.device)
    d = torch.gather(d, 4, idx).permute(0, 1, 3, 2, 4, 5).reshape(E, FT, R, nkb * row_bytes)
    if planes == 2:
        return d.reshape(E, FT, 2, 64, -1).permute(0, 2, 1, 3, 4).reshape(E, 2, FT * 64, -1)
    return d.reshape(E, 1, FT * 128, -1)


def _check_dims(hidden: int, inter: int) -> None:
    if hidden % 8 or inter % 8:
        raise NotImplementedError(
            f"hidden ({hidden}) and intermediate ({inter}) sizes must be multiples of 8")


def fp8_experts(gate: torch.Tensor, gate_scale: torch.Tensor, up: torch.Tensor,
                up_scale: torch.Tensor, down: torch.Tensor, down_scale: torch.Tensor,
                block: tuple[int, int]) -> ExpertWeights:
    """gate/up: e4m3 [E, I, H] with scales [E, ceil(I/br), ceil(H/bc)];
    down: e4m3 [E, H, I] with scales [E, ceil(H/br), ceil(I/bc)]."""
    E, inter, hidden = gate.shape
    _check_dims(hidden, inter)
    br, bc = block
    if bc % 16:
        raise NotImplementedError(f"FP8 scale blocks must be a multiple of 16 columns, got {bc}")
    dev = gate.device
    I_p, H_k, H_f = _ceil(inter, 128), _ceil(hidden, 64), _ceil(hidden, 128)
    w1 = torch.zeros(E, 2, I_p, H_k, device=dev, dtype=torch.uint8)
    w1[:, 0, :inter, :hidden] = gate.view(torch.uint8)
    w1[:, 1, :inter, :hidden] = up.view(torch.uint8)
    w2 = torch.zeros(E, H_f, I_p, device=dev, dtype=torch.uint8)
    w2[:, :hidden, :inter] = down.view(torch.uint8)
    s1 = torch.stack([gate_scale.float(), up_scale.float()], dim=1).contiguous()
    s2 = down_scale.float().contiguous()
    return ExpertWeights(_lib.W_FP8, E, hidden, inter,
                         pack_fp8_blobs(w1, s1, 2, inter, (br, bc)),
                         pack_fp8_blobs(w2.unsqueeze(1), s2.unsqueeze(1), 1, hidden, (br, bc)),
                         block=(br, bc))


def quantize_int8(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[..., channels, K] -> int8 of the same shape and fp32 scales [...,
    channels]: amax / 127 per channel (1 for a channel of zeros, NaN for one
    that holds NaN or an infinity, with codes 0), round to nearest even."""
    w = w.float()
    scale = w.abs().amax(dim=-1) / 127.0
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    scale = torch.where(scale.isfinite(), scale, torch.full_like(scale, torch.nan))
    return torch.round(w / scale[..., None]).clamp_(-127, 127).nan_to_num_(0.0).to(torch.int8), scale


def _int8_rows(t: torch.Tensor) -> torch.Tensor:
    """[E, planes, F_p, ...] -> [E, feat_tiles, 128, ...] in the int8 tiles' row
    order (two planes: 16 gate rows, then the 16 up rows of the same features)."""
    E, P, F = t.shape[:3]
    rest = tuple(t.shape[3:])
    if P == 2:
        return t.reshape(E, 2, F // 16, 16, *rest).transpose(1, 2).reshape(E, F // 64, 128, *rest)
    return t.reshape(E, F // 128, 128, *rest)


def _int8_tiles(w: torch.Tensor, feat_pad: int, k_pad: int) -> torch.Tensor:
    """int8 [E, planes, F, K] -> [E, feat_tiles, k_pad / 128, 128, 128] images."""
    E, P, F, K = w.shape
    ft, nkb = feat_pad // (64 if P == 2 else 128), k_pad // 128
    out = torch.empty(E, ft, nkb, 128, 128, device=w.device, dtype=torch.int8)
    words = out.view(torch.int64).view(E, ft, nkb, 16, 8, 8, 2)     # [.., row / 8, row % 8, 16-byte chunk, word]
    chunk = torch.arange(8, device=w.device)
    step = max(1, (256 << 20) // (P * feat_pad * k_pad))            # experts at a time: bounds the scratch memory
    for e in range(0, E, step):
        part = w[e:e + step]
        if (F, K) != (feat_pad, k_pad) or not part.is_contiguous() or part.data_ptr() % 8:
            full = torch.zeros(part.shape[0], P, feat_pad, k_pad, device=w.device, dtype=torch.int8)
            full[:, :, :F, :K] = part
            part = full
        rows = _int8_rows(part.view(torch.int64)).view(-1, ft, 16, 8, nkb, 8, 2)
        for r in range(8):
            words[e:e + step, :, :, :, r] = rows[:, :, :, r].index_select(4, chunk ^ r).transpose(2, 3)
    return out


def _int8_channels(v: torch.Tensor | None, feat_pad: int) -> torch.Tensor | None:
    """fp32 [E, planes, F] -> [E, feat_tiles, 128] in the tiles' row order."""
    if v is None:
        return None
    E, P, F = v.shape
    full = torch.zeros(E, P, feat_pad, device=v.device, dtype=torch.float32)
    full[:, :, :F] = v
    return _int8_rows(full).contiguous()


def _check_int8(w: torch.Tensor, scale: torch.Tensor, what: str) -> None:
    if w.dtype != torch.int8:
        raise ValueError(f"{what} weights must be int8, got {w.dtype}")
    if scale.shape != w.shape[:-1]:
        raise ValueError(f"{what} needs one scale per channel {tuple(w.shape[:-1])}, got {tuple(scale.shape)}")


def _planes(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """[E, 2, I, H] of the two; no copy where they already lie so in memory."""
    E, inter, hidden = gate.shape
    size = inter * hidden
    if (gate.stride() == up.stride() == (2 * size, hidden, 1) and up.data_ptr() == gate.data_ptr() + size
            and gate.untyped_storage().data_ptr() == up.untyped_storage().data_ptr()):
        return gate.as_strided((E, 2, inter, hidden), (2 * size, size, hidden, 1))
    return torch.stack([gate, up], dim=1)


def int8_experts(gate: torch.Tensor, gate_scale: torch.Tensor, up: torch.Tensor, up_scale: torch.Tensor,
                 down: torch.Tensor, down_scale: torch.Tensor, gate_bias: torch.Tensor | None = None,
                 up_bias: torch.Tensor | None = None, down_bias: torch.Tensor | None = None,
                 gated_epilogue: int = _lib.EPI_SWIGLU_F32, alpha: float = 1.702,
                 limit: float = 7.0) -> ExpertWeights:
    """gate/up: int8 [E, I, H] with scales [E, I]; down: int8 [E, H, I] with
    scales [E, H]; biases [E, I] / [E, H]."""
    E, inter, hidden = gate.shape
    _check_dims(hidden, inter)
    for w, s, what in ((gate, gate_scale, "gate"), (up, up_scale, "up"), (down, down_scale, "down")):
        _check_int8(w, s, what)
    if up.shape != gate.shape or down.shape != (E, hidden, inter):
        raise ValueError("gate, up and down shapes disagree")
    if gated_epilogue not in (_lib.EPI_SWIGLU_F32, _lib.EPI_CLAMP_SWIGLU_F32):
        raise ValueError("int8 experts gate with SWIGLU_F32 or CLAMP_SWIGLU_F32")
    if (gate_bias is None) != (up_bias is None):
        raise ValueError("gate and up biases come together")
    I_p, H_p = _ceil(inter, 128), _ceil(hidden, 128)
    b1 = None if gate_bias is None else torch.stack([gate_bias.float(), up_bias.float()], dim=1)
    b2 = None if down_bias is None else down_bias.float()[:, None]
    m1 = Int8Matrix(E, 2, inter, hidden, I_p, H_p, _int8_tiles(_planes(gate, up), I_p, H_p),
                    _int8_channels(torch.stack([gate_scale.float(), up_scale.float()], dim=1), I_p),
                    _int8_channels(b1, I_p), gated_epilogue, alpha, limit)
    m2 = Int8Matrix(E, 1, hidden, inter, H_p, I_p, _int8_tiles(down[:, None], H_p, I_p),
                    _int8_channels(down_scale.float()[:, None], H_p), _int8_channels(b2, H_p), _lib.EPI_DOWN_ONCE)
    return ExpertWeights(_lib.W_INT8, E, hidden, inter, m1.weight, m2.weight, s1=m1.scale, s2=m2.scale, b1=m1.bias,
                         b2=m2.bias, gated_epilogue=gated_epilogue, alpha=alpha, limit=limit, m1=m1, m2=m2)


def int8_experts_from(gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, **more) -> ExpertWeights:
    """``int8_experts`` of floating-point weights, quantised per channel."""
    parts = [t for w in (gate, up, down) for t in quantize_int8(w)]
    return int8_experts(*parts, **more)


def int8_linear(weight: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None) -> Int8Matrix:
    """A dense projection: int8 weight [N, K] with one scale per output channel
    [N], bias [N]."""
    if weight.dim() != 2:
        raise ValueError("weight must be [out_features, in_features]")
    _check_int8(weight, scale, "linear")
    N, K = weight.shape
    _check_dims(K, N)
    N_p, K_p = _ceil(N, 128), _ceil(K, 128)
    return Int8Matrix(1, 1, N, K, N_p, K_p, _int8_tiles(weight[None, None], N_p, K_p),
                      _int8_channels(scale.float()[None, None], N_p),
                      _int8_channels(None if bias is None else bias.float()[None, None], N_p), _lib.EPI_DOWN_ONCE)


def bf16_experts(gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor,
                 gate_bias: torch.Tensor | None = None, up_bias: torch.Tensor | None = None,
                 down_bias: torch.Tensor | None = None,
                 gated_epilogue: int = _lib.EPI_SWIGLU, alpha: float = 1.702,
                 limit: float = 7.0) -> ExpertWeights:
    """K-major bf16: gate/up [E, I, H], down [E, H, I]."""
    E, inter, hidden = gate.shape
    _check_dims(hidden, inter)
    dev = gate.device
    I_p, H_k, H_f = _ceil(inter, 128), _ceil(hidden, 64), _ceil(hidden, 128)
    w1 = torch.zeros(E, 2, I_p, H_k, device=dev, dtype=torch.bfloat16)
    w1[:, 0, :inter, :hidden] = gate
    w1[:, 1, :inter, :hidden] = up
    w2 = torch.zeros(E, H_f, I_p, device=dev, dtype=torch.bfloat16)
    w2[:, :hidden, :inter] = down
    b1 = b2 = None
    if gate_bias is not None:
        b1 = torch.zeros(E, 2, I_p, device=dev, dtype=torch.bfloat16)
        b1[:, 0, :inter] = gate_bias
        b1[:, 1, :inter] = up_bias
    if down_bias is not None:
        b2 = torch.zeros(E, H_f, device=dev, dtype=torch.bfloat16)
        b2[:, :hidden] = down_bias
    return ExpertWeights(_lib.W_BF16, E, hidden, inter, w1, w2, b1=b1, b2=b2,
                         gated_epilogue=gated_epilogue, alpha=alpha, limit=limit)


def gpt_oss_mxfp4_experts(gu_blocks: torch.Tensor, gu_scales: torch.Tensor,
                          gu_bias: torch.Tensor, dn_blocks: torch.Tensor,
                          dn_scales: torch.Tensor, dn_bias: torch.Tensor, alpha: float,
                          limit: float) -> ExpertWeights:
    """GPT-OSS packed experts: gate_up blocks [E, 2I, H/32, 16] u8 (interleaved
    gate/up rows), scales [E, 2I, H/32]; down blocks [E, H, I/32, 16]."""
    E, two_i, G, _ = gu_blocks.shape
    inter = two_i // 2
    hidden = G * 32
    _check_dims(hidden, inter)
    if dn_blocks.shape[1] != hidden or dn_blocks.shape[2] * 32 != inter:
        raise ValueError("down_proj blocks do not match gate_up_proj blocks")
    dev = gu_blocks.device
    I_p, H_k, H_f = _ceil(inter, 128), _ceil(hidden, 64), _ceil(hidden, 128)
    G1 = H_k // 32
    w1 = torch.zeros(E, 2, I_p, G1 * 16, device=dev, dtype=torch.uint8)
    s1 = torch.full((E, 2, I_p, G1), 127, device=dev, dtype=torch.uint8)
    gu = gu_blocks.reshape(E, two_i, G * 16)
    w1[:, 0, :inter, : G * 16] = gu[:, 0::2]
    w1[:, 1, :inter, : G * 16] = gu[:, 1::2]
    s1[:, 0, :inter, :G] = gu_scales[:, 0::2]
    s1[:, 1, :inter, :G] = gu_scales[:, 1::2]
    b1 = torch.zeros(E, 2, I_p, device=dev, dtype=torch.bfloat16)
    b1[:, 0, :inter] = gu_bias[:, 0::2].to(torch.bfloat16)
    b1[:, 1, :inter] = gu_bias[:, 1::2].to(torch.bfloat16)
    G2 = dn_blocks.shape[2]
    G2p = I_p // 32
    w2 = torch.zeros(E, H_f, G2p * 16, device=dev, dtype=torch.uint8)
    s2 = torch.full((E, H_f, G2p), 127, device=dev, dtype=torch.uint8)
    w2[:, :hidden, : G2 * 16] = dn_blocks.reshape(E, hidden, G2 * 16)
    s2[:, :hidden, :G2] = dn_scales
    b2 = torch.zeros(E, H_f, device=dev, dtype=torch.bfloat16)
    b2[:, :hidden] = dn_bias.to(torch.bfloat16)
    return ExpertWeights(_lib.W_MXFP4, E, hidden, inter, pack_mxfp4_blobs(w1, s1, 2),
                         pack_mxfp4_blobs(w2.unsqueeze(1), s2.unsqueeze(1), 1), b1=b1, b2=b2,
                         gated_epilogue=_lib.EPI_CLAMP_SWIGLU, alpha=alpha, limit=limit)


def gpt_oss_bf16_experts(gate_up: torch.Tensor, gate_up_bias: torch.Tensor,
                         down: torch.Tensor, down_bias: torch.Tensor, alpha: float,
                         limit: float) -> ExpertWeights:
    """GPT-OSS bf16 storage: gate_up [E, H, 2I] (interleaved columns), down [E, I, H]."""
    gate = gate_up[:, :, 0::2].transpose(1, 2)
    up = gate_up[:, :, 1::2].transpose(1, 2)
    return bf16_experts(gate, up, down.transpose(1, 2), gate_up_bias[:, 0::2],
                        gate_up_bias[:, 1::2], down_bias,
                        gated_epilogue=_lib.EPI_CLAMP_SWIGLU, alpha=alpha, limit=limit)
