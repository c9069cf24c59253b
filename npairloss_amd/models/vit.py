"""ViT-B/16 embedding backbones (from scratch): 768-d embeddings, fp8-capable
MFMA similarity path, batches sized for the 288 GB HBM3E per MI355X.

ViTB16 takes images of one size with learned positions.  RotaryViTB16 takes images
of any size, one size to a batch or packed into rows, on this framework's own
operators: RMS norm with the residual's addition, rotary positions over rows and
columns, attention under a document mask."""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch
from torch import nn

from ..ops import attention, rms_norm, rotary, rotary_frequencies


class Block(nn.Module):
    def __init__(self, dim: int, heads: int, mlp_ratio: float = 4.0):
        super().__init__()
        self.norm1 = nn.LayerNorm(dim)
        self.attn = nn.MultiheadAttention(dim, heads, batch_first=True)
        self.norm2 = nn.LayerNorm(dim)
        hidden = int(dim * mlp_ratio)
        self.mlp = nn.Sequential(nn.Linear(dim, hidden), nn.GELU(), nn.Linear(hidden, dim))

    def forward(self, x):
        a, _ = self.attn(self.norm1(x), self.norm1(x), self.norm1(x), need_weights=False)
        x = x + a
        return x + self.mlp(self.norm2(x))


class ViTB16(nn.Module):
    def __init__(self, image_size: int = 224, patch: int = 16, dim: int = 768,
                 depth: int = 12, heads: int = 12, embed_dim: int = 768):
        super().__init__()
        self.embed_dim = embed_dim
        self.patch_embed = nn.Conv2d(3, dim, patch, stride=patch)
        n_patches = (image_size // patch) ** 2
        self.cls = nn.Parameter(torch.zeros(1, 1, dim))
        self.pos = nn.Parameter(torch.zeros(1, n_patches + 1, dim))
        self.blocks = nn.Sequential(*[Block(dim, heads) for _ in range(depth)])
        self.norm = nn.LayerNorm(dim)
        self.proj = nn.Identity() if embed_dim == dim else nn.Linear(dim, embed_dim)
        nn.init.trunc_normal_(self.pos, std=0.02)
        nn.init.trunc_normal_(self.cls, std=0.02)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x = self.patch_embed(x).flatten(2).transpose(1, 2)  # B x N x D
        x = torch.cat([self.cls.expand(x.shape[0], -1, -1), x], dim=1) + self.pos
        x = self.norm(self.blocks(x))
        return self.proj(x[:, 0])


class RotaryBlock(nn.Module):
    """A pre-norm block over a stream and the branch that is to be added to it: the
    addition happens in the norm that reads the sum."""

    def __init__(self, dim: int, heads: int, mlp_ratio: float = 4.0, softcap: float = 0.0):
        super().__init__()
        self.heads, self.softcap = heads, softcap
        self.norm1 = nn.Parameter(torch.ones(dim))
        self.qkv = nn.Linear(dim, 3 * dim)
        self.out = nn.Linear(dim, dim)
        self.norm2 = nn.Parameter(torch.ones(dim))
        hidden = int(dim * mlp_ratio)
        self.mlp = nn.Sequential(nn.Linear(dim, hidden), nn.GELU(), nn.Linear(hidden, dim))

    def forward(self, branch: Optional[torch.Tensor], stream: torch.Tensor, positions: torch.Tensor, turns: Tuple[torch.Tensor, float],
                documents: Optional[torch.Tensor] = None, read: Optional[torch.Tensor] = None,
                read_documents: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(branch, stream) behind the block.  With `read` [rows, tokens] (places of
        tokens at position 0) only those go on: they attend to all tokens."""
        frequencies, amplitude = turns
        if branch is None:
            h = rms_norm(stream, self.norm1)
        else:
            h, stream = rms_norm(branch, self.norm1, stream)
        B, N, dim = h.shape
        heads = lambda x, parts: x.view(B, x.shape[1], parts, self.heads, dim // self.heads).unbind(2)  # noqa: E731
        if read is None:
            q, k, v = heads(self.qkv(h), 3)
            q, k = rotary(q, k, positions, frequencies, amplitude=amplitude)
            a = attention(q, k, v, softcap=self.softcap, documents=documents)
        else:
            at = read.unsqueeze(-1).expand(-1, -1, dim)
            stream = stream.gather(1, at)
            (q,) = heads(nn.functional.linear(h.gather(1, at), self.qkv.weight[:dim], self.qkv.bias[:dim]), 1)
            k, v = heads(nn.functional.linear(h, self.qkv.weight[dim:], self.qkv.bias[dim:]), 2)
            k = rotary(k, None, positions, frequencies, amplitude=amplitude)
            q = q if amplitude == 1.0 else q * amplitude  # a turn by no angle
            a = attention(q, k, v, softcap=self.softcap, documents=read_documents, key_documents=documents)
        h, stream = rms_norm(self.out(a.reshape(B, -1, dim)), self.norm2, stream)
        return self.mlp(h), stream


class RotaryViTB16(nn.Module):
    """ViT-B/16 with RMS norms and rotary positions over the rows and columns of an
    image's patches.  The class token stands at (0, 0), patches at (1, 1) and on; the
    last block computes the class token's row alone."""

    def __init__(self, patch: int = 16, dim: int = 768, depth: int = 12, heads: int = 12, embed_dim: int = 768,
                 softcap: float = 0.0, base: float = 100.0, scaling: Optional[str] = None, factor: float = 1.0,
                 original_length: int = 0):
        super().__init__()
        if dim % heads or dim // heads % 4:
            raise ValueError(f"RotaryViTB16: {heads} heads of {dim} have no two axes of pairs")
        self.embed_dim, self.patch, self.dim = embed_dim, patch, dim
        self.patch_embed = nn.Linear(3 * patch * patch, dim)
        self.cls = nn.Parameter(torch.zeros(dim))
        self.blocks = nn.ModuleList([RotaryBlock(dim, heads, softcap=softcap) for _ in range(depth)])
        self.norm = nn.Parameter(torch.ones(dim))
        self.proj = nn.Identity() if embed_dim == dim else nn.Linear(dim, embed_dim)
        frequencies, self.amplitude = rotary_frequencies(dim // heads, axes=2, base=base, scaling=scaling, factor=factor,
                                                         original_length=original_length)
        self._frequencies = {None: frequencies}  # fp64 on every device, whatever type the model is cast to
        nn.init.trunc_normal_(self.cls, std=0.02)

    def _turns(self, device: torch.device) -> Tuple[torch.Tensor, float]:
        if device not in self._frequencies:
            with torch.inference_mode(False):  # training may come after: it cannot save what inference mode made
                self._frequencies[device] = self._frequencies[None].to(device)
        return self._frequencies[device], self.amplitude

    def _patches(self, image: torch.Tensor) -> torch.Tensor:
        """[..., 3, h, w] to [..., patches, 3 patch^2], row by row."""
        p = self.patch
        *lead, c, h, w = image.shape
        if h % p or w % p or h == 0 or w == 0:
            raise ValueError(f"RotaryViTB16: sides are multiples of {p}, got {h} x {w}")
        image = image.reshape(*lead, c, h // p, p, w // p, p)
        n = len(lead)
        return image.permute(*range(n), n + 1, n + 3, n, n + 2, n + 4).reshape(*lead, (h // p) * (w // p), c * p * p)

    @staticmethod
    def _grid(rows: int, columns: int, device: torch.device) -> torch.Tensor:
        """Positions of the class token and the patches, [1 + rows * columns, 2]."""
        r = torch.arange(1, rows + 1, device=device).repeat_interleave(columns)
        c = torch.arange(1, columns + 1, device=device).repeat(rows)
        return torch.cat([torch.zeros(1, 2, dtype=torch.long, device=device), torch.stack([r, c], -1)])

    def _run(self, x, positions, documents, read, read_documents):
        turns = self._turns(x.device)
        branch, stream = None, x
        for block in self.blocks[:-1]:
            branch, stream = block(branch, stream, positions, turns, documents)
        branch, stream = self.blocks[-1](branch, stream, positions, turns, documents, read, read_documents)
        return rms_norm(branch, self.norm, stream)[0]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """Embeddings of a batch of images of one size."""
        B, _, h, w = x.shape
        patches = self.patch_embed(self._patches(x))
        tokens = torch.cat([self.cls.to(patches.dtype).expand(B, 1, -1), patches], 1)
        positions = self._grid(h // self.patch, w // self.patch, x.device)
        read = torch.zeros(B, 1, dtype=torch.long, device=x.device)
        return self.proj(self._run(tokens, positions, None, read, None)[:, 0])

    def forward_packed(self, images: Sequence[torch.Tensor], row_length: int = 0) -> torch.Tensor:
        """Embeddings [images, embed_dim] of images [3, h, w] of any sizes, packed into
        rows of `row_length` tokens (by default what the largest image needs, at least
        1024), each image seeing itself alone.  The plan is the host's: shapes say it all."""
        if not images:
            raise ValueError("RotaryViTB16: no images")
        device = images[0].device
        grids = [(im.shape[-2] // self.patch, im.shape[-1] // self.patch) for im in images]
        lengths = [1 + r * c for r, c in grids]
        row_length = row_length or max(1024, max(lengths))
        if max(lengths) > row_length:
            raise ValueError(f"RotaryViTB16: an image of {max(lengths)} tokens does not fit rows of {row_length}")
        rows: List[List[int]] = []
        left: List[int] = []
        for i in sorted(range(len(images)), key=lambda i: -lengths[i]):  # the first row that has room, largest first
            for r, room in enumerate(left):
                if lengths[i] <= room:
                    break
            else:
                r = len(rows)
                rows.append([])
                left.append(row_length)
            rows[r].append(i)
            left[r] -= lengths[i]
        order = [i for row in rows for i in row]
        most = max(len(row) for row in rows)
        documents = torch.full((len(rows), row_length), -1, dtype=torch.int32)
        read = torch.zeros(len(rows), most, dtype=torch.long)
        read_documents = torch.full((len(rows), most), -1, dtype=torch.int32)
        place = torch.empty(len(images), dtype=torch.long)       # of an image's answer
        cls_at, patch_at = [], []                                 # of tokens in the rows, laid flat
        for r, row in enumerate(rows):
            at = 0
            for n, i in enumerate(row):
                documents[r, at:at + lengths[i]] = n
                read[r, n], read_documents[r, n], place[i] = at, n, r * most + n
                cls_at.append(r * row_length + at)
                patch_at.append(torch.arange(r * row_length + at + 1, r * row_length + at + lengths[i]))
                at += lengths[i]
        documents, read, read_documents, place = (x.to(device) for x in (documents, read, read_documents, place))
        cls_at, patch_at = torch.tensor(cls_at, device=device), torch.cat(patch_at).to(device)
        patches = self.patch_embed(torch.cat([self._patches(images[i]) for i in order]))
        flat = patches.new_zeros(len(rows) * row_length, self.dim)
        flat = flat.index_copy(0, patch_at, patches).index_copy(0, cls_at, self.cls.to(patches.dtype).expand(len(order), -1))
        positions = torch.zeros(len(rows) * row_length, 2, dtype=torch.long, device=device)
        grid = torch.cat([self._grid(*grids[i], device)[1:] for i in order])
        positions[patch_at] = grid
        out = self._run(flat.view(len(rows), row_length, -1), positions.view(len(rows), row_length, 2), documents, read, read_documents)
        return self.proj(out.reshape(-1, out.shape[-1])[place])
