"""Temporal attention over whole clips: a residual block along the frame axis, for models that look further back than the receptive field
of the dilated convolutions (243 frames at most in the reference's configurations).

    out = LayerNorm(x + Dropout(W_o A(rot(W_q x), rot(W_k x), W_v x)))        x: (B, T, J, C), every joint a sequence of its own

A is causal linear attention with a decay for each head, rot the rotary positions (gast_hip/temporal.py), so a frame costs the same
however long the clip is, and `step` continues a stream frame by frame on a state of heads x D x D numbers per joint.  The reference has no
such block; this one is trainable and fp32 like the stand-alone graph sub-modules (gast_hip/modules.py), whose GEMMs it runs on."""
import torch
from torch import nn


class TemporalState:
    """Where a batch of streams is: S (B, J, H, D, D) float32 and the position (B, 1) int64 of the next frame of each."""

    def __init__(self, S, position):
        self.S, self.position = S, position


class TemporalAttention(nn.Module):
    """block = TemporalAttention(channels, heads=4, dropout=None); y = block(x, lengths=None) with x (B, T, J, C)
       state = block.state(batch, joints); y = block.step(frame, state) with frame (B, J, C): eval mode, one frame per call
       shortest / longest: the decays of the first and the last head, in frames (the others lie between them, evenly in the logarithm)"""

    def __init__(self, channels, heads=4, dropout=None, rotary_dim=None, base=10000.0, shortest=32.0, longest=4096.0):
        super().__init__()
        if channels % heads:
            raise ValueError('TemporalAttention: %d channels do not divide into %d heads' % (channels, heads))
        if not 1.0 <= shortest <= longest:
            raise ValueError('TemporalAttention: 1 <= shortest <= longest, got %r and %r' % (shortest, longest))
        from gast_hip.temporal import rotary_frequencies
        self.channels, self.heads = channels, heads
        width = channels // heads
        rotary_dim = width // 2 * 2 if rotary_dim is None else rotary_dim
        if rotary_dim > width:
            raise ValueError('TemporalAttention: rotary_dim %d of %d channels a head' % (rotary_dim, width))
        self.qkv = nn.Linear(channels, 3 * channels)
        self.out = nn.Linear(channels, channels)
        self.norm = nn.LayerNorm(channels)
        self.dropout = None if dropout is None else nn.Dropout(dropout)
        frames = shortest * (longest / shortest) ** torch.linspace(0.0, 1.0, heads, dtype=torch.float64)
        self.register_buffer('log_decay', torch.log1p(-1.0 / frames.clamp(min=1.0 + 1e-9)).float())
        self._freqs = rotary_frequencies(rotary_dim, base) if rotary_dim else None      # (not a buffer: .half() must not round it)

    def freqs(self, dev):
        if self._freqs is not None and self._freqs.device != dev:
            self._freqs = self._freqs.to(dev)
        return self._freqs

    def forward(self, x, lengths=None):
        """x (B, T, J, C); lengths (B,): the frames of each clip, the rest is padding that no frame sees"""
        from gast_hip.modules import temporal_attention_forward
        return temporal_attention_forward(self, x, lengths)

    def state(self, batch, joints):
        dev, D = self.qkv.weight.device, self.channels // self.heads
        return TemporalState(torch.zeros(batch, joints, self.heads, D, D, dtype=torch.float32, device=dev),
                             torch.zeros(batch, 1, dtype=torch.int64, device=dev))

    def step(self, x, state, active=None):
        """x (B, J, C): the next frame of every stream -> (B, J, C), `state` moved on in place.  active (B,) int32: streams with 0 have no
        frame this time (their state stays; their rows of the result mean nothing)"""
        from gast_hip.modules import temporal_attention_step
        return temporal_attention_step(self, x, state, active)
