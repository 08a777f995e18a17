"""sparc_amd: MI355X-native (gfx950) SPARC chunked diagonal linear scan.

Drop-in for the reference's ``sparc`` module surface on the scan path
(sparc-kernal/sparc.py): ``SPARCMixer`` and the scan operators, dispatching
to hand-written HIP kernels through the C ABI in include/sparc_hip.h.
"""
from .attention import linear_attention, linear_attention_step, qk_norm_rotary, rotary_table
from .beam import BeamStep, beam_search_step, reorder_states
from .clip import clip_grad_norm_, grad_norm
from .control import latest_sparc_write, make_controls, make_scan_inputs
from .decode import latest_sparc_decode, prepare_decode, run_decode_step
from .embed import embedding
from .feed_forward import gated_linear_unit
from .norm import layer_norm
from .ops import (
    chunk_scan,
    complex_scan,
    complex_scan_with_last,
    grouped_real_scan,
    polar_chunk_scan,
    real_chunk_scan,
    real_scan,
    real_scan_with_last,
    scan_step,
    sparc_chunk_scan,
    sparc_scan,
    sparc_scan_with_last,
    sparc_tiled_serial_scan,
    sparc_training_scan_dispatch,
)
from .mixer import backward_form, get_mixer_path, set_backward_plan, set_mixer_path
from .sparc import SPARCMixer, run_sequence

__all__ = [
    "SPARCMixer", "run_sequence", "make_controls", "make_scan_inputs", "latest_sparc_write",
    "prepare_decode", "run_decode_step", "latest_sparc_decode", "chunk_scan", "complex_scan",
    "complex_scan_with_last", "real_scan", "real_chunk_scan", "real_scan_with_last",
    "sparc_scan", "sparc_scan_with_last", "sparc_chunk_scan", "sparc_tiled_serial_scan",
    "sparc_training_scan_dispatch", "polar_chunk_scan", "grouped_real_scan", "scan_step",
    "set_mixer_path", "get_mixer_path", "set_backward_plan", "backward_form",
    "layer_norm", "embedding", "grad_norm", "clip_grad_norm_", "BeamStep", "beam_search_step", "reorder_states",
    "rotary_table", "qk_norm_rotary", "linear_attention", "linear_attention_step", "gated_linear_unit",
]
