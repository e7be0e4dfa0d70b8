"""specdec on MI355X: the speculative-decoding verification path as HIP kernels.

Drop-in for the reference package's hot path:
  specdec.sampling      to_probs, sample_from_probs, residual_probs, gather_prob,
                        rejection_sample (+ token_logprobs, penalize_logits)
  specdec.kvcache       RaggedCache (+ PagedKVCache for the shared-block-table layout,
                        build_block_tables, paged_slot_mapping, append_paged_slots, compact_paged,
                        free_page_list, fork_block_tables, copy_pages)
  specdec.attention     verify_attention_paged, shared_prefix_attention_paged,
                        tree_attention_paged
  specdec.tree          tree_layout, tree_accept
  specdec.proposer_ops  greedy_draft_tokens, drafting_slot_mapping
  specdec.controller    expected_speedup, best_k
The native library (libspecdec_amd.so) is loaded on first use.
"""
__version__ = "0.1.0"
