"""Data transforms (split/rANS codec, fp8 packing) and losses over the vocabulary."""
