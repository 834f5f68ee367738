/* The operators' gfx950 code object, embedded beside the executor's. */
    .section .rodata
    .global mx_ops_hsaco
    .p2align 12
mx_ops_hsaco:
    .incbin HSACO_PATH
    .byte 0
    .section .note.GNU-stack,"",@progbits
