/* A gfx950 code object, embedded under the name BLOB. */
    .section .rodata
    .global BLOB
    .p2align 12
BLOB:
    .incbin HSACO_PATH
    .byte 0
    .section .note.GNU-stack,"",@progbits
